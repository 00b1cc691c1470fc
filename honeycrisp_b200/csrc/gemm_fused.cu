// The tensor-core kernel with the fused epilogue (kFused), one instantiation for each tile shape that the
// planner of gemm_tc.cu chooses; a cut contraction applies the epilogue in the kernel that sums its parts.
#include "tc_kernel.cuh"

namespace hc {

TcLaunchFn fused_kernel(bool f32, int shape) {
  if (f32) {
    switch (shape) {
      case SHAPE_PAIR_128: return TcConfig<4, 128, 4, 8, true, 2, 1, 1, false, kFused>::launch;
      case SHAPE_PAIR_64: return TcConfig<4, 64, 4, 8, true, 2, 1, 1, false, kFused>::launch;
      case SHAPE_C1_128: return TcConfig<4, 128, 3, 8, true, 1, 1, 1, false, kFused>::launch;
      default: return nullptr;
    }
  }
  switch (shape) {
    case SHAPE_PAIR_128: return TcConfig<2, 128, 3, 4, false, 2, 1, 2, false, kFused>::launch;
    case SHAPE_PAIR_64: return TcConfig<2, 64, 4, 4, false, 2, 1, 2, false, kFused>::launch;
    case SHAPE_PAIR:
      return TcConfig<2, 256, 4, 8, false, 2, 1, 1, false, kFused>::launch;
    case SHAPE_C1_256: return TcConfig<2, 256, 3, 4, false, 1, 1, 1, false, kFused>::launch;
    case SHAPE_C1_128: return TcConfig<2, 128, 5, 4, false, 1, 1, 1, false, kFused>::launch;
    default: return nullptr;
  }
}

}  // namespace hc
