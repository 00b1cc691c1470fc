// The tensor-core kernel with the fused epilogue (kFused), one instantiation for each tile shape that the
// planner of gemm_tc.cu chooses; a cut contraction applies the epilogue in the kernel that sums its parts.
#include "tc_kernel.cuh"

namespace hc {

// Epilogue warps and operand slots share the shared memory of a 256x256 tile: eight warps leave four slots, four warps five.  Five
// slots keep the tensor cores busier (8192 x 4096 x 8192, no extras: 389 -> 372 us, the plain product's time; with the
// pre-activation kept 472 -> 438); eight warps are needed where an epilogue would outlast the main loop (8192 x 1024 x 8192 with
// GELU: 126 us, with four warps 149; x 2048 with residual and pre-activation 278, 400; times a slope 243, 270).
TcLaunchFn fused_kernel(bool f32, int shape, int kslabs, const FusedEpilogue& fe) {
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
      if (kslabs >= 64 || (kslabs >= 32 && !(fe.aux && (fe.grad || fe.pre))))
        return TcConfig<2, 256, 5, 4, false, 2, 1, 1, false, kFused>::launch;
      return TcConfig<2, 256, 4, 8, false, 2, 1, 1, false, kFused>::launch;
    case SHAPE_C1_256: return TcConfig<2, 256, 3, 4, false, 1, 1, 1, false, kFused>::launch;
    case SHAPE_C1_128: return TcConfig<2, 128, 5, 4, false, 1, 1, 1, false, kFused>::launch;
    default: return nullptr;
  }
}

}  // namespace hc
