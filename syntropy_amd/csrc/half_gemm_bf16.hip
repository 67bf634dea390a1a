// half_gemm.hpp's kernels over BF16 values (a file a type: each takes minutes to compile).
#include "half_gemm.hpp"

namespace syn {

void launch_half_gemm_bf16(int tile, const HalfArgs& a, hipStream_t stream) { launch_half_tile<T_BF16>(tile, a, stream); }

}  // namespace syn
