// attention.cu -- attention over packed sequences and over a prefix that a batch shares (reaxmoe_attention).
#include <cstring>

#include "attention_rows.cuh"
#include "kernels.cuh"

namespace reaxmoe {
namespace attn {

template <int D, bool BF>
__global__ void __launch_bounds__(256) rows_kernel(const __grid_constant__ reaxmoe_attention_args a) {
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int t = (int)(row / a.q_heads);
  if (t >= min(__ldg(a.cu_q + a.seqs), (int)a.q_tokens)) return;
  row_by_warp<D, BF>(a, t, (int)(row % a.q_heads));
}

template <int D>
static int launch_d(const AttentionLaunch& l, cudaStream_t s) {
  const int64_t blocks = ceil_div64(l.a.q_tokens * l.a.q_heads, 8);
  if (l.a.dtype == REAXMOE_BF16)
    rows_kernel<D, true><<<(unsigned)blocks, 256, 0, s>>>(l.a);
  else
    rows_kernel<D, false><<<(unsigned)blocks, 256, 0, s>>>(l.a);
  return cudaPeekAtLastError() == cudaSuccess ? 0 : REAXMOE_ERR_CUDA;
}

}  // namespace attn

size_t attention_workspace(const reaxmoe_attention_args&, int) { return 256; }

int launch_attention(const AttentionLaunch& l, cudaStream_t s) {
  switch (l.a.head_dim) {
    case 64: return attn::launch_d<64>(l, s);
    case 128: return attn::launch_d<128>(l, s);
    default: return attn::launch_d<256>(l, s);
  }
}

}  // namespace reaxmoe
