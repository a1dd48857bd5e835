// Attention of decoded tokens over a paged latent cache.
//
//   s[r, t] = scale * (q_latent[r] . c[t] + q_rope[r] . k[t]),   out[r] = sum_t softmax(s)[r, t] c[t]
//
// A CTA a query row, its warps take the positions in turn; running maximum and sum in 32 bits.
#include "latent.cuh"

namespace gemq {
namespace latent {
namespace {

constexpr int kWarps = 8;

template <typename T>
__global__ void __launch_bounds__(32 * kWarps) latent_decode_row_kernel(const gemq_latent_decode_t P) {
  __shared__ float part_o[kWarps][512];
  __shared__ float part_m[kWarps], part_l[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row = blockIdx.x;
  const int h = static_cast<int>(row % P.heads), i = static_cast<int>(row / P.heads % P.steps), b = static_cast<int>(row / P.heads / P.steps);
  const int pieces = P.rank / 8, width = P.rank + kRope;
  const uint4* ql = reinterpret_cast<const uint4*>(static_cast<const T*>(P.q_latent) + b * P.q_latent_stride[0] + i * P.q_latent_stride[1] +
                                                   h * P.q_latent_stride[2]);
  const uint32_t* qr = reinterpret_cast<const uint32_t*>(static_cast<const T*>(P.q_rope) + b * P.q_rope_stride[0] +
                                                         i * P.q_rope_stride[1] + h * P.q_rope_stride[2]);
  float q[16], o[16];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint4 v = lane + 32 * k < pieces ? ql[lane + 32 * k] : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = Pair<T>::f(reinterpret_cast<const uint32_t*>(&v)[j]);
      q[8 * k + 2 * j] = f.x;
      q[8 * k + 2 * j + 1] = f.y;
      o[8 * k + 2 * j] = o[8 * k + 2 * j + 1] = 0.f;
    }
  }
  const float2 qp = Pair<T>::f(qr[lane]);

  int prefix = 0, group = 0;
  if (P.groups > 0) {
    if (row == 0 && threadIdx.x == 0 && !offsets_ok(P.starts, P.groups, P.batch, true)) atomicExch(P.err, GEMQ_LATENT_BAD_LENGTH);
    while (group + 1 < P.groups && P.starts[group + 1] <= b) ++group;
    prefix = clamp_length(P.prefix_lens[group], P.prefix_pitch, P.page_size, P.err);
  }
  const int own = clamp_length(P.lens[b], P.table_pitch, P.page_size, P.err);
  const int limit = prefix + own - (P.steps - 1 - i);
  float m = -INFINITY, l = 0.f;
  for (int t = warp; t < limit; t += kWarps) {
    const bool pre = t < prefix;
    const int at = pre ? t : t - prefix;
    const int page = pre ? P.prefix_table[static_cast<long long>(group) * P.prefix_pitch + at / P.page_size]
                         : P.table[static_cast<long long>(b) * P.table_pitch + at / P.page_size];
    float s;
    uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if (page < 0 || page >= P.n_pages) {
      if (lane == 0) atomicExch(P.err, GEMQ_LATENT_BAD_PAGE);
      s = __int_as_float(0x7fc00000);
    } else {
      const uint4* c = reinterpret_cast<const uint4*>(static_cast<const T*>(P.cache) + page * P.page_stride + (at % P.page_size) * width);
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (lane + 32 * k < pieces) v[k] = c[lane + 32 * k];
      const float2 kp = Pair<T>::f(reinterpret_cast<const uint32_t*>(c + pieces)[lane]);
      s = qp.x * kp.x + qp.y * kp.y;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = Pair<T>::f(reinterpret_cast<const uint32_t*>(&v[k])[j]);
          s = fmaf(q[8 * k + 2 * j], f.x, fmaf(q[8 * k + 2 * j + 1], f.y, s));
        }
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      s *= P.scale;
    }
    const float now = fmaxf(m, s), base = now == -INFINITY ? 0.f : now;
    const float f = __expf(m - base), p = __expf(s - base);
    m = now;
    l = fmaf(l, f, p);
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 g = Pair<T>::f(reinterpret_cast<const uint32_t*>(&v[k])[j]);
        o[8 * k + 2 * j] = fmaf(o[8 * k + 2 * j], f, p * g.x);
        o[8 * k + 2 * j + 1] = fmaf(o[8 * k + 2 * j + 1], f, p * g.y);
      }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (lane + 32 * k < pieces) part_o[warp][(lane + 32 * k) * 8 + j] = o[8 * k + j];
  if (lane == 0) {
    part_m[warp] = m;
    part_l[warp] = l;
  }
  __syncthreads();
  float top = -INFINITY, sum = 0.f, f[kWarps];
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, part_m[w]);
  const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    f[w] = __expf(part_m[w] - base);
    sum = fmaf(part_l[w], f[w], sum);
  }
  T* out = static_cast<T*>(P.out) + row * P.rank;
  for (int d = threadIdx.x * 2; d < P.rank; d += 64 * kWarps) {
    float a = 0.f, c = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      a = fmaf(part_o[w][d], f[w], a);
      c = fmaf(part_o[w][d + 1], f[w], c);
    }
    *reinterpret_cast<uint32_t*>(out + d) = limit > 0 ? Pair<T>::r(a / sum, c / sum) : 0u;
  }
  if (threadIdx.x == 0) P.lse[row] = limit > 0 ? top + logf(sum) : -INFINITY;
}

int check(const gemq_latent_decode_t* A) {
  if (!A || !A->q_latent || !A->q_rope || !A->cache || !A->table || !A->lens || !A->out || !A->lse || !A->err) return GEMQ_ERR_BAD_ARG;
  if (A->batch < 0 || A->steps <= 0 || A->heads <= 0 || A->n_pages <= 0 || A->table_pitch < 0 || A->groups < 0) return GEMQ_ERR_BAD_ARG;
  if (A->groups && (!A->prefix_table || !A->prefix_lens || !A->starts || A->prefix_pitch < 0)) return GEMQ_ERR_BAD_ARG;
  if (!rank_ok(A->rank) || !page_ok(A->page_size)) return GEMQ_ERR_BAD_SHAPE;
  if (static_cast<long long>(A->batch) * A->steps * A->heads > (1 << 30)) return GEMQ_ERR_BAD_SHAPE;
  if (!aligned16(A->q_latent) || !aligned16(A->q_rope) || !aligned16(A->cache) || !aligned16(A->out) || (A->page_stride & 7))
    return GEMQ_ERR_ALIGN;
  for (int i = 0; i < 3; ++i)
    if ((A->q_latent_stride[i] | A->q_rope_stride[i]) & 7) return GEMQ_ERR_ALIGN;
  return GEMQ_OK;
}

}  // namespace
}  // namespace latent
}  // namespace gemq

using namespace gemq;
using namespace gemq::latent;

extern "C" size_t gemq_latent_decode_scratch_bytes(const gemq_latent_decode_t* A) { return 0; }

extern "C" int gemq_latent_decode(const gemq_latent_decode_t* A, void* scratch, size_t scratch_bytes, gemq_stream_t stream) {
  const int rc = check(A);
  if (rc) return rc;
  const int rows = A->batch * A->steps * A->heads;
  if (!rows) return GEMQ_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (A->is_bf16)
    latent_decode_row_kernel<__nv_bfloat16><<<rows, 32 * kWarps, 0, st>>>(*A);
  else
    latent_decode_row_kernel<__half><<<rows, 32 * kWarps, 0, st>>>(*A);
  return launch_status();
}
