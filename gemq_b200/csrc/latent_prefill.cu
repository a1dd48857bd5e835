// Attention of whole prompts over expanded keys and values, head size 128 + 64 and 128.
//
//   s[i, j] = scale * (q_nope[i] . k_nope[j] + q_rope[i] . k_rope[j]),   out[i] = sum_j softmax(s)[i, j] v[j],   j <= i + keys - queries
//
// A warp a query row of one head; running maximum and sum in 32 bits.
#include "latent.cuh"

namespace gemq {
namespace latent {
namespace {

constexpr int kWarps = 8;
constexpr int kNope = 128, kValue = 128;

template <typename T>
__global__ void __launch_bounds__(32 * kWarps) latent_prefill_row_kernel(const gemq_latent_prefill_t P) {
  const int lane = threadIdx.x & 31;
  const long long at = blockIdx.x * static_cast<long long>(kWarps) + (threadIdx.x >> 5);
  const int row = static_cast<int>(at / P.heads), h = static_cast<int>(at % P.heads);
  if (row >= P.q_rows) return;
  if (at == 0 && lane == 0 && !(offsets_ok(P.cu_q, P.batch, P.q_rows, false) && offsets_ok(P.cu_k, P.batch, P.k_rows, false)))
    atomicExch(P.err, GEMQ_LATENT_BAD_LENGTH);
  int b = -1;
  for (int i = 0; i < P.batch; ++i)
    if (row >= P.cu_q[i] && row < P.cu_q[i + 1]) { b = i; break; }
  int limit = 0, k0 = 0;
  if (b >= 0) {
    const int q0 = P.cu_q[b], q1 = P.cu_q[b + 1];
    int k1 = P.cu_k[b + 1];
    k0 = P.cu_k[b];
    if (k0 < 0 || k1 < k0 || k1 > P.k_rows) {
      if (lane == 0) atomicExch(P.err, GEMQ_LATENT_BAD_LENGTH);
      k0 = max(k0, 0);
      k1 = max(min(k1, P.k_rows), k0);
    }
    limit = P.causal ? row - q0 + 1 + (k1 - k0) - (q1 - q0) : k1 - k0;
  }
  const T* qn = static_cast<const T*>(P.q_nope) + row * P.q_nope_stride[0] + h * P.q_nope_stride[1];
  const T* qr = static_cast<const T*>(P.q_rope) + row * P.q_rope_stride[0] + h * P.q_rope_stride[1];
  const uint2 qv = reinterpret_cast<const uint2*>(qn)[lane];
  const float2 q0 = Pair<T>::f(qv.x), q1 = Pair<T>::f(qv.y), q2 = Pair<T>::f(reinterpret_cast<const uint32_t*>(qr)[lane]);
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < limit; ++j) {
    const T* kv = static_cast<const T*>(P.kv) + (k0 + j) * P.kv_stride[0] + h * P.kv_stride[1];
    const uint2 kn = reinterpret_cast<const uint2*>(kv)[lane], v = reinterpret_cast<const uint2*>(kv + kNope)[lane];
    const float2 a = Pair<T>::f(kn.x), c = Pair<T>::f(kn.y);
    const float2 d = Pair<T>::f(reinterpret_cast<const uint32_t*>(static_cast<const T*>(P.k_rope) + (k0 + j) * P.k_rope_stride)[lane]);
    float s = q0.x * a.x + q0.y * a.y + q1.x * c.x + q1.y * c.y + q2.x * d.x + q2.y * d.y;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= P.scale;
    const float now = fmaxf(m, s), base = now == -INFINITY ? 0.f : now;
    const float f = __expf(m - base), p = __expf(s - base);
    m = now;
    l = fmaf(l, f, p);
    const float2 v0 = Pair<T>::f(v.x), v1 = Pair<T>::f(v.y);
    o[0] = fmaf(o[0], f, p * v0.x);
    o[1] = fmaf(o[1], f, p * v0.y);
    o[2] = fmaf(o[2], f, p * v1.x);
    o[3] = fmaf(o[3], f, p * v1.y);
  }
  const long long out = static_cast<long long>(row) * P.heads + h;
  const float r = limit > 0 ? 1.f / l : 0.f;
  reinterpret_cast<uint2*>(static_cast<T*>(P.out) + out * kValue)[lane] = make_uint2(Pair<T>::r(o[0] * r, o[1] * r), Pair<T>::r(o[2] * r, o[3] * r));
  if (lane == 0) P.lse[out] = limit > 0 ? m + logf(l) : -INFINITY;
}

}  // namespace
}  // namespace latent
}  // namespace gemq

using namespace gemq;
using namespace gemq::latent;

extern "C" int gemq_latent_prefill(const gemq_latent_prefill_t* A, gemq_stream_t stream) {
  if (!A) return GEMQ_ERR_BAD_ARG;
  if (A->q_rows == 0) return GEMQ_OK;
  if (!A->q_nope || !A->q_rope || !A->cu_q || !A->cu_k || !A->out || !A->lse || !A->err || A->batch < 0 || A->q_rows < 0 || A->k_rows < 0 ||
      A->heads <= 0 || (A->k_rows && (!A->kv || !A->k_rope)))
    return GEMQ_ERR_BAD_ARG;
  if (static_cast<long long>(A->q_rows) * A->heads > (1ll << 31)) return GEMQ_ERR_BAD_SHAPE;
  for (const void* p : {A->q_nope, A->q_rope, A->kv, A->k_rope, static_cast<const void*>(A->out)})
    if (p && !aligned16(p)) return GEMQ_ERR_ALIGN;
  if ((A->q_nope_stride[0] | A->q_nope_stride[1] | A->q_rope_stride[0] | A->q_rope_stride[1] | A->kv_stride[0] | A->kv_stride[1] |
       A->k_rope_stride) & 7)
    return GEMQ_ERR_ALIGN;
  const long long rows = static_cast<long long>(A->q_rows) * A->heads;
  const unsigned grid = static_cast<unsigned>((rows + kWarps - 1) / kWarps);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (A->is_bf16)
    latent_prefill_row_kernel<__nv_bfloat16><<<grid, 32 * kWarps, 0, st>>>(*A);
  else
    latent_prefill_row_kernel<__half><<<grid, 32 * kWarps, 0, st>>>(*A);
  return launch_status();
}
