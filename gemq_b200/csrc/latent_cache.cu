// Rows of a paged latent cache: made from a projection's output and stored (gemq_latent_append), and copied from page to
// page (gemq_copy_pages).
//
//   row = { c * rsqrt(mean(c^2) + eps) * w,  rot(k, p) },   rot(x, p)[2i, 2i+1] = m * (x0 cos a - x1 sin a, x0 sin a + x1 cos a),  a = p * f_i
//
// Both move bytes and compute next to nothing.  Measured: 8191 rows of rank 512 with 16 heads' queries, 62 MB: 12.4 us (5.0 TB/s; 15.4 before
// the queries were asked for ahead of the norm); 391 pages in 27 layers, 1.56 GB: 269 us (5.8 TB/s, 0.88 of a plain copy's rate).
#include "latent.cuh"

namespace gemq {
namespace {

using latent::kRope;
using latent::Pair;
using latent::rank_ok;

struct AppendArgs {
  const void* kv;
  long long kv_stride;
  const void* q;
  long long q_token, q_head;
  const void* w;
  float eps;
  const float* inv_freq;
  float rope_scale;
  const long long* positions;
  const long long* slots;
  void* cache;
  long long page_stride;
  int n_pages, page_size;
  void* rows;
  void* q_out;
  int tokens, heads, rank;
  int* err;
};

// A warp a token: lane i has the angle of pair i.  The angle is formed in 64 bits and brought into [-pi, pi] there: in 32 bits a
// position of 160,000 times a frequency near 1 is off by up to 0.008.
constexpr int kAppendWarps = 4;

template <typename T>
__global__ void __launch_bounds__(32 * kAppendWarps) latent_append_kernel(const AppendArgs P) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, t = blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
  if (t >= P.tokens) return;
  const int width = P.rank + kRope;
  const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(P.kv) + t * P.kv_stride);
  const uint4* w = static_cast<const uint4*>(P.w);
  uint4 v[2];
  const int pieces = P.rank / 8;  // of eight numbers, at most two a lane
#pragma unroll
  for (int i = 0; i < 2; ++i) v[i] = lane + 32 * i < pieces ? src[lane + 32 * i] : make_uint4(0, 0, 0, 0);
  const uint32_t kp = reinterpret_cast<const uint32_t*>(src + pieces)[lane];

  // the first 16 heads' queries are asked for here: eight lanes a head, four pairs a lane (those of more heads behind the norm)
  const T* q = static_cast<const T*>(P.q) + t * P.q_token + (lane & 7) * 8;
  uint4 early[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int h = (lane >> 3) + 4 * i;
    if (h < P.heads) early[i] = *reinterpret_cast<const uint4*>(q + h * P.q_head);
  }

  const double turns = static_cast<double>(P.positions[t]) * static_cast<double>(P.inv_freq[lane]) * 0.15915494309189535;  // 1 / 2 pi
  float sn, cs;
  sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &sn, &cs);
  sn *= P.rope_scale;
  cs *= P.rope_scale;

  long long slot = P.slots[t];
  if (slot < -1 || slot >= static_cast<long long>(P.n_pages) * P.page_size) {
    if (lane == 0) atomicExch(P.err, GEMQ_LATENT_BAD_SLOT);
    slot = -1;
  }
  uint4* row = reinterpret_cast<uint4*>(static_cast<T*>(P.rows) + static_cast<long long>(t) * width);
  uint4* stored = slot < 0 ? nullptr
                           : reinterpret_cast<uint4*>(static_cast<T*>(P.cache) + slot / P.page_size * P.page_stride + slot % P.page_size * width);

  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t* e = reinterpret_cast<const uint32_t*>(&v[i]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = Pair<T>::f(e[k]);
      ss = fmaf(f.x, f.x, fmaf(f.y, f.y, ss));
    }
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, x);
  const float r = rsqrtf(ss / P.rank + P.eps);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = lane + 32 * i;
    if (at >= pieces) continue;
    const uint4 wv = w[at];
    uint4 o;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = Pair<T>::f(reinterpret_cast<const uint32_t*>(&v[i])[k]);
      const float2 g = Pair<T>::f(reinterpret_cast<const uint32_t*>(&wv)[k]);
      reinterpret_cast<uint32_t*>(&o)[k] = Pair<T>::r(f.x * r * g.x, f.y * r * g.y);
    }
    row[at] = o;
    if (stored) stored[at] = o;
  }
  {
    const float2 f = Pair<T>::f(kp);
    const uint32_t o = Pair<T>::r(f.x * cs - f.y * sn, f.x * sn + f.y * cs);
    reinterpret_cast<uint32_t*>(row + pieces)[lane] = o;
    if (stored) reinterpret_cast<uint32_t*>(stored + pieces)[lane] = o;
  }
  float c4[4], s4[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    c4[k] = __shfl_sync(0xffffffffu, cs, (lane & 7) * 4 + k);
    s4[k] = __shfl_sync(0xffffffffu, sn, (lane & 7) * 4 + k);
  }
  T* qo = static_cast<T*>(P.q_out) + static_cast<long long>(t) * P.heads * kRope + (lane & 7) * 8;
  auto turn = [&](int h, const uint4& x) {
    uint4 o;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = Pair<T>::f(reinterpret_cast<const uint32_t*>(&x)[k]);
      reinterpret_cast<uint32_t*>(&o)[k] = Pair<T>::r(f.x * c4[k] - f.y * s4[k], f.x * s4[k] + f.y * c4[k]);
    }
    *reinterpret_cast<uint4*>(qo + h * kRope) = o;
  };
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int h = (lane >> 3) + 4 * i;
    if (h < P.heads) turn(h, early[i]);
  }
#pragma unroll 4
  for (int h = (lane >> 3) + 16; h < P.heads; h += 4) turn(h, *reinterpret_cast<const uint4*>(q + h * P.q_head));
}

// A CTA copies 16 KB of a page of one layer at a time, four 16-byte loads a thread in flight.
constexpr int kCopyThreads = 256, kCopyUnroll = 4, kCopyPiece = kCopyThreads * kCopyUnroll;  // in 16 bytes

struct CopyArgs {
  uint4* cache;
  long long layer_stride, page_stride;  // in 16 bytes
  int layers, n_pages;
  long long page_len;  // in 16 bytes
  const long long* src;
  const long long* dst;
  int copies;
  int* err;
};

__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const CopyArgs P) {
  const long long pieces = (P.page_len + kCopyPiece - 1) / kCopyPiece, total = pieces * P.copies * P.layers;
  for (long long i = blockIdx.x; i < total; i += gridDim.x) {
    const long long piece = i % pieces, rest = i / pieces;
    const int c = static_cast<int>(rest % P.copies);
    const long long layer = rest / P.copies;
    const long long a = P.src[c], b = P.dst[c];
    if (a < 0 || a >= P.n_pages || b < 0 || b >= P.n_pages) {
      if (threadIdx.x == 0) atomicExch(P.err, GEMQ_LATENT_BAD_PAGE);
      continue;
    }
    if (a == b) continue;
    uint4* base = P.cache + layer * P.layer_stride;
    const uint4* from = base + a * P.page_stride;
    uint4* to = base + b * P.page_stride;
    uint4 v[kCopyUnroll];
    const long long at = piece * kCopyPiece + threadIdx.x;
#pragma unroll
    for (int k = 0; k < kCopyUnroll; ++k)
      if (at + k * kCopyThreads < P.page_len) v[k] = __ldcs(from + at + k * kCopyThreads);
#pragma unroll
    for (int k = 0; k < kCopyUnroll; ++k)
      if (at + k * kCopyThreads < P.page_len) __stcs(to + at + k * kCopyThreads, v[k]);
  }
}

__global__ void take_error_kernel(int* err, int* code) { *code = atomicExch(err, 0); }

}  // namespace
}  // namespace gemq

using namespace gemq;

extern "C" int gemq_latent_take_error(int32_t* err, int32_t* code, gemq_stream_t stream) {
  if (!err || !code) return GEMQ_ERR_BAD_ARG;
  take_error_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(err, code);
  return launch_status();
}

extern "C" int gemq_latent_append(const void* kv, int64_t kv_stride, const void* q_rope, int64_t q_token_stride, int64_t q_head_stride,
                                  const void* norm_weight, float eps, const float* inv_freq, float rope_scale, const int64_t* positions,
                                  const int64_t* slots, void* cache, int64_t page_stride, int n_pages, int page_size, void* rows,
                                  void* q_out, int tokens, int heads, int rank, int is_bf16, int32_t* err, gemq_stream_t stream) {
  if (tokens == 0) return GEMQ_OK;
  if (!kv || !norm_weight || !inv_freq || !positions || !slots || !cache || !rows || !err || (heads && (!q_rope || !q_out)) || tokens < 0 ||
      heads < 0 || n_pages <= 0 || page_size <= 0)
    return GEMQ_ERR_BAD_ARG;
  if (!rank_ok(rank) || tokens > (1 << 30)) return GEMQ_ERR_BAD_SHAPE;
  for (const void* p : {kv, q_rope, norm_weight, static_cast<const void*>(cache), static_cast<const void*>(rows), static_cast<const void*>(q_out)})
    if (p && !aligned16(p)) return GEMQ_ERR_ALIGN;
  if ((kv_stride | q_token_stride | q_head_stride | page_stride) & 7) return GEMQ_ERR_ALIGN;
  const AppendArgs P = {kv, kv_stride, q_rope, q_token_stride, q_head_stride, norm_weight, eps, inv_freq, rope_scale,
                        reinterpret_cast<const long long*>(positions), reinterpret_cast<const long long*>(slots), cache, page_stride,
                        n_pages, page_size, rows, q_out, tokens, heads, rank, err};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cdiv(tokens, kAppendWarps));
  cfg.blockDim = dim3(32 * kAppendWarps);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = is_bf16 ? cudaLaunchKernelEx(&cfg, latent_append_kernel<__nv_bfloat16>, P)
                                : cudaLaunchKernelEx(&cfg, latent_append_kernel<__half>, P);
  return e == cudaSuccess ? GEMQ_OK : GEMQ_ERR_LAUNCH;
}

extern "C" int gemq_copy_pages(void* cache, int64_t layer_stride, int64_t page_stride, int layers, int n_pages, int64_t page_bytes,
                               const int64_t* src, const int64_t* dst, int copies, int32_t* err, gemq_stream_t stream) {
  if (copies == 0) return GEMQ_OK;
  if (!cache || !src || !dst || !err || copies < 0 || layers <= 0 || n_pages <= 0 || page_bytes <= 0) return GEMQ_ERR_BAD_ARG;
  if (!aligned16(cache) || ((layer_stride | page_stride | page_bytes) & 15)) return GEMQ_ERR_ALIGN;
  const CopyArgs P = {static_cast<uint4*>(cache), layer_stride / 16, page_stride / 16, layers, n_pages, page_bytes / 16,
                      reinterpret_cast<const long long*>(src), reinterpret_cast<const long long*>(dst), copies, err};
  const int sms = sm_count();
  if (sms <= 0) return GEMQ_ERR_LAUNCH;
  const long long pieces = (P.page_len + kCopyPiece - 1) / kCopyPiece * copies * layers, most = 8ll * sms;
  copy_pages_kernel<<<static_cast<int>(pieces < most ? pieces : most), kCopyThreads, 0, static_cast<cudaStream_t>(stream)>>>(P);
  return launch_status();
}
