// Attention of whole prompts over expanded keys and values, head size 128 + 64 and 128.
//
//   s[i, j] = scale * (q_nope[i] . k_nope[j] + q_rope[i] . k_rope[j]),   out[i] = sum_j softmax(s)[i, j] v[j],   j <= i + keys - queries
//
// What bounds it: 640 operations for each visible (query, key) of a head, against 16 to 32 exponentials a clock of a multiprocessor for one
// each: the tensor cores, with the exponentials close behind (a 128 x 128 tile: 1280 cycles of MMAs, 1024 of ex2).
//
// A CTA has 256 queries of one head as two tiles of 128, each with a warp group for its softmax (a thread has a row), over the same
// tiles of 128 keys: while the exponentials of one tile are formed the MMAs of the other run.  Scores, and in their place the weights
// (16 bits), and the sums stay in tensor memory: 2 x (128 + 128) columns, all of it.
//   warp 0      TMA: queries once, then two places of keys (48 KB) and one of values (32 KB)
//   warps 1, 2  MMAs of either tile: O of keys j, then S of keys j + 1 in its weights' place.  (One warp for both left the tensor cores idle for
//               250 to 600 cycles between any two products.)
//   warp 3      a second pass only, see below
//   warps 4-7, 8-11   softmax of either tile, results
// The reference of a row's weights moves only when its own scores exceed it by 2^8; then its sums are corrected in tensor memory.  Weights are
// rounded to the type for the second product, their sums are not (the logarithm of the sum keeps all of its bits).
//
// What a query must not see is given a weight of 0.  If such a row of v holds an infinity or a NaN the product still is NaN: a block with a
// result that is not finite is computed once more, and warp 3 sets to zero, in the tiles that not all of its queries see whole, what
// is hidden from all and what is not finite; a query that sees one of the latter gets a NaN for its weight.  Every wait is bounded.
//
// Measured: 8192 queries x 16 heads, 344 GFLOP: 336 us in a loop of calls (1.02 PFLOP/s at 1.7 GHz, the power limit), 284 in short bursts
// (1.21); a round of both tiles 3550 to 3900 cycles of 2560 of MMAs.  Tried: values in a ring of their own depth with the keys (the tiles fall into
// step and share the exponentials' units: 5100 to 5500 cycles; made to take turns: 3700 and the same time).
#include "latent.cuh"

namespace gemq {

// tma.cu
bool tensor_map_heads(CUtensorMap* out, const void* base, int width, int heads, long long head_stride, long long rows, long long row_stride,
                      int box_rows);

namespace latent {
namespace {

constexpr int kNope = 128, kValue = 128;
constexpr int kRows = 128;                 // of a tile: queries, and keys
constexpr int kBlock = kRows * 128;        // bytes of 128 rows x 64 numbers
constexpr int kThreads = 384, kSoftWarp = 4;

constexpr int kAllKeys = 0x40000000;
struct Item { int row0, rows, k0, keys, first; };  // query rows, key rows; what the first query sees (none if not above 0), or kAllKeys

struct Smem {
  alignas(1024) unsigned char q[2][3][kBlock];
  unsigned char k[2][3][kBlock];
  unsigned char v[2][kBlock];
  alignas(8) unsigned long long q_full[2], k_full[2], k_free[2], v_full, v_free, v_clean, s_full[2], p_full[2][2], o_full[2];
  uint32_t poison[4];
  Item item;
  uint32_t tmem_base;
  int abort;
};
static_assert(sizeof(Smem) <= 232448, "more shared memory than a CTA has");

struct Args {
  CUtensorMap q_nope, q_rope, kv, k_rope;
  gemq_latent_prefill_t a;
  float scale;  // times log2 e
};

// Two 32-bit numbers in a register pair: one instruction for both.
__device__ __forceinline__ unsigned long long both(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void fma2(float& x, float& y, unsigned long long m, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(both(x, y)), "l"(m), "l"(c));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(r));
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Stays where it stands among the stores and hand-overs: those of the second half are not to be formed ahead of the first half's.
__device__ __forceinline__ float exp2_here(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A wait of the MMA warp, which stands between two products: it looks again and again (about a second in all).
__device__ __forceinline__ void spin_for(unsigned long long* bar, uint32_t parity, int* abort, int* err) {
  for (int i = 0; i < (1 << 25); ++i) {
    if (mbar_test_wait(bar, parity)) return;
    if ((i & 0xfff) == 0xfff && *reinterpret_cast<volatile int*>(abort)) return;
  }
  *reinterpret_cast<volatile int*>(abort) = 1;
  atomicExch(err, GEMQ_LATENT_WAIT);
}

// Whether any thread of the CTA says so; all its threads come here.
__device__ __forceinline__ bool any_in_cta(bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 0, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(mine))
      : "memory");
  return any != 0;
}

__device__ __forceinline__ int within(int v, int most) { return min(max(v, 0), most); }

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) latent_prefill_kernel(const __grid_constant__ Args P) {
  constexpr float kOffset = Pair<T>::kBf16 ? 0.f : 7.f;  // fp16 weights are 2^7 times as large: those above 2^-21 keep all their bits
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  Smem& S = *reinterpret_cast<Smem*>(smem_raw);
  const gemq_latent_prefill_t& A = P.a;
  int* const err = A.err;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = blockIdx.x % A.heads, at = blockIdx.x / A.heads;  // at: blocks of 256 queries, the last of a sequence first
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S.q_full[i], 1);
      mbar_init(&S.k_full[i], 1);
      mbar_init(&S.k_free[i], 2);
      mbar_init(&S.s_full[i], 1);
      mbar_init(&S.p_full[i][0], 4);
      mbar_init(&S.p_full[i][1], 4);
      mbar_init(&S.o_full[i], 1);
    }
    mbar_init(&S.v_full, 1);
    mbar_init(&S.v_free, 2);
    mbar_init(&S.v_clean, 1);
    S.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&S.tmem_base, 512);
  if (warp == 2 && lane < 4) prefetch_map(lane == 0 ? &P.q_nope : lane == 1 ? &P.q_rope : lane == 2 ? &P.kv : &P.k_rope);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == 0) {
    // The block's sequence.  Behind the last there is one more, of the query rows that no sequence has.  n rows behind row q0 fill
    // at most (q0 + n) / 256 - q0 / 256 + 1 blocks, so 32 sequences from b0 have the blocks from cu_q[b0] / 256 + b0 to that of the
    // next 32, some of them without work: found by comparing 32 starts at a time.  2048 sequences of 16 rows x 16 heads take 1.59 ms;
    // with every sequence's blocks counted on the way it was 2.93.
    auto first = [&](int b) { return within(A.cu_q[b], A.q_rows) / (2 * kRows) + b; };
    int group = 0;
    for (int groups = A.batch / 32 + 1; groups > 1;) {
      const int step = cdiv(groups, 32), mine = lane * step;
      const unsigned below = __ballot_sync(0xffffffffu, mine < groups && first(32 * (group + mine)) <= at);
      const int skip = below ? (31 - __clz(below)) * step : 0;
      group += skip;
      groups = min(step, groups - skip);
    }
    const int b = 32 * group + lane;
    int q0 = 0, n = 0, k0 = 0, keys = 0;
    if (b <= A.batch) {
      q0 = within(A.cu_q[b], A.q_rows);
      n = (b < A.batch ? within(A.cu_q[b + 1], A.q_rows) : A.q_rows) - q0;
      k0 = within(A.cu_k[b], A.k_rows);
      keys = b < A.batch ? max(within(A.cu_k[b + 1], A.k_rows) - k0, 0) : 0;
    }
    const int nth = at - (__shfl_sync(0xffffffffu, q0, 0) / (2 * kRows) + 32 * group);
    // Those of many keys first (of 32 sequences at a time): what begins last should be short.
    const int mine = n > 0 ? cdiv(n, 2 * kRows) : 0;
    int upto = mine;
#pragma unroll 4
    for (int d = 1; d < 32; ++d) {
      const int who = (lane + d) & 31, k = __shfl_sync(0xffffffffu, keys, who), m = __shfl_sync(0xffffffffu, mine, who);
      if (k > keys || (k == keys && who < lane)) upto += m;
    }
    const bool hit = nth >= upto - mine && nth < upto;
    if (hit) {
      const int r0 = (upto - 1 - nth) * 2 * kRows;
      S.item = {q0 + r0, min(n - r0, 2 * kRows), k0, keys, A.causal ? r0 + 1 + keys - n : kAllKeys};
    }
    if (!__any_sync(0xffffffffu, hit) && lane == 0) S.item = {0, 0, 0, 0, 0};
  }
  if (blockIdx.x == 0 && threadIdx.x == 32 * 11 && !(offsets_ok(A.cu_q, A.batch, A.q_rows) && offsets_ok(A.cu_k, A.batch, A.k_rows)))
    atomicExch(err, GEMQ_LATENT_BAD_LENGTH);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  // Only now: a CTA of the next kernel must not take this SM's tensor memory first.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = S.tmem_base;
  const int row0 = uniform(S.item.row0), rows = uniform(S.item.rows), k0 = uniform(S.item.k0), keys = uniform(S.item.keys), first = uniform(S.item.first);
  // query i of the block sees keys 0 .. limit(i) - 1
  auto limit_of = [&](int i) { return first == kAllKeys ? keys : min(first + i, keys); };
  int tiles[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int n = min(rows - t * kRows, kRows);
    tiles[t] = n > 0 ? cdiv(max(limit_of(t * kRows + n - 1), 0), kRows) : 0;
  }
  const int most = max(tiles[0], tiles[1]);

  // A second pass goes on with the barriers: how often each was completed in the first.
  const int k_uses[2] = {(most + 1) >> 1, most >> 1};
  const int least_of_all = max(limit_of(0), 0), most_of_all = max(limit_of(max(rows, 1) - 1), 0);
  if (warp < kSoftWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 0) {
      const uint32_t q = smem_u32(S.q[0][0]), k = smem_u32(S.k[0][0]), v = smem_u32(S.v[0]);
      auto load_q = [&](int t) {
        const uint32_t bar = smem_u32(&S.q_full[t]), dst = q + t * 3 * kBlock;
        const int r = row0 + t * kRows;
        if (elect_lane()) {
          mbar_expect_at(bar, 3 * kBlock);
          tma_load_3d_at(dst, &P.q_nope, 0, head, r, bar);
          tma_load_3d_at(dst + kBlock, &P.q_nope, 64, head, r, bar);
          tma_load_3d_at(dst + 2 * kBlock, &P.q_rope, 0, head, r, bar);
        }
        __syncwarp();
      };
      for (int pass = 0;; ++pass) {
        auto load_k = [&](int j) {
          const int s = j & 1;
          wait_for(&S.k_free[s], ((pass * k_uses[s] + (j >> 1)) & 1) ^ 1, &S.abort, err);
          const uint32_t bar = smem_u32(&S.k_full[s]), dst = k + s * 3 * kBlock;
          const int r = k0 + j * kRows;
          if (elect_lane()) {
            mbar_expect_at(bar, 3 * kBlock);
            tma_load_3d_at(dst, &P.kv, 0, head, r, bar);
            tma_load_3d_at(dst + kBlock, &P.kv, 64, head, r, bar);
            tma_load_3d_at(dst + 2 * kBlock, &P.k_rope, 0, 0, r, bar);
          }
          __syncwarp();
        };
        if (most > 0) {
          if (pass == 0 && tiles[0] > 0) load_q(0);
          load_k(0);
          if (pass == 0 && tiles[1] > 0) load_q(1);
          for (int j = 0; j < most; ++j) {
            if (j + 1 < most) load_k(j + 1);
            wait_for(&S.v_free, ((pass * most + j) & 1) ^ 1, &S.abort, err);
            const uint32_t bar = smem_u32(&S.v_full);
            if (elect_lane()) {
              mbar_expect_at(bar, 2 * kBlock);
              tma_load_3d_at(v, &P.kv, kNope, head, k0 + j * kRows, bar);
              tma_load_3d_at(v + kBlock, &P.kv, kNope + 64, head, k0 + j * kRows, bar);
            }
            __syncwarp();
          }
        }
        if (!any_in_cta(false) || pass == 1) break;
      }
      // The copies in flight end before the CTA does: the MMAs waited for all of them, unless a wait ran out.
      if (*reinterpret_cast<volatile int*>(&S.abort))
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    } else if (warp < 3) {
      const int t = warp - 1, mine = tiles[t];
      const uint32_t idesc_s = umma_idesc_f16(Pair<T>::kBf16, kRows, kRows), idesc_o = umma_idesc_f16(Pair<T>::kBf16, kRows, kValue) | kUmmaTransposeB;
      const uint64_t q = umma_desc_k_sw128(smem_u32(S.q[t][0])), k = umma_desc_k_sw128(smem_u32(S.k[0][0])),
                     v = umma_desc_mn_sw128(smem_u32(S.v[0]), kBlock);
      const uint32_t s_at = tmem + t * kRows, o_at = tmem + 2 * kRows + t * kValue;
      if (mine > 0) wait_for(&S.q_full[t], 0, &S.abort, err);
      for (int pass = 0;; ++pass) {
        // S of keys j; a place of keys, and that of the values, is free when both tiles are done with it or have no use for it
        auto scores = [&](int j) {
          const int s = j & 1;
          spin_for(&S.k_full[s], (pass * k_uses[s] + (j >> 1)) & 1, &S.abort, err);
          if (j < mine) {
            tc_fence_after_sync();
            const uint64_t b = k + s * (3 * kBlock >> 4);
            if (elect_lane()) {
#pragma unroll
              for (int i = 0; i < 12; ++i)
                umma_ss_f16(s_at, q + (i >> 2) * (kBlock >> 4) + (i & 3) * 2, b + (i >> 2) * (kBlock >> 4) + (i & 3) * 2, idesc_s, i != 0);
              umma_commit(&S.s_full[t]);
              umma_commit(&S.k_free[s]);
            }
          } else if (elect_lane()) {
            mbar_arrive(&S.k_free[s]);
          }
          __syncwarp();
        };
        if (most > 0) scores(0);
        for (int j = 0; j < most; ++j) {
          if (j < mine) {  // by the halves of the weights: the first is multiplied while the second is formed
            spin_for(&S.p_full[t][0], (pass * mine + j) & 1, &S.abort, err);
            spin_for(pass ? &S.v_clean : &S.v_full, j & 1, &S.abort, err);
            tc_fence_after_sync();
            if (elect_lane()) {
#pragma unroll
              for (int i = 0; i < kRows / 32; ++i) umma_ts_f16_one(o_at, s_at + i * 8, v + i * (2048 >> 4), idesc_o, j != 0 || i != 0);
            }
            __syncwarp();
            spin_for(&S.p_full[t][1], (pass * mine + j) & 1, &S.abort, err);
            tc_fence_after_sync();
            if (elect_lane()) {
#pragma unroll
              for (int i = kRows / 32; i < kRows / 16; ++i) umma_ts_f16_one(o_at, s_at + i * 8, v + i * (2048 >> 4), idesc_o, 1);
              umma_commit(&S.v_free);
              if (j == mine - 1) umma_commit(&S.o_full[t]);
            }
          } else {
            spin_for(&S.v_full, (pass * most + j) & 1, &S.abort, err);
            if (elect_lane()) mbar_arrive(&S.v_free);
          }
          __syncwarp();
          if (j + 1 < most) scores(j + 1);
        }
        if (!any_in_cta(false) || pass == 1) break;
      }
    } else if (any_in_cta(false)) {
      for (int j = 0; j < most; ++j) {
        wait_for(&S.v_full, (most + j) & 1, &S.abort, err);
        uint32_t poison[4] = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; ++w)
          for (int r = max(least_of_all - j * kRows - 32 * w, 0); r < 32; ++r) {
            uint2* at = reinterpret_cast<uint2*>(S.v[lane >> 4] + (32 * w + r) * 128) + (lane & 15);
            bool wipe = j * kRows + 32 * w + r >= most_of_all;
            if (!wipe) {
              const uint2 x = *at;
              wipe = __any_sync(0xffffffffu, has_nonfinite<T>(x.x) || has_nonfinite<T>(x.y));
              if (wipe) poison[w] |= 1u << r;
            }
            if (wipe) *at = make_uint2(0, 0);
          }
        if (lane < 4) S.poison[lane] = lane == 0 ? poison[0] : lane == 1 ? poison[1] : lane == 2 ? poison[2] : poison[3];
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.v_clean);
      }
      any_in_cta(false);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int t = (warp - kSoftWarp) >> 2, quad = warp & 3, i = t * kRows + 32 * quad + lane;
    const uint32_t lanes = static_cast<uint32_t>(32 * quad) << 16, s = tmem + lanes + t * kRows, o = tmem + lanes + 2 * kRows + t * kValue;
    const int limit = limit_of(i), least = limit_of(t * kRows + 32 * quad);
    for (int pass = 0;; ++pass) {
      float ref = 0.f, sum = 0.f;
      bool none = true;
      for (int j = 0; j < tiles[t]; ++j) {
        wait_for(&S.s_full[t], (pass * tiles[t] + j) & 1, &S.abort, err);
        tc_fence_after_sync();
        uint32_t raw[kRows];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_load32(s + 32 * c, raw + 32 * c);
        tmem_loaded(raw);
        float* v = reinterpret_cast<float*>(raw);
        {
          const unsigned long long m = both(P.scale, P.scale), c2 = both(-ref, -ref);
#pragma unroll
          for (int c = 0; c < kRows; c += 2) fma2(v[c], v[c + 1], m, c2);
        }
        if (pass) {
          wait_for(&S.v_clean, j & 1, &S.abort, err);
#pragma unroll
          for (int c = 0; c < kRows; ++c)
            if (S.poison[c >> 5] >> (c & 31) & 1) v[c] = __int_as_float(0x7fc00000);
        }
        if ((j + 1) * kRows > least) {
          const int here = limit - j * kRows;
#pragma unroll
          for (int c = 0; c < kRows; ++c)
            if (c >= here) v[c] = -INFINITY;
        }
        float most4[4] = {v[0], v[1], v[2], v[3]};  // four chains
#pragma unroll
        for (int c = 4; c + 1 < kRows; c += 2) most4[(c >> 1) & 3] = max3(most4[(c >> 1) & 3], v[c], v[c + 1]);
        const float top = fmaxf(fmaxf(most4[0], most4[1]), fmaxf(most4[2], most4[3]));
        if (__any_sync(0xffffffffu, none ? top > -INFINITY : top > kOffset + 8.f)) {
          // a row's own scores decide: its neighbours in the warp, and what those see, are to change none of its bits
          const float up = none || top > kOffset + 8.f ? top - kOffset : 0.f, by = up == -INFINITY ? 0.f : up;
          const float f = none ? 1.f : exp2_fast(-by);
          none = none && up == -INFINITY;
          ref += by;
          sum *= f;
#pragma unroll
          for (int c = 0; c < kRows; ++c) v[c] -= by;
          if (j > 0) {
#pragma unroll
            for (int c = 0; c < kValue; c += 16) {
              uint32_t x[16];
              tmem_load16(o + c, x);
              tmem_loaded(x);
#pragma unroll
              for (int y = 0; y < 16; ++y) x[y] = __float_as_uint(__uint_as_float(x[y]) * f);
              tmem_store16(o + c, x);
            }
          }
        }
        unsigned long long part[2] = {0, 0};  // sums of the even and the odd keys, twice
#pragma unroll
        for (int c = 0; c < kRows; c += 32) {
          uint32_t w[16];
#pragma unroll
          for (int y = 0; y < 16; ++y) {
            const float a = exp2_here(v[c + 2 * y]), b = exp2_here(v[c + 2 * y + 1]);
            part[y & 1] = add2(part[y & 1], both(a, b));
            w[y] = Pair<T>::r(a, b);
          }
          tmem_store16(s + c / 2, w);
          if (c & 32) {  // a half is there
            tmem_stored();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.p_full[t][c >> 6]);
          }
        }
        float even, odd;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(even), "=f"(odd) : "l"(add2(part[0], part[1])));
        sum += even + odd;
      }
      bool bad = false;
      if (t * kRows + 32 * quad < rows) {  // the warp has rows
        const bool on = i < rows;
        const long long out = static_cast<long long>(row0 + i) * A.heads + head;
        T* const to = static_cast<T*>(A.out) + out * kValue;
        if (tiles[t] > 0) {
          wait_for(&S.o_full[t], pass, &S.abort, err);
          tc_fence_after_sync();
          const float f = limit > 0 ? 1.f / sum : 0.f;
          float check = 0.f;
#pragma unroll 1
          for (int c = 0; c < kValue; c += 64) {
            uint32_t x[64];
            tmem_load32(o + c, x);
            tmem_load32(o + c + 32, x + 32);
            tmem_loaded(x);
#pragma unroll
            for (int y = 0; y < 64; y += 8) {
              uint32_t w[4];
#pragma unroll
              for (int z = 0; z < 4; ++z) {
                const float a = __uint_as_float(x[y + 2 * z]) * f, b = __uint_as_float(x[y + 2 * z + 1]) * f;
                check += (a - a) + (b - b);  // 0, or NaN
                w[z] = Pair<T>::r(a, b);
              }
              if (on) *reinterpret_cast<uint4*>(to + c + y) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          bad = on && check != 0.f;
        } else if (on) {
          for (int c = 0; c < kValue; c += 8) *reinterpret_cast<uint4*>(to + c) = make_uint4(0, 0, 0, 0);
        }
        if (on) A.lse[out] = limit > 0 && tiles[t] > 0 ? (ref + log2f(sum)) * kLn2 : -INFINITY;
      }
      tc_fence_before_sync();
      // where all rows see all of the tiles a second pass would find the same
      if (!any_in_cta(bad && least_of_all < most * kRows) || pass == 1) break;
      tc_fence_after_sync();
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T>
int launch(const Args& P, unsigned ctas, cudaStream_t st) {
  static bool set[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return GEMQ_ERR_LAUNCH;
  if (!set[dev]) {
    if (cudaFuncSetAttribute(latent_prefill_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Smem)) != cudaSuccess) return GEMQ_ERR_LAUNCH;
    set[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, latent_prefill_kernel<T>, P) == cudaSuccess ? GEMQ_OK : GEMQ_ERR_LAUNCH;
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
  const long long blocks = (A->q_rows / (2ll * kRows) + A->batch + 1) * A->heads;
  if (blocks > 0x7fffffff || A->q_rows > 0x3fffffff || A->k_rows > 0x3fffffff) return GEMQ_ERR_BAD_SHAPE;
  for (const void* p : {A->q_nope, A->q_rope, A->kv, A->k_rope, static_cast<const void*>(A->out)})
    if (p && !aligned16(p)) return GEMQ_ERR_ALIGN;
  if ((A->q_nope_stride[0] | A->q_nope_stride[1] | A->q_rope_stride[0] | A->q_rope_stride[1] | A->kv_stride[0] | A->kv_stride[1] |
       A->k_rope_stride) & 7)
    return GEMQ_ERR_ALIGN;
  // a tiled copy has no stride of 0
  if (A->q_rows > 1 && (A->q_nope_stride[0] <= 0 || A->q_rope_stride[0] <= 0)) return GEMQ_ERR_BAD_SHAPE;
  if (A->k_rows > 1 && (A->kv_stride[0] <= 0 || A->k_rope_stride <= 0)) return GEMQ_ERR_BAD_SHAPE;
  if (A->heads > 1 && (A->q_nope_stride[1] <= 0 || A->q_rope_stride[1] <= 0 || (A->k_rows && A->kv_stride[1] <= 0))) return GEMQ_ERR_BAD_SHAPE;
  Args P;
  P.a = *A;
  P.scale = A->scale * kLog2e;
  // without keys no tile is loaded: any valid map does
  const void* kv = A->k_rows ? A->kv : A->q_nope;
  const void* kr = A->k_rows ? A->k_rope : A->q_rope;
  const long long kn = A->k_rows ? A->k_rows : 1;
  if (!tensor_map_heads(&P.q_nope, A->q_nope, kNope, A->heads, A->q_nope_stride[1], A->q_rows, A->q_nope_stride[0], kRows) ||
      !tensor_map_heads(&P.q_rope, A->q_rope, kRope, A->heads, A->q_rope_stride[1], A->q_rows, A->q_rope_stride[0], kRows) ||
      !tensor_map_heads(&P.kv, kv, A->k_rows ? kNope + kValue : 64, A->k_rows ? A->heads : 1, A->kv_stride[1], kn, A->kv_stride[0], kRows) ||
      !tensor_map_heads(&P.k_rope, kr, kRope, 1, 0, kn, A->k_rope_stride, kRows))
    return GEMQ_ERR_LAUNCH;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return A->is_bf16 ? launch<__nv_bfloat16>(P, static_cast<unsigned>(blocks), st) : launch<__half>(P, static_cast<unsigned>(blocks), st);
}
