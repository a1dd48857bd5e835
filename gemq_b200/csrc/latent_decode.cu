// Attention of decoded tokens over a paged latent cache, for any batch of sequences, with or without shared prefixes.
//
//   s[r, t] = scale * (q_latent[r] . c[t] + q_rope[r] . k[t]),   out[r] = sum_t softmax(s)[r, t] c[t],   r = (sequence, step, head)
//
// What bounds it.  A cached row is rank + 64 numbers (1152 bytes at rank 512) that all heads of a sequence use: 16 rows of queries make
// 30 operations of a byte, so a batch of sequences is bound by HBM; a prefix that 64 sequences share, 1024 rows, by the tensor cores.
//
// Both products have the cached tile as their wide operand, straight as TMA brought it:
//   S^T [64 positions, N rows] = C [64, rank + 64] * Q^T        M = 64, both operands K-major
//   O^T [rank, N rows]        += C^T [rank, 64] * P^T           M = 128, the tile read along M; P^T K-major, written by the softmax warps
// so that a row tile of N = 16, 32 or 64 query rows costs what it has.  (With the queries as the M operand 16 rows would take an eighth
// of an MMA's 128, and 512 columns of results all of the tensor memory.)
//
// Persistent, one CTA an SM.  All row tiles of all sequences (and groups) times their 64-row tiles of the cache are one list, cut
// into equal shares; a CTA's share is a run of pieces (row tile, range of tiles).  A piece that is all of a row tile is finished in
// place, others leave their sums (fp32), maximum and sum of weights to the second kernel, which joins them in order of position.
//   warp 0     TMA: a ring of blocks of 64 rows x 64 numbers, latent ones in pairs (2.75 tiles deep at N = 16), rope ones apart
//   warp 1     MMA: S of tile k, then O of tile k - 1
//   warps 2-3  the queries of the next piece into shared memory
//   warps 4-7  softmax (a thread has two positions x N / 4 rows), O's correction, results
// The maximum that the weights refer to moves only when a row's scores exceed it by 2^8: O is corrected in tensor memory a few times per
// sequence.  Rows behind what is seen are zeroed in shared memory before they are multiplied by weights of 0: what lies there may be NaN.
// Every wait is bounded.
#include "latent.cuh"
#include "ptx.cuh"

namespace gemq {

// tma.cu
bool tensor_map_pages(CUtensorMap* out, const void* base, int blocks, int page_size, long long page_stride, int pages, int box_rows,
                      int box_blocks);

namespace latent {
namespace {

constexpr int kTile = 64;            // positions of a tile
constexpr int kBlock = kTile * 128;  // bytes of 64 positions x 64 numbers
constexpr int kThreads = 256;
constexpr int kSoftWarp = 4;
constexpr int kSlots = 16;           // tiles in flight that are told apart; the ring holds 11 at most (rank 128)

// Blocks of the ring: what 227 KB hold beside the queries.
template <int N> struct Ring;
template <> struct Ring<16> { static constexpr int kLatent = 22, kRopes = 3; };
template <> struct Ring<32> { static constexpr int kLatent = 20, kRopes = 3; };
template <> struct Ring<64> { static constexpr int kLatent = 16, kRopes = 2; };

struct Start { int e, rt, t, left, rto; };

template <int N>
struct Smem {
  static constexpr int kLatent = Ring<N>::kLatent, kRopes = Ring<N>::kRopes;
  alignas(1024) unsigned char ring[kLatent][kBlock];
  unsigned char rope[kRopes][kBlock];
  unsigned char q[9][N * 128];
  unsigned char p[N * 128];
  float wmax[2][4][N];
  float fac[N];
  alignas(8) unsigned long long full[kLatent / 2], rope_full[kRopes];
  unsigned long long done[kSlots], told[kSlots];  // the tile's MMAs are complete; its pages are known
  unsigned long long s_full[2], s_free[2], p_full, q_full, q_free, o_full, o_free;
  int bad[kSlots];  // of the tile's four quarters: on a page outside the cache
  int sums[kThreads / 32][2];
  Start start;
  uint32_t tmem_base;
  int abort;
};

struct Args {
  CUtensorMap latent_map, rope_map;
  gemq_latent_decode_t a;
  int* ctl;          // [0] total tiles, [1] CTAs that have some, then per entry: first tile, first row tile
  float* part_o;     // [slots][N][rank]
  float2* part_ml;   // [slots][N]: reference of the weights (in powers of two) and their sum
  int slots;
  float scale;       // times log2 e
  int box_blocks;    // latent blocks of a TMA box: 2, or 1 where pages are shorter than a tile
};

// ---- the list of work -----------------------------------------------------------------------------
__device__ __forceinline__ int start_of(const gemq_latent_decode_t& A, int g) {  // within the batch, whatever the device has
  return g <= 0 ? 0 : g >= A.groups ? A.batch : min(max(A.starts[g], 0), A.batch);
}
struct Entry { int len, tiles, row0, rows; };  // positions, tiles of 64, first query row (of batch * steps * heads), query rows

__device__ __forceinline__ Entry entry_of(const gemq_latent_decode_t& A, int e) {
  const int per = A.steps * A.heads;
  Entry x;
  if (e < A.groups) {
    const int s0 = start_of(A, e), s1 = start_of(A, e + 1);
    x.row0 = s0 * per;
    x.rows = max(s1 - s0, 0) * per;
    x.len = clamp_length(A.prefix_lens[e], A.prefix_pitch, A.page_size, A.err);
  } else {
    const int b = e - A.groups;
    x.row0 = b * per;
    x.rows = per;
    x.len = clamp_length(A.lens[b], A.table_pitch, A.page_size, A.err);
  }
  x.tiles = cdiv(x.len, kTile);
  return x;
}
// The CTA that has a tile of the list: CTA c has tiles floor(c T / C) .. floor((c + 1) T / C) - 1.
__device__ __forceinline__ int cta_of(long long tile, long long total, int ctas) {
  return static_cast<int>(((tile + 1) * ctas - 1) / total);
}

struct Piece {
  Entry x;
  int e, t0, n;      // entry, first tile, tiles
  int row0, rows;    // first query row, query rows of the row tile
  int rt;            // row tile of the launch
  bool whole;        // all tiles of the row tile
};

template <int N>
struct Walk {
  const gemq_latent_decode_t& A;
  int e, rt, t, left, rto;
  Entry x;
  __device__ __forceinline__ Walk(const gemq_latent_decode_t& a, const Start& s) : A(a), e(s.e), rt(s.rt), t(s.t), left(s.left), rto(s.rto) {
    if (left > 0) x = entry_of(A, e);
  }
  __device__ __forceinline__ bool next(Piece& p) {
    if (left <= 0) return false;
    while (t >= x.tiles || rt * N >= x.rows) {
      if (x.tiles > 0 && (rt + 1) * N < x.rows) {
        ++rt;
        t = 0;
      } else {
        rto += cdiv(x.rows, N);
        rt = t = 0;
        if (++e >= A.groups + A.batch) { left = 0; return false; }
        x = entry_of(A, e);
      }
    }
    p.x = x;
    p.e = e;
    p.t0 = t;
    p.n = min(left, x.tiles - t);
    p.row0 = x.row0 + rt * N;
    p.rows = min(N, x.rows - rt * N);
    p.rt = rto + rt;
    p.whole = p.n == x.tiles;
    t += p.n;
    left -= p.n;
    return true;
  }
};

// What query row r sees of entry e's positions.
__device__ __forceinline__ int limit_of(const gemq_latent_decode_t& A, const Entry& x, bool prefix, int r) {
  const int per = A.steps * A.heads, b = r / per, hidden = A.steps - 1 - (r % per) / A.heads;
  if (!prefix) return x.len - hidden;
  return x.len - max(hidden - clamp_length(A.lens[b], A.table_pitch, A.page_size, A.err), 0);
}

// ---- waits ------------------------------------------------------------------------------------------
// A wait that runs out (about a second) is reported and ends all waits of the CTA.
__device__ __forceinline__ void wait_for(unsigned long long* bar, uint32_t parity, int* abort, int* err) {
  if (mbar_test_wait(bar, parity)) return;
  for (int i = 0; i < (1 << 16); ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(20000)
        : "memory");
    if (ok || *reinterpret_cast<volatile int*>(abort)) return;
  }
  *reinterpret_cast<volatile int*>(abort) = 1;
  atomicExch(err, GEMQ_LATENT_WAIT);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ bool has_nonfinite(uint4 v) {
  constexpr uint32_t kExp = Pair<T>::kBf16 ? 0x7f80u : 0x7c00u;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = reinterpret_cast<const uint32_t*>(&v)[i];
    bad |= (w & kExp) == kExp || ((w >> 16) & kExp) == kExp;
  }
  return bad;
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads, 1) latent_decode_kernel(const __grid_constant__ Args P) {
  constexpr int kLatent = Ring<N>::kLatent, kRopes = Ring<N>::kRopes;
  constexpr uint32_t kTmemCols = N == 16 ? 128 : N == 32 ? 256 : 512;
  constexpr uint32_t kTmemO = 2 * N;
  constexpr int kCols = N / 4;  // rows of queries that a softmax thread has
  constexpr float kOffset = Pair<T>::kBf16 ? 0.f : 7.f;  // fp16 weights are 2^7 times as large: those above 2^-21 keep all their bits
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  Smem<N>& S = *reinterpret_cast<Smem<N>*>(smem_raw);
  const gemq_latent_decode_t& A = P.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int blocks = A.rank / 64;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kLatent / 2; ++i) mbar_init(&S.full[i], 1);
    for (int i = 0; i < kRopes; ++i) mbar_init(&S.rope_full[i], 1);
    for (int i = 0; i < kSlots; ++i) { mbar_init(&S.done[i], 1); mbar_init(&S.told[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&S.s_full[i], 1); mbar_init(&S.s_free[i], 4); }
    mbar_init(&S.p_full, 4);
    mbar_init(&S.q_full, 2);
    mbar_init(&S.q_free, 1);
    mbar_init(&S.o_full, 1);
    mbar_init(&S.o_free, 4);
    S.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&S.tmem_base, kTmemCols);
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // Every CTA adds up the list: a thread has a run of entries.
  const int entries = A.groups + A.batch, run = cdiv(entries, kThreads);
  int tiles = 0, rts = 0;
  for (int k = 0; k < run; ++k) {
    const int e = static_cast<int>(threadIdx.x) * run + k;
    if (e >= entries) break;
    const Entry x = entry_of(A, e);
    const int n = cdiv(x.rows, N);
    tiles += n * x.tiles;
    rts += n;
  }
  int before = tiles, rts_before = rts;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, before, d), b = __shfl_up_sync(0xffffffffu, rts_before, d);
    if (lane >= d) { before += a; rts_before += b; }
  }
  if (lane == 31) { S.sums[warp][0] = before; S.sums[warp][1] = rts_before; }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  // Only now: a CTA of the next kernel must not take this SM's tensor memory first.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  before -= tiles;
  rts_before -= rts;
  int total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) { before += S.sums[w][0]; rts_before += S.sums[w][1]; }
    total += S.sums[w][0];
  }
  const int ctas = min(static_cast<int>(gridDim.x), total), c = blockIdx.x;
  const int first = c < ctas ? static_cast<int>(static_cast<long long>(c) * total / ctas) : 0;
  const int last = c < ctas ? static_cast<int>(static_cast<long long>(c + 1) * total / ctas) : 0;
  if (c == 0 && threadIdx.x == 0) {
    P.ctl[0] = total;
    P.ctl[1] = ctas;
    if (A.groups > 0 && !offsets_ok(A.starts, A.groups, A.batch, true)) atomicExch(A.err, GEMQ_LATENT_BAD_LENGTH);
  }
  if (c == 0 || (c < ctas && first >= before && first < before + tiles)) {
    int at = before, rto = rts_before;
    for (int k = 0; k < run; ++k) {
      const int e = static_cast<int>(threadIdx.x) * run + k;
      if (e >= entries) break;
      const Entry x = entry_of(A, e);
      const int n = cdiv(x.rows, N), all = n * x.tiles;
      if (c == 0) {
        P.ctl[2 + 2 * e] = at;
        P.ctl[3 + 2 * e] = rto;
      }
      if (c < ctas && first >= at && first < at + all) S.start = {e, (first - at) / x.tiles, (first - at) % x.tiles, last - first, rto};
      at += all;
      rto += n;
    }
  }
  __syncthreads();
  const uint32_t tmem = S.tmem_base;
  const Start start = c < ctas ? S.start : Start{0, 0, 0, 0, 0};
  int* const err = A.err;

  if (warp == 0) {
    Walk<N> walk(A, start);
    Piece p;
    int block = 0, freed = 0;      // latent blocks asked for so far; tiles known to be done
    uint32_t k = 0;
    const int per_tile = A.page_size < kTile ? kTile / A.page_size : 1, quarters = A.page_size < kTile ? A.page_size / 16 : 4;
    const int box_rows = min(A.page_size, kTile);
    while (walk.next(p)) {
      const bool prefix = p.e < A.groups;
      const int* table = prefix ? A.prefix_table + static_cast<long long>(p.e) * A.prefix_pitch
                                : A.table + static_cast<long long>(p.e - A.groups) * A.table_pitch;
      const int pages = (p.x.len + A.page_size - 1) / A.page_size;
      int base = -64, ids = 0;     // lane i has the id of page base + i
      for (int t = p.t0; t < p.t0 + p.n; ++t, ++k) {
        const int pg = A.page_size < kTile ? t * per_tile : t * kTile / A.page_size;
        const int here = min(per_tile, pages - pg);  // pages of the tile
        if (pg < base || pg + here > base + 32) {
          base = pg;
          ids = base + lane < pages ? table[base + lane] : 0;
        }
        const bool out = (ids < 0 || ids >= A.n_pages) && base + lane < pages;
        const uint32_t outs = __ballot_sync(0xffffffffu, out) >> (pg - base);
        int bad = 0;
        for (int i = 0; i < here; ++i)
          if ((outs >> i) & 1) bad |= ((1 << quarters) - 1) << (i * quarters);
        if (lane == 0) {
          S.bad[k % kSlots] = bad;
          mbar_arrive(&S.told[k % kSlots]);
          if (bad) atomicExch(err, GEMQ_LATENT_BAD_PAGE);
        }
        const int row = A.page_size < kTile ? 0 : t * kTile % A.page_size;
        const uint32_t bytes = here * box_rows * 128;
        // Block q of the ring was block q - kLatent, of tile (q - kLatent) / blocks.
        for (int d = 0; d <= blocks; d += 2) {
          const bool rope = d == blocks;
          const int need = rope ? static_cast<int>(k) - kRopes + 1 : (block + 1 - kLatent) / blocks + (block + 1 >= kLatent ? 1 : 0);
          for (; freed < need; ++freed) wait_for(&S.done[freed % kSlots], (freed / kSlots) & 1, &S.abort, err);
          unsigned char* dst = rope ? S.rope[k % kRopes] : S.ring[block % kLatent];
          unsigned long long* bar = rope ? &S.rope_full[k % kRopes] : &S.full[block % kLatent / 2];
          if (lane == 0) mbar_arrive_expect_tx(bar, rope ? bytes : 2 * bytes);
          __syncwarp();
          const int boxes = rope ? 1 : 2 / P.box_blocks;
          for (int i = 0; i < here; ++i) {
            const int id = __shfl_sync(0xffffffffu, out ? 0 : ids, pg - base + i);
            if (elect_lane()) {
              for (int j = 0; j < boxes; ++j)
                tma_load_4d(dst + j * kBlock + i * A.page_size * 128, rope ? &P.rope_map : &P.latent_map, 0, row, d + j, id, bar);
            }
            __syncwarp();
          }
          if (!rope) block += 2;
        }
      }
    }
    // The copies in flight end before the CTA does: the MMAs of the last tile waited for them, unless a wait ran out.
    if (*reinterpret_cast<volatile int*>(&S.abort))
      for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  } else if (warp == 1) {
    Walk<N> walk(A, start);
    Piece p;
    uint32_t k = 0, piece = 0;
    const uint32_t idesc_s = umma_idesc_f16(Pair<T>::kBf16, kTile, N), idesc_o = umma_idesc_f16(Pair<T>::kBf16, 128, N) | kUmmaTransposeA;
    const uint64_t q0 = umma_desc_k_sw128(smem_u32(S.q[0])), p0 = umma_desc_k_sw128(smem_u32(S.p));
    const uint32_t ring0 = smem_u32(S.ring[0]);
    // O of a tile: its place in the ring, 16-row steps, whether it is the piece's first and last
    int prev_block = -1, prev_steps = 0;
    bool prev_first = false, prev_last = false;
    uint32_t prev_k = 0, prev_piece = 0;
    auto values = [&]() {
      if (prev_first) wait_for(&S.o_free, (prev_piece & 1) ^ 1, &S.abort, err);
      wait_for(&S.p_full, prev_k & 1, &S.abort, err);
      tc_fence_after_sync();
      if (elect_lane()) {
        int at = prev_block % kLatent;
        for (int m = 0; m < blocks / 2; ++m) {
          const uint64_t a = umma_desc_mn_sw128(ring0 + at * kBlock, kBlock);
          for (int s = 0; s < prev_steps; ++s)
            umma_ss_f16(tmem + kTmemO + m * N, a + s * (2048 >> 4), p0 + s * (32 >> 4), idesc_o, !prev_first || s != 0);
          at = at + 2 == kLatent ? 0 : at + 2;
        }
        umma_commit(&S.done[prev_k % kSlots]);
        if (prev_last) umma_commit(&S.o_full);
      }
      __syncwarp();
    };
    int block = 0;
    while (walk.next(p)) {
      for (int i = 0; i < p.n; ++i, ++k, block += blocks) {
        if (i == 0) wait_for(&S.q_full, piece & 1, &S.abort, err);
        wait_for(&S.s_free[k & 1], ((k >> 1) & 1) ^ 1, &S.abort, err);
        tc_fence_after_sync();
        const uint32_t s = tmem + (k & 1) * N;
        for (int d = 0; d <= blocks; ++d) {
          const bool rope = d == blocks;
          const int q = block + d;
          if (rope) wait_for(&S.rope_full[k % kRopes], (k / kRopes) & 1, &S.abort, err);
          else if (!(d & 1)) wait_for(&S.full[q % kLatent / 2], (q / kLatent) & 1, &S.abort, err);
          if (elect_lane()) {
            const uint64_t a = umma_desc_k_sw128(rope ? smem_u32(S.rope[k % kRopes]) : ring0 + q % kLatent * kBlock);
            const uint64_t b = q0 + d * (N * 128 >> 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) umma_ss_f16(s, a + j * 2, b + j * 2, idesc_s, d != 0 || j != 0);
          }
          __syncwarp();
        }
        if (elect_lane()) {
          umma_commit(&S.s_full[k & 1]);
          if (i == p.n - 1) umma_commit(&S.q_free);
        }
        __syncwarp();
        if (prev_block >= 0) values();
        prev_block = block;
        prev_k = k;
        prev_piece = piece;
        prev_first = i == 0;
        prev_last = i == p.n - 1;
        prev_steps = cdiv(min(p.x.len - (p.t0 + i) * kTile, kTile), 16);
      }
      ++piece;
    }
    if (prev_block >= 0) values();
  } else if (warp < kSoftWarp) {
    Walk<N> walk(A, start);
    Piece p;
    const int tid = static_cast<int>(threadIdx.x) - 64, per = A.steps * A.heads, chunks = A.rank / 8 + 8;
    for (uint32_t piece = 0; walk.next(p); ++piece) {
      wait_for(&S.q_free, (piece & 1) ^ 1, &S.abort, err);
      // eight lanes a row's 128 bytes
      for (int r = tid >> 3; r < N; r += 8) {
        const int row = p.row0 + r, b = row / per, i = row % per / A.heads, h = row % A.heads;
        const bool on = r < p.rows;
        const uint4* ql = reinterpret_cast<const uint4*>(static_cast<const T*>(A.q_latent) + b * A.q_latent_stride[0] + i * A.q_latent_stride[1] +
                                                         h * A.q_latent_stride[2]);
        const uint4* qr = reinterpret_cast<const uint4*>(static_cast<const T*>(A.q_rope) + b * A.q_rope_stride[0] + i * A.q_rope_stride[1] +
                                                         h * A.q_rope_stride[2]);
        uint4 v[9];
#pragma unroll
        for (int d = 0; d < 9; ++d) {
          const int at = d * 8 + (tid & 7);
          v[d] = make_uint4(0, 0, 0, 0);
          if (on && at < chunks) v[d] = at < chunks - 8 ? ql[at] : qr[at - (chunks - 8)];
        }
#pragma unroll
        for (int d = 0; d < 9; ++d)
          if (d <= blocks) *reinterpret_cast<uint4*>(S.q[d] + r * 128 + (((tid & 7) ^ (r & 7)) << 4)) = v[d];
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.q_full);
    }
  } else {
    Walk<N> walk(A, start);
    Piece p;
    const int quad = warp & 3;
    const uint32_t lanes = static_cast<uint32_t>(32 * quad) << 16;
    uint32_t k = 0;
    for (uint32_t piece = 0; walk.next(p); ++piece) {
      const bool prefix = p.e < A.groups;
      float ref[kCols], sum[kCols];
      int limit[kCols], least = p.x.len, most = 0;
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        const int col = 8 * (j >> 1) + 2 * (lane & 3) + (j & 1);
        ref[j] = -INFINITY;
        sum[j] = 0.f;
        limit[j] = 0;
        if (col < p.rows) {
          limit[j] = limit_of(A, p.x, prefix, p.row0 + col);
          least = min(least, limit[j]);
          most = max(most, limit[j]);
        }
      }
#pragma unroll
      for (int x = 1; x < 4; x <<= 1) {
        least = min(least, __shfl_xor_sync(0xffffffffu, least, x));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, x));
      }
      for (int i = 0; i < p.n; ++i, ++k) {
        const int t0 = (p.t0 + i) * kTile;
        wait_for(&S.told[k % kSlots], (k / kSlots) & 1, &S.abort, err);
        const int bad = S.bad[k % kSlots];
        wait_for(&S.s_full[k & 1], (k >> 1) & 1, &S.abort, err);
        tc_fence_after_sync();
        uint32_t raw[2 * kCols];
#pragma unroll
        for (int j = 0; j < N / 16; ++j) tmem_load_fragments(tmem + lanes + (k & 1) * N + 16 * j, raw + 8 * j);
        tmem_loaded(raw);
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.s_free[k & 1]);
        // v[2 j + r]: row of queries 8 (j / 2) + 2 (lane % 4) + j % 2, position 16 quad + lane / 4 + 8 r
        float v[2 * kCols];
#pragma unroll
        for (int j = 0; j < kCols; ++j)
#pragma unroll
          for (int r = 0; r < 2; ++r) v[2 * j + r] = __uint_as_float(raw[4 * (j >> 1) + 2 * r + (j & 1)]) * P.scale;
        const int mine = t0 + 16 * quad + (lane >> 2);
        const bool edge = t0 + kTile > least;
        if (edge) {
#pragma unroll
          for (int j = 0; j < kCols; ++j)
#pragma unroll
            for (int r = 0; r < 2; ++r)
              if (mine + 8 * r >= limit[j]) v[2 * j + r] = -INFINITY;
        }
        float top[kCols];
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          top[j] = fmaxf(v[2 * j], v[2 * j + 1]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], x));
        }
        if (lane < 4) {
#pragma unroll
          for (int j = 0; j < kCols; j += 2)
            *reinterpret_cast<float2*>(&S.wmax[k & 1][quad][4 * j + 2 * lane]) = make_float2(top[j], top[j + 1]);
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int j = 0; j < kCols; j += 2) {
            const float2 f = *reinterpret_cast<const float2*>(&S.wmax[k & 1][w][4 * j + 2 * (lane & 3)]);
            top[j] = fmaxf(top[j], f.x);
            top[j + 1] = fmaxf(top[j + 1], f.y);
          }
        bool move = false;
#pragma unroll
        for (int j = 0; j < kCols; ++j) move |= top[j] > ref[j] + (kOffset + 8.f);
        // the weights' place, and O, are free once the MMAs of the tile before are complete
        if (i > 0) wait_for(&S.done[(k - 1) % kSlots], ((k - 1) / kSlots) & 1, &S.abort, err);
        if (__any_sync(0xffffffffu, move)) {  // the same in all four warps
          float f[kCols];
#pragma unroll
          for (int j = 0; j < kCols; ++j) {
            const float now = fmaxf(ref[j], top[j] - kOffset);
            f[j] = now == -INFINITY ? 1.f : exp2_fast(ref[j] - now);
            ref[j] = now;
            sum[j] *= f[j];
          }
          if (i > 0) {
            if (lane < 4 && quad == 0) {
#pragma unroll
              for (int j = 0; j < kCols; j += 2) *reinterpret_cast<float2*>(&S.fac[4 * j + 2 * lane]) = make_float2(f[j], f[j + 1]);
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            tc_fence_after_sync();
            for (int m = 0; m < blocks / 2; ++m)
#pragma unroll
              for (int j = 0; j < N; j += 16) {
                uint32_t o[16];
                tmem_load16(tmem + lanes + kTmemO + m * N + j, o);
                tmem_loaded(o);
#pragma unroll
                for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * S.fac[j + x]);
                tmem_store16(tmem + lanes + kTmemO + m * N + j, o);
              }
            tmem_stored();
            tc_fence_before_sync();
          }
        }
        // Rows of the tile that not all queries see: nothing of them may come through a weight of 0.
        uint32_t poison = 0;
        if (edge) {
          const int block = static_cast<int>(k) * blocks + (lane >> 2);  // lane: 32 bytes of one of the rank's blocks
          for (int d = 0; d < blocks; d += 2) {  // complete, as S is: that this thread sees what TMA wrote
            const int q = static_cast<int>(k) * blocks + d;
            wait_for(&S.full[q % kLatent / 2], (q / kLatent) & 1, &S.abort, err);
          }
          for (int r = max(least - t0 - 16 * quad, 0); r < 16; ++r) {
            const int pos = t0 + 16 * quad + r;
            uint4* at = reinterpret_cast<uint4*>(S.ring[block % kLatent] + (16 * quad + r) * 128) + 2 * (lane & 3);
            const bool have = (lane >> 2) < blocks;
            bool wipe = pos >= most;
            if (!wipe) {
              wipe = __any_sync(0xffffffffu, have && (has_nonfinite<T>(at[0]) || has_nonfinite<T>(at[1])));
              if (wipe) poison |= 1u << r;
            }
            if (wipe && have) at[0] = at[1] = make_uint4(0, 0, 0, 0);
          }
        }
        if (bad >> quad & 1) poison = 0xffff;
        uint32_t w[kCols];
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          const float base = ref[j] == -INFINITY ? 0.f : ref[j];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float x = exp2_fast(v[2 * j + r] - base);
            if (poison >> ((lane >> 2) + 8 * r) & 1) x = __int_as_float(0x7fc00000);
            if (edge && mine + 8 * r >= limit[j]) x = 0.f;
            v[2 * j + r] = x;
          }
          sum[j] += v[2 * j] + v[2 * j + 1];
        }
#pragma unroll
        for (int j = 0; j < kCols; j += 2) {
          w[j] = Pair<T>::r(v[2 * j], v[2 * j + 2]);          // position lane / 4
          w[j + 1] = Pair<T>::r(v[2 * j + 1], v[2 * j + 3]);  // ... + 8
        }
        // transposed 8 x 8 blocks: a row of queries has its 64 weights in 128 bytes, 16-byte pieces swizzled by the row
#pragma unroll
        for (int j = 0; j < N / 16; ++j) {
          const int row = 16 * j + 8 * (lane >> 4) + (lane & 7), piece16 = 2 * quad + ((lane >> 3) & 1);
          asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(
                           smem_u32(S.p) + row * 128 + ((piece16 ^ (row & 7)) << 4)),
                       "r"(w[4 * j]), "r"(w[4 * j + 1]), "r"(w[4 * j + 2]), "r"(w[4 * j + 3])
                       : "memory");
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.p_full);
      }
      // sums of the weights over the positions, through the place of the maxima of the tile before the last
#pragma unroll
      for (int j = 0; j < kCols; ++j)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], x);
      if (lane < 4) {
#pragma unroll
        for (int j = 0; j < kCols; j += 2)
          *reinterpret_cast<float2*>(&S.wmax[k & 1][quad][4 * j + 2 * lane]) = make_float2(sum[j], sum[j + 1]);
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");  // the last correction's factors are read
      if (lane < 4 && quad == 0) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) S.fac[4 * (j & ~1) + 2 * lane + (j & 1)] = ref[j];
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      const bool whole = p.whole && A.groups == 0;
      const int slot = p.rt + c;  // pieces of the launch in order: either grows
      if (slot >= P.slots) atomicExch(err, GEMQ_LATENT_BAD_LENGTH);
      // thread 32 quad + lane: dimension 128 m + that of all rows of queries; first its row's sums
      const int me = 32 * quad + lane;
      const float(&lsum)[4][N] = S.wmax[k & 1];
      if (me < p.rows && (whole || slot < P.slots)) {
        const float l = lsum[0][me] + lsum[1][me] + lsum[2][me] + lsum[3][me], m = S.fac[me];
        if (whole) A.lse[p.row0 + me] = limit_of(A, p.x, prefix, p.row0 + me) > 0 ? (m + log2f(l)) * kLn2 : -INFINITY;
        else P.part_ml[static_cast<long long>(slot) * N + me] = make_float2(m, l);
      }
      wait_for(&S.o_full, piece & 1, &S.abort, err);
      tc_fence_after_sync();
      for (int m = 0; m < blocks / 2; ++m)
#pragma unroll 1
        for (int j = 0; j < N; j += 16) {
          uint32_t o[16];
          tmem_load16(tmem + lanes + kTmemO + m * N + j, o);
          tmem_loaded(o);
          if (whole) {
            T* out = static_cast<T*>(A.out) + static_cast<long long>(p.row0 + j) * A.rank + 128 * m + (me & ~1);
#pragma unroll
            for (int x = 0; x < 16; x += 2) {  // an even lane takes row x of a pair of dimensions, its neighbour row x + 1
              const float give = __uint_as_float(lane & 1 ? o[x] : o[x + 1]), keep = __uint_as_float(lane & 1 ? o[x + 1] : o[x]);
              const float got = __shfl_xor_sync(0xffffffffu, give, 1);
              const int r = x + (lane & 1), col = j + r;
              if (col < p.rows) {
                const float l = lsum[0][col] + lsum[1][col] + lsum[2][col] + lsum[3][col];
                const float f = l == 0.f && limit_of(A, p.x, prefix, p.row0 + col) <= 0 ? 0.f : 1.f / l;
                *reinterpret_cast<uint32_t*>(out + r * static_cast<long long>(A.rank)) =
                    lane & 1 ? Pair<T>::r(got * f, keep * f) : Pair<T>::r(keep * f, got * f);
              }
            }
          } else if (slot < P.slots) {
            float* out = P.part_o + (static_cast<long long>(slot) * N + j) * A.rank + 128 * m + me;
#pragma unroll
            for (int x = 0; x < 16; ++x)
              if (j + x < p.rows) out[x * static_cast<long long>(A.rank)] = __uint_as_float(o[x]);
          }
        }
      tc_fence_before_sync();
      asm volatile("bar.sync 1, 128;" ::: "memory");  // sums and references are read
      if (lane == 0) mbar_arrive(&S.o_free);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ---- pieces of a row joined ---------------------------------------------------------------------------
// 128 numbers of a row at a time: four warps take its pieces in turn and add in a fixed order.
template <typename T>
__global__ void __launch_bounds__(128) latent_join_kernel(const __grid_constant__ Args P, int N) {
  __shared__ float4 part[4][32];
  __shared__ float part_l[4];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const gemq_latent_decode_t& A = P.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = A.steps * A.heads, cuts = A.rank / 128;
  const int total = P.ctl[0], ctas = P.ctl[1];
  const long long jobs = static_cast<long long>(A.batch) * per * cuts;
  for (long long job = blockIdx.x; job < jobs; job += gridDim.x) {
    const int row = static_cast<int>(job / cuts), cut = static_cast<int>(job % cuts);
    const int b = row / per, hidden = A.steps - 1 - row % per / A.heads;
    // runs of slots: of the group's prefix, of the sequence's own tiles
    int slot[2] = {0, 0}, count[2] = {0, 0}, at[2] = {0, 0}, len = 0;
    bool whole = false;
    if (total > 0) {
      if (A.groups > 0) {
        int g = 0, hi = A.groups;  // the last group that begins at b or before (g < hi)
        while (hi - g > 1) {
          const int mid = (g + hi) >> 1;
          if (start_of(A, mid) <= b) g = mid;
          else hi = mid;
        }
        const Entry x = entry_of(A, g);
        const int r = row - x.row0;
        if (x.tiles > 0 && r >= 0 && r < x.rows) {
          len += x.len;
          const long long t = P.ctl[2 + 2 * g] + static_cast<long long>(r / N) * x.tiles;
          const int c0 = cta_of(t, total, ctas), c1 = cta_of(t + x.tiles - 1, total, ctas);
          slot[0] = P.ctl[3 + 2 * g] + r / N + c0;
          count[0] = c1 - c0 + 1;
          at[0] = r % N;
        }
      }
      const int e = A.groups + b;
      const Entry x = entry_of(A, e);
      len += x.len;
      if (x.tiles > 0) {
        const int r = row - x.row0;
        const long long t = P.ctl[2 + 2 * e] + static_cast<long long>(r / N) * x.tiles;
        const int c0 = cta_of(t, total, ctas), c1 = cta_of(t + x.tiles - 1, total, ctas);
        slot[1] = P.ctl[3 + 2 * e] + r / N + c0;
        count[1] = c1 - c0 + 1;
        at[1] = r % N;
        whole = A.groups == 0 && c0 == c1;
      }
    }
    if (whole) continue;  // written already
    const int pieces = count[0] + count[1];
    auto place = [&](int i) -> long long {  // row of the scratch
      return i < count[0] ? static_cast<long long>(slot[0] + i) * N + at[0] : static_cast<long long>(slot[1] + i - count[0]) * N + at[1];
    };
    const long long rows = static_cast<long long>(P.slots) * N;
    float top = -INFINITY;
    for (int i = lane; i < pieces; i += 32)
      if (place(i) < rows) top = fmaxf(top, P.part_ml[place(i)].x);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float base = top == -INFINITY ? 0.f : top;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll 4
    for (int i = warp; i < pieces; i += 4) {
      const long long q = place(i);
      if (q >= rows) continue;
      const float2 ml = P.part_ml[q];
      const float4 v = reinterpret_cast<const float4*>(P.part_o + q * A.rank + cut * 128)[lane];
      const float f = exp2_fast(ml.x - base);
      l = fmaf(ml.y, f, l);
      o.x = fmaf(v.x, f, o.x);
      o.y = fmaf(v.y, f, o.y);
      o.z = fmaf(v.z, f, o.z);
      o.w = fmaf(v.w, f, o.w);
    }
    part[warp][lane] = o;
    if (lane == 0) part_l[warp] = l;
    __syncthreads();
    if (warp == 0) {
      l = part_l[0] + part_l[1] + part_l[2] + part_l[3];
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        const float4 v = part[w][lane];
        o.x += v.x;
        o.y += v.y;
        o.z += v.z;
        o.w += v.w;
      }
      const bool empty = len - hidden <= 0;
      const float f = 1.f / l;
      reinterpret_cast<uint2*>(static_cast<T*>(A.out) + static_cast<long long>(row) * A.rank + cut * 128)[lane] =
          empty ? make_uint2(0, 0) : make_uint2(Pair<T>::r(o.x * f, o.y * f), Pair<T>::r(o.z * f, o.w * f));
      if (lane == 0 && cut == 0) A.lse[row] = empty ? -INFINITY : (top + log2f(l)) * kLn2;
    }
    __syncthreads();
  }
}

int check(const gemq_latent_decode_t* A) {
  if (!A || !A->q_latent || !A->q_rope || !A->cache || !A->table || !A->lens || !A->out || !A->lse || !A->err) return GEMQ_ERR_BAD_ARG;
  if (A->batch < 0 || A->steps <= 0 || A->heads <= 0 || A->n_pages <= 0 || A->table_pitch < 0 || A->groups < 0) return GEMQ_ERR_BAD_ARG;
  if (A->groups && (!A->prefix_table || !A->prefix_lens || !A->starts || A->prefix_pitch < 0)) return GEMQ_ERR_BAD_ARG;
  if (!rank_ok(A->rank) || !page_ok(A->page_size)) return GEMQ_ERR_BAD_SHAPE;
  const long long rows = static_cast<long long>(A->batch) * A->steps * A->heads;
  if (rows > (1 << 30) || A->groups > (1 << 24)) return GEMQ_ERR_BAD_SHAPE;
  // the list of work is counted in 32 bits
  const long long own = static_cast<long long>(A->table_pitch) * A->page_size, pre = static_cast<long long>(A->prefix_pitch) * A->page_size;
  const long long tiles = (rows / 16 + A->batch) * (own / kTile + 1) + (A->groups ? (rows / 16 + A->groups) * (pre / kTile + 1) : 0);
  if (own > 0x7fffff00 || pre > 0x7fffff00 || tiles > 0x7fffffff) return GEMQ_ERR_BAD_SHAPE;
  if (!aligned16(A->q_latent) || !aligned16(A->q_rope) || !aligned16(A->cache) || !aligned16(A->out) || (A->page_stride & 7))
    return GEMQ_ERR_ALIGN;
  for (int i = 0; i < 3; ++i)
    if ((A->q_latent_stride[i] | A->q_rope_stride[i]) & 7) return GEMQ_ERR_ALIGN;
  return GEMQ_OK;
}

// Rows of queries of a row tile: as many as a sequence has, or all of a group may have.
int row_tile(const gemq_latent_decode_t* A) {
  const long long per = static_cast<long long>(A->steps) * A->heads, rows = A->groups ? per * A->batch : per;
  return rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
}
struct Scratch { int slots; size_t ctl, ml, o, bytes; };
Scratch scratch_of(const gemq_latent_decode_t* A) {
  const int N = row_tile(A);
  const long long per = static_cast<long long>(A->steps) * A->heads;
  Scratch s;
  long long rts = static_cast<long long>(A->batch) * ((per + N - 1) / N);
  if (A->groups) rts += per * A->batch / N + A->groups;
  s.slots = static_cast<int>(rts + sm_count_or_default());
  s.ctl = 0;
  s.ml = (sizeof(int) * (2 + 2 * (static_cast<size_t>(A->groups) + A->batch)) + 255) & ~size_t(255);
  s.o = (s.ml + sizeof(float2) * s.slots * N + 255) & ~size_t(255);
  s.bytes = s.o + sizeof(float) * s.slots * static_cast<size_t>(N) * A->rank;
  return s;
}

template <typename T, int N>
int launch(const Args& P, int ctas, cudaStream_t st) {
  static bool set[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return GEMQ_ERR_LAUNCH;
  if (!set[dev]) {
    if (cudaFuncSetAttribute(latent_decode_kernel<T, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Smem<N>)) != cudaSuccess)
      return GEMQ_ERR_LAUNCH;
    set[dev] = true;
  }
  static_assert(sizeof(Smem<N>) <= 232448, "more shared memory than a CTA has");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Smem<N>);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, latent_decode_kernel<T, N>, P) != cudaSuccess) return GEMQ_ERR_LAUNCH;
  const long long jobs = static_cast<long long>(P.a.batch) * P.a.steps * P.a.heads * (P.a.rank / 128), most = 8ll * ctas;
  cfg.gridDim = dim3(static_cast<unsigned>(jobs < most ? jobs : most));
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, latent_join_kernel<T>, P, N) == cudaSuccess ? GEMQ_OK : GEMQ_ERR_LAUNCH;
}

template <typename T>
int launch(const Args& P, int N, int ctas, cudaStream_t st) {
  return N == 16 ? launch<T, 16>(P, ctas, st) : N == 32 ? launch<T, 32>(P, ctas, st) : launch<T, 64>(P, ctas, st);
}

}  // namespace
}  // namespace latent
}  // namespace gemq

using namespace gemq;
using namespace gemq::latent;

extern "C" size_t gemq_latent_decode_scratch_bytes(const gemq_latent_decode_t* A) {
  return check(A) != GEMQ_OK || A->batch == 0 ? 0 : scratch_of(A).bytes;
}

extern "C" int gemq_latent_decode(const gemq_latent_decode_t* A, void* scratch, size_t scratch_bytes, gemq_stream_t stream) {
  const int rc = check(A);
  if (rc) return rc;
  if (!A->batch) return GEMQ_OK;
  const Scratch s = scratch_of(A);
  if (!scratch || scratch_bytes < s.bytes) return GEMQ_ERR_WORKSPACE;
  if (!aligned16(scratch)) return GEMQ_ERR_ALIGN;
  const int sms = sm_count();
  if (sms <= 0) return GEMQ_ERR_LAUNCH;
  Args P;
  P.a = *A;
  P.ctl = reinterpret_cast<int*>(static_cast<char*>(scratch) + s.ctl);
  P.part_ml = reinterpret_cast<float2*>(static_cast<char*>(scratch) + s.ml);
  P.part_o = reinterpret_cast<float*>(static_cast<char*>(scratch) + s.o);
  P.slots = s.slots;
  P.scale = A->scale * kLog2e;
  const int rows = A->page_size < kTile ? A->page_size : kTile;
  P.box_blocks = A->page_size < kTile ? 1 : 2;
  const int blocks = A->rank / 64 + 1;
  if (!tensor_map_pages(&P.latent_map, A->cache, blocks, A->page_size, A->page_stride, A->n_pages, rows, P.box_blocks) ||
      !tensor_map_pages(&P.rope_map, A->cache, blocks, A->page_size, A->page_stride, A->n_pages, rows, 1))
    return GEMQ_ERR_LAUNCH;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int N = row_tile(A);
  return A->is_bf16 ? launch<__nv_bfloat16>(P, N, sms, st) : launch<__half>(P, N, sms, st);
}
