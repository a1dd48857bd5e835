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
// into shares of equal cost; a CTA's share is a run of pieces (row tile, range of tiles).  A piece that is all of a row tile is finished
// in place, others leave their sums (fp32), maximum and sum of weights to the second kernel, which joins them in order of position.
//   warp 0       TMA: a ring of blocks of 64 rows x 64 numbers, latent ones in pairs (2.75 tiles deep at N = 16), rope ones apart
//   warps 1, 2   MMAs of S, of O.  (One warp for S of tile k + 1, then O of tile k: the latter waited for tile k + 1 to arrive, and the
//                ring for it.)
//   warps 4-7    softmax (a thread has two positions x N / 4 rows), O's correction
//   warps 8-11   the queries of the next piece into shared memory, results of the last
// The maximum that a row's weights refer to moves only when its own scores exceed it by 2^8: O is corrected in tensor memory a few times per
// sequence, and no row's bits depend on what others of its tile hold or see.  Weights are rounded to the type for the second product, their sums are
// not: as 16 bits are what the product takes, and the logarithm of the sum keeps all of its own.  Rows behind what is seen are zeroed in shared memory before they are multiplied by weights of 0: what lies there may be NaN.
// Every wait is bounded.
//
// Measured (rank 512; the call with both launches): 37 sequences of 60 to 9000 positions, 16 heads, 80 MB: 35 us, 2.3 TB/s; 2 sequences of 70,001
// and 131,072, 48 rows each, 232 MB: 67 us, 3.5 TB/s; 64 sequences behind a prefix of 8000, 18 GFLOP: 50 us; one of 700: 11.5 us.  A CTA's 64
// positions take 3100 to 3300 cycles with all SMs at work: 16 rows what HBM gives (3100), 64 rows the two products' reads of shared memory
// (2000 cycles of MMAs, 340 KB at 128 bytes a cycle) and a ring of two tiles.  The rest is fixed: 3 to 5 us to the first copy, 3 to the first
// weights, 1 to 4 for results (64 rows: 131 KB at 32 bytes a cycle), 2 to 6 for the join.
#include "latent.cuh"

namespace gemq {

// tma.cu
bool tensor_map_pages(CUtensorMap* out, const void* base, int blocks, int page_size, long long page_stride, int pages, int box_rows,
                      int box_blocks);

namespace latent {
namespace {

constexpr int kTile = 64;            // positions of a tile
constexpr int kBlock = kTile * 128;  // bytes of 64 positions x 64 numbers
constexpr int kThreads = 384;
constexpr int kSoftWarp = 4, kEdgeWarp = 8;  // four each: a warp reads the quarter of the tensor memory that its number names
constexpr int kSlots = 8;            // tiles in flight that are told apart: one more than the rope blocks, 4, at most

// Blocks of the ring: what 227 KB hold beside the queries.
template <int N> struct Ring;
template <> struct Ring<16> { static constexpr int kLatent = 22, kRopes = 3; };
template <> struct Ring<32> { static constexpr int kLatent = 20, kRopes = 3; };
template <> struct Ring<64> { static constexpr int kLatent = 16, kRopes = 2; };

// Positions, tiles of 64, first query row (of batch * steps * heads), query rows; what a piece costs beside its tiles, in quarters of a tile, and
// what a row tile costs.
struct Entry { int len, tiles, row0, rows, piece, cost; };
struct Start { int e, rt, base, from, to, rto; Entry x; };  // Walk's

template <int N>
struct Smem {
  static constexpr int kLatent = Ring<N>::kLatent, kRopes = Ring<N>::kRopes;
  static constexpr int kOs = N <= 32 ? 2 : 1;  // accumulators that tensor memory holds
  alignas(1024) unsigned char ring[kLatent][kBlock];
  unsigned char rope[kRopes][kBlock];
  unsigned char q[9][N * 128];
  unsigned char p[N * 128];
  float wmax[4][N];
  float fac[N];
  float2 result[N];  // reference and sum of the weights of the piece that is finished
  int limit[N];
  alignas(8) unsigned long long full[kLatent / 2], empty[kLatent / 2], rope_full[kRopes];
  unsigned long long done[kSlots], told[kSlots];  // the tile's MMAs are complete; its pages are known
  unsigned long long s_full[2], s_free[2], p_full, q_full, q_free, o_full[kOs], o_free[kOs], r_full, r_free;
  int bad[kSlots];  // of the tile's four quarters: on a page outside the cache
  int sums[kThreads / 32][2];
  Start start;
  uint32_t tmem_base;
  int abort;
};

struct Args {
  CUtensorMap latent_map, rope_map;
  gemq_latent_decode_t a;
  int* ctl;          // [0] cost of the list, -1 without one (start_wrong); from [2] per entry: where it begins in it, first row tile
  float* part_o;     // [slots][N][rank]
  float2* part_ml;   // [slots][N]: reference of the weights (in powers of two) and their sum
  int slots;
  float scale;       // times log2 e
  Div per, heads;    // query rows of a sequence; heads
};

// ---- the list of work -----------------------------------------------------------------------------
__device__ __forceinline__ int start_of(const gemq_latent_decode_t& A, int g) {  // within the batch, whatever the device has
  return g <= 0 ? 0 : g >= A.groups ? A.batch : min(max(A.starts[g], 0), A.batch);
}
__device__ __forceinline__ Entry entry_here(const Args& P, int e) {
  const gemq_latent_decode_t& A = P.a;
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
  // Measured at rank 512, two and more pieces of a CTA against one: 16 rows 3.4 us a piece and 2.2 a tile, 64 rows 4 us and 1.7.  (A tile of a lower
  // rank is shorter beside its piece: shares are less even there.)
  x.piece = x.rows <= 32 ? 6 : 9;
  x.cost = x.tiles ? 4 * x.tiles + x.piece : 0;
  return x;
}
// Out of line, as it is wanted in many places: see wait_on.
__device__ __noinline__ Entry entry_of(const Args& P, int e) { return entry_here(P, e); }

// Starts rise from 0 to the batch: this is what group g says of it.  Where they do not there is no list, and results are NaN: groups that each
// had the batch would make one beyond its 32 bits, and more pieces than there are slots.
__device__ __forceinline__ bool start_wrong(const gemq_latent_decode_t& A, int g) {
  const int from = A.starts[g], to = A.starts[g + 1];
  return from > to || (g == 0 && from != 0) || (g == A.groups - 1 && to != A.batch);
}

// Tile t of a row tile that begins at `base` of the list is at base + piece + 4 t.  The list is cut into shares of `share` or, the first
// `longer` of them, one more.  A share is a tile or more: no CTA between a row tile's first and last is without one.
struct Cut {
  int ctas, share, longer;
  __device__ __forceinline__ Cut(int total, int most) {
    ctas = min(most, max(total / 4, 1));
    share = total / ctas;
    longer = total - share * ctas;
  }
  __device__ __forceinline__ int from(int c) const { return c * share + min(c, longer); }
};
// The CTA that has `at`: quotients below 2^10 by 32-bit products are off by less than 2^-10, so their whole parts by one at most.  (By integer
// division the join took 0.3 to 0.6 us more.)
struct Find : Cut {
  float per_long, per_share;
  __device__ __forceinline__ Find(int total, int most) : Cut(total, most) {
    per_long = __fdividef(1.f, static_cast<float>(share + 1));
    per_share = __fdividef(1.f, static_cast<float>(max(share, 1)));
  }
  __device__ __forceinline__ int cta_of(int at) const {
    const int over = at - longer * (share + 1);
    const int c = over < 0 ? static_cast<int>(static_cast<float>(at) * per_long) : longer + static_cast<int>(static_cast<float>(over) * per_share);
    return at < from(c) ? c - 1 : at >= from(c + 1) ? c + 1 : c;
  }
};

// Where a piece of row tile rt leaves its sums.  With prefixes each does, and pieces of the launch in order grow by their row tile or their
// CTA.  Without, a CTA has two such pieces at most: the end of a row tile that others began, and one that others go on with.
__device__ __forceinline__ int slot_of(bool groups, int rt, int cta, bool last) { return groups ? rt + cta : 2 * cta + (last ? 0 : 1); }

struct Piece {
  Entry x;
  int e, t0, n;      // entry, first tile, tiles
  int row0, rows;    // first query row, query rows of the row tile
  int rt;            // row tile of the launch
  __device__ __forceinline__ int width() const { return (rows + 15) & ~15; }
  __device__ __forceinline__ bool whole() const { return n == x.tiles; }
  __device__ __forceinline__ bool last() const { return t0 + n == x.tiles; }
};

template <int N, bool CALL = true>
struct Walk {
  const Args& P;
  Start s;
  Entry x;
  __device__ __forceinline__ Walk(const Args& args, const Start& at)
      : P(args),
        s{uniform(at.e), uniform(at.rt), uniform(at.base), uniform(at.from), uniform(at.to), uniform(at.rto), {}},
        x{uniform(at.x.len), uniform(at.x.tiles), uniform(at.x.row0), uniform(at.x.rows), uniform(at.x.piece), uniform(at.x.cost)} {}
  __device__ __forceinline__ void enter() {
    const Entry y = CALL ? entry_of(P, s.e) : entry_here(P, s.e);
    x = {uniform(y.len), uniform(y.tiles), uniform(y.row0), uniform(y.rows), uniform(y.piece), uniform(y.cost)};
  }
  __device__ __forceinline__ bool next(Piece& p) {
    while (s.base < s.to && s.from < s.to) {
      if (x.cost == 0 || s.rt * N >= x.rows) {
        s.rto += cdiv(x.rows, N);
        s.rt = 0;
        if (++s.e >= P.a.groups + P.a.batch) { s.to = s.from; return false; }
        enter();
        continue;
      }
      const int t0 = min(max((s.from - s.base - x.piece + 3) >> 2, 0), x.tiles);
      const int t1 = min(max((s.to - s.base - x.piece + 3) >> 2, 0), x.tiles);
      p.x = x;
      p.e = s.e;
      p.t0 = t0;
      p.n = t1 - t0;
      p.row0 = x.row0 + s.rt * N;
      p.rows = min(N, x.rows - s.rt * N);
      p.rt = s.rto + s.rt;
      s.base += x.cost;
      ++s.rt;
      if (t1 > t0) return true;
    }
    return false;
  }
};

// Sequence, step and head of a query row.
struct Row {
  int b, i, h;
  __device__ __forceinline__ Row(const Args& P, int r) {
    b = P.per(r);
    const int rest = r - b * P.a.steps * P.a.heads;
    i = P.heads(rest);
    h = rest - i * P.a.heads;
  }
};
// What query row r sees of entry e's positions.
__device__ __forceinline__ int limit_of(const Args& P, const Entry& x, bool prefix, int r) {
  const gemq_latent_decode_t& A = P.a;
  const Row row(P, r);
  const int hidden = A.steps - 1 - row.i;
  if (!prefix) return x.len - hidden;
  return x.len - max(hidden - clamp_length(A.lens[row.b], A.table_pitch, A.page_size, A.err), 0);
}

// Whether any of the 128 softmax threads says so; a barrier of theirs.
__device__ __forceinline__ bool any_of_softmax(bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(mine))
      : "memory");
  return any != 0;
}

// ---- the softmax warps: one piece ---------------------------------------------------------------------
template <typename T, int N, int NP>
__device__ __forceinline__ void softmax_piece(Smem<N>& S, const Args& P, const Piece& p, uint32_t& k, uint32_t piece, uint32_t tmem,
                                              uint32_t acc) {
  constexpr int kLatent = Ring<N>::kLatent;
  constexpr int kCols = NP / 4;  // rows of queries that a thread has
  constexpr float kOffset = Pair<T>::kBf16 ? 0.f : 7.f;  // fp16 weights are 2^7 times as large: those above 2^-21 keep all their bits
  const gemq_latent_decode_t& A = P.a;
  int* const err = A.err;
  const int lane = threadIdx.x & 31, quad = (threadIdx.x >> 5) & 3, blocks = A.rank / 64;
  const bool prefix = p.e < A.groups;
  const uint32_t lanes = static_cast<uint32_t>(32 * quad) << 16;
  float ref[kCols], sum[kCols];  // what the weights refer to, their sums over the thread's positions
  const int me = 32 * quad + lane;
  float my_ref = 0.f;            // of row `me`
  bool my_none = true;           // all its scores so far are -inf, the reference is 0
#pragma unroll
  for (int j = 0; j < kCols; ++j) ref[j] = sum[j] = 0.f;
  int least = p.x.len, most = 0;
  for (int r = lane; r < NP; r += 32) {
    const int limit = r < p.rows ? limit_of(P, p.x, prefix, p.row0 + r) : 0;
    if (quad == 0) S.limit[r] = limit;
    if (r < p.rows) {
      least = min(least, limit);
      most = max(most, limit);
    }
  }
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  asm volatile("bar.sync 1, 128;" ::: "memory");
  bool unset = true;
  for (int i = 0; i < p.n; ++i, ++k) {
    const int t0 = (p.t0 + i) * kTile;
    wait_for(&S.told[k % kSlots], (k / kSlots) & 1, &S.abort, err);
    const int bad = S.bad[k % kSlots];
    wait_for(&S.s_full[k & 1], (k >> 1) & 1, &S.abort, err);
    tc_fence_after_sync();
    uint32_t raw[2 * kCols];
#pragma unroll
    for (int j = 0; j < NP / 16; ++j) tmem_load_fragments(tmem + lanes + (k & 1) * N + 16 * j, raw + 8 * j);
    tmem_loaded(raw);
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(&S.s_free[k & 1]);
    // v[2 j + r]: row of queries 8 (j / 2) + 2 (lane % 4) + j % 2, position 16 quad + lane / 4 + 8 r
    float v[2 * kCols];
#pragma unroll
    for (int j = 0; j < kCols; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) v[2 * j + r] = fmaf(__uint_as_float(raw[4 * (j >> 1) + 2 * r + (j & 1)]), P.scale, -ref[j]);
    const int mine = t0 + 16 * quad + (lane >> 2);
    const bool edge = t0 + kTile > least;
    if (edge) {
#pragma unroll
      for (int j = 0; j < kCols; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r)
          if (mine + 8 * r >= S.limit[8 * (j >> 1) + 2 * (lane & 3) + (j & 1)]) v[2 * j + r] = -INFINITY;
    }
    // Weights above 2^8 times the reference move it: as a rule none, and no maximum is formed.
    float high = v[0];
#pragma unroll
    for (int j = 1; j < 2 * kCols; ++j) high = fmaxf(high, v[j]);
    const bool move = any_of_softmax(unset || high > kOffset + 8.f);
    // the weights' place, and O, are free once the MMAs of the tile before are complete
    if (k > 0) wait_for(&S.done[(k - 1) % kSlots], ((k - 1) / kSlots) & 1, &S.abort, err);
    if (move) {
      // A thread a row of queries from here: short code, as most launches come here once, with nothing of it in the instruction cache (all
      // threads with the maxima of their rows, by shuffles: 6500 cycles for 48 rows).  The maxima meet in the place of the weights.
      float* const scratch = reinterpret_cast<float*>(S.p);
#pragma unroll
      for (int j = 0; j < kCols; j += 2)
        *reinterpret_cast<float2*>(scratch + (8 * quad + (lane >> 2)) * NP + 4 * j + 2 * (lane & 3)) =
            make_float2(fmaxf(v[2 * j], v[2 * j + 1]), fmaxf(v[2 * j + 2], v[2 * j + 3]));
      asm volatile("bar.sync 1, 128;" ::: "memory");
      bool still = false;
      if (me < NP) {
        float top = -INFINITY;
#pragma unroll 4
        for (int r = 0; r < 32; ++r) top = fmaxf(top, scratch[r * NP + me]);
        // Relative to the reference so far; a row that has none takes what there is.  Only a row of its own scores: which others stand beside it
        // in the tile, and what those see, is to change none of its bits.
        const float up = my_none || top > kOffset + 8.f ? top - kOffset : 0.f;
        const bool nothing = my_none && up == -INFINITY;
        const float by = nothing ? 0.f : up;
        still = nothing && S.limit[me] > 0;
        S.wmax[0][me] = by;
        S.fac[me] = my_none ? 1.f : exp2_fast(-by);
        my_none = my_none && nothing;
        my_ref += by;
      }
      unset = any_of_softmax(still);
#pragma unroll
      for (int j = 0; j < kCols; j += 2) {
        const float2 by = *reinterpret_cast<const float2*>(&S.wmax[0][4 * j + 2 * (lane & 3)]);
        const float2 f = *reinterpret_cast<const float2*>(&S.fac[4 * j + 2 * (lane & 3)]);
        ref[j] += by.x;
        ref[j + 1] += by.y;
        sum[j] *= f.x;
        sum[j + 1] *= f.y;
        v[2 * j] -= by.x;
        v[2 * j + 1] -= by.x;
        v[2 * j + 2] -= by.y;
        v[2 * j + 3] -= by.y;
      }
      if (i > 0) {
        tc_fence_after_sync();
        for (int m = 0; m < blocks / 2; ++m)
#pragma unroll 1
          for (int j = 0; j < NP; j += 16) {
            uint32_t o[16];
            tmem_load16(acc + lanes + m * N + j, o);
            tmem_loaded(o);
#pragma unroll
            for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * S.fac[j + x]);
            tmem_store16(acc + lanes + m * N + j, o);
          }
        tmem_stored();
        tc_fence_before_sync();
      }
    }
#pragma unroll
    for (int j = 0; j < 2 * kCols; ++j) v[j] = exp2_fast(v[j]);
    // Rows of the tile that not all queries see: nothing of them may come through a weight of 0.  A page that is none: NaN.
    if (edge || bad) {
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
#pragma unroll
      for (int j = 0; j < kCols; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if (poison >> ((lane >> 2) + 8 * r) & 1) v[2 * j + r] = __int_as_float(0x7fc00000);
          if (mine + 8 * r >= S.limit[8 * (j >> 1) + 2 * (lane & 3) + (j & 1)]) v[2 * j + r] = 0.f;
        }
    }
    uint32_t w[kCols];
#pragma unroll
    for (int j = 0; j < kCols; ++j) sum[j] += v[2 * j] + v[2 * j + 1];
#pragma unroll
    for (int j = 0; j < kCols; j += 2) {
      w[j] = Pair<T>::r(v[2 * j], v[2 * j + 2]);          // position lane / 4
      w[j + 1] = Pair<T>::r(v[2 * j + 1], v[2 * j + 3]);  // ... + 8
    }
    // transposed 8 x 8 blocks: a row of queries has its 64 weights in 128 bytes, 16-byte pieces swizzled by the row
#pragma unroll
    for (int j = 0; j < NP / 16; ++j) {
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
  // sums of the weights over the positions
#pragma unroll
  for (int j = 0; j < kCols; ++j)
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], x);
  asm volatile("bar.sync 1, 128;" ::: "memory");  // what the last correction left there is read
  if (lane < 4) {
#pragma unroll
    for (int j = 0; j < kCols; j += 2) *reinterpret_cast<float2*>(&S.wmax[quad][4 * j + 2 * lane]) = make_float2(sum[j], sum[j + 1]);
  }
  wait_for(&S.r_free, (piece & 1) ^ 1, &S.abort, err);
  asm volatile("bar.sync 1, 128;" ::: "memory");
  if (me < NP) S.result[me] = make_float2(my_none ? -INFINITY : my_ref, S.wmax[0][me] + S.wmax[1][me] + S.wmax[2][me] + S.wmax[3][me]);
  __syncwarp();
  if (lane == 0) mbar_arrive(&S.r_full);
}

// ---- the warps at a piece's two ends ------------------------------------------------------------------
// Its queries: eight lanes a row's 128 bytes of a block, all copies in flight.
template <typename T, int N>
__device__ __forceinline__ void load_queries(Smem<N>& S, const Args& P, const Piece& p, uint32_t piece) {
  const gemq_latent_decode_t& A = P.a;
  const int tid = static_cast<int>(threadIdx.x) - 32 * kEdgeWarp, blocks = A.rank / 64;
  wait_for<N != 64>(&S.q_free, (piece & 1) ^ 1, &S.abort, A.err);
  for (int r = tid >> 3; r < p.width(); r += 16) {
    const Row row(P, r < p.rows ? p.row0 + r : p.row0);
    const uint4* ql = reinterpret_cast<const uint4*>(static_cast<const T*>(A.q_latent) + row.b * A.q_latent_stride[0] + row.i * A.q_latent_stride[1] +
                                                     row.h * A.q_latent_stride[2]);
    const uint4* qr = reinterpret_cast<const uint4*>(static_cast<const T*>(A.q_rope) + row.b * A.q_rope_stride[0] + row.i * A.q_rope_stride[1] +
                                                     row.h * A.q_rope_stride[2]);
    const uint32_t dst = smem_u32(S.q[0]) + r * 128 + (((tid & 7) ^ (r & 7)) << 4), bytes = r < p.rows ? 16 : 0;  // 0: zeros
    for (int d = 0; d <= blocks; ++d) {
      const uint4* src = d < blocks ? ql + d * 8 + (tid & 7) : qr + (tid & 7);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + d * (N * 128)),
                   "l"(bytes ? static_cast<const void*>(src) : A.q_latent), "r"(bytes)
                   : "memory");
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  fence_async_smem();
  __syncwarp();
  if ((tid & 31) == 0) mbar_arrive(&S.q_full);
}

// Its results: thread 32 quad + lane has dimension 128 m + that of all rows of queries.
template <typename T, int N>
__device__ __forceinline__ void finish_piece(Smem<N>& S, const Args& P, const Piece& p, uint32_t piece, uint32_t acc) {
  constexpr int kOs = Smem<N>::kOs;
  const gemq_latent_decode_t& A = P.a;
  const int lane = threadIdx.x & 31, quad = (threadIdx.x >> 5) & 3, me = 32 * quad + lane;
  const uint32_t lanes = static_cast<uint32_t>(32 * quad) << 16;
  const bool prefix = p.e < A.groups, whole = p.whole() && A.groups == 0;
  const int slot = slot_of(A.groups > 0, p.rt, blockIdx.x, p.last());
  const bool fits = static_cast<unsigned>(slot) < static_cast<unsigned>(P.slots);
  if (!fits) atomicExch(A.err, GEMQ_LATENT_BAD_LENGTH);
  wait_for<N != 64>(&S.r_full, piece & 1, &S.abort, A.err);
  if (me < p.rows && (whole || fits)) {
    const float2 r = S.result[me];
    if (whole) {
      const bool empty = limit_of(P, p.x, prefix, p.row0 + me) <= 0;
      A.lse[p.row0 + me] = empty ? -INFINITY : (r.x + log2f(r.y)) * kLn2;
      S.result[me].y = empty ? 0.f : __fdividef(1.f, r.y);
    } else {
      P.part_ml[static_cast<long long>(slot) * N + me] = r;
    }
  }
  if (whole) asm volatile("bar.sync 2, 128;" ::: "memory");  // the factors
  wait_for<N != 64>(&S.o_full[piece % kOs], (piece / kOs) & 1, &S.abort, A.err);
  tc_fence_after_sync();
  // 16 rows of queries at a time, all their dimensions in flight
  const int quarters = A.rank / 128;
#pragma unroll 1
  for (int j = 0; j < p.rows; j += 16) {
    uint32_t o[64];
#pragma unroll
    for (int m = 0; m < 4; ++m)
      if (m < quarters) tmem_load16(acc + lanes + m * N + j, o + 16 * m);
    tmem_loaded(o);
    if (whole) {
      T* out = static_cast<T*>(A.out) + static_cast<long long>(p.row0 + j + (lane & 1)) * A.rank + (me & ~1);
#pragma unroll
      for (int x = 0; x < 16; x += 2) {  // an even lane takes row x of a pair of dimensions, its neighbour row x + 1
        const float f = S.result[j + x + (lane & 1)].y;
        const bool on = j + x + (lane & 1) < p.rows;
#pragma unroll
        for (int m = 0; m < 4; ++m)
          if (m < quarters) {
            const float a = __uint_as_float(o[16 * m + x]), b = __uint_as_float(o[16 * m + x + 1]);
            const float got = __shfl_xor_sync(0xffffffffu, lane & 1 ? a : b, 1) * f, keep = (lane & 1 ? b : a) * f;
            if (on) *reinterpret_cast<uint32_t*>(out + 128 * m) = lane & 1 ? Pair<T>::r(got, keep) : Pair<T>::r(keep, got);
          }
        out += 2 * A.rank;
      }
    } else if (fits) {
      float* out = P.part_o + (static_cast<long long>(slot) * N + j) * A.rank + me;
#pragma unroll
      for (int x = 0; x < 16; ++x, out += A.rank)
        if (j + x < p.rows) {
#pragma unroll
          for (int m = 0; m < 4; ++m)
            if (m < quarters) out[128 * m] = __uint_as_float(o[16 * m + x]);
        }
    }
  }
  tc_fence_before_sync();
  __syncwarp();
  if (lane == 0) {
    mbar_arrive(&S.r_free);
    mbar_arrive(&S.o_free[piece % kOs]);
  }
}

// ---- the warps that feed: tiles by TMA, the two products -----------------------------------------------
template <int N>
__device__ __forceinline__ void load_tiles(Smem<N>& S, const Args& P, const Start& start) {
  constexpr int kLatent = Ring<N>::kLatent, kRopes = Ring<N>::kRopes;
  const gemq_latent_decode_t& A = P.a;
  const int lane = threadIdx.x & 31, blocks = A.rank / 64;
  int* const err = A.err;
  Walk<N> walk(P, start);
  Piece p;
  int place = 0, freed = 0;  // next latent block of the ring; tiles known to be done
  uint32_t k = 0, phase = 1;
  const bool small = A.page_size < kTile;
  const int per_tile = small ? kTile / A.page_size : 1, quarters = small ? A.page_size / 16 : 4, tiles_a_page = small ? 1 : A.page_size / kTile;
  const int box_rows = min(A.page_size, kTile), page_bits = A.page_size == 16 ? 4 : 5;  // of small pages
  const uint32_t ring0 = smem_u32(S.ring[0]), rope0 = smem_u32(S.rope[0]), full0 = smem_u32(&S.full[0]), rope_full0 = smem_u32(&S.rope_full[0]);
  int rope_at = 0;
  while (walk.next(p)) {
    const bool prefix = p.e < A.groups;
    const int* table = prefix ? A.prefix_table + static_cast<long long>(p.e) * A.prefix_pitch
                              : A.table + static_cast<long long>(p.e - A.groups) * A.table_pitch;
    const int pitch = prefix ? A.prefix_pitch : A.table_pitch;
    int pg = small ? p.t0 * per_tile : tiles_a_page == 1 ? p.t0 : p.t0 / tiles_a_page, row = small ? 0 : (p.t0 - pg * tiles_a_page) * kTile;
    int base = pg, ids = base + lane < pitch ? table[base + lane] : 0;  // lane i has the id of page base + i
    for (int i = 0; i < p.n; ++i, ++k) {
      const int here = small ? (min(p.x.len - (p.t0 + i) * kTile, kTile) + A.page_size - 1) >> page_bits : 1;  // pages of the tile
      if (pg + here > base + 32) {
        base = pg;
        ids = base + lane < pitch ? table[base + lane] : 0;
      }
      const bool out = ids < 0 || ids >= A.n_pages;
      const uint32_t outs = __ballot_sync(0xffffffffu, out) >> (pg - base);
      int bad = 0;
      for (int j = 0; j < here; ++j)
        if ((outs >> j) & 1) bad |= ((1 << quarters) - 1) << (j * quarters);
      if (lane == 0) {
        S.bad[k % kSlots] = bad;
        mbar_arrive(&S.told[k % kSlots]);
        if (bad) atomicExch(err, GEMQ_LATENT_BAD_PAGE);
      }
      const uint32_t bytes = here * box_rows * 128;
      if (!small) {
        const int id = __shfl_sync(0xffffffffu, out ? 0 : ids, pg - base);
        for (int d = 0; d < blocks; d += 2) {
          wait_for<N != 64>(&S.empty[place >> 1], phase, &S.abort, err);
          if (elect_lane()) {
            mbar_expect_at(full0 + place * 4, 2 * kBlock);
            tma_load_4d_at(ring0 + place * kBlock, &P.latent_map, row, d, id, full0 + place * 4);
          }
          __syncwarp();
          place += 2;
          if (place == kLatent) { place = 0; phase ^= 1; }
        }
        if (static_cast<int>(k) >= kRopes + freed) {
          wait_for<N != 64>(&S.done[freed % kSlots], (freed / kSlots) & 1, &S.abort, err);
          ++freed;
        }
        if (elect_lane()) {
          mbar_expect_at(rope_full0 + rope_at * 8, kBlock);
          tma_load_4d_at(rope0 + rope_at * kBlock, &P.rope_map, row, blocks, id, rope_full0 + rope_at * 8);
        }
        __syncwarp();
      } else {
        int id[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) id[j] = __shfl_sync(0xffffffffu, out ? 0 : ids, (pg - base + j) & 31);
        const uint32_t page_bytes = A.page_size * 128;
        for (int d = 0; d < blocks; d += 2) {
          wait_for<N != 64>(&S.empty[place >> 1], phase, &S.abort, err);
          const uint32_t dst = ring0 + place * kBlock, bar = full0 + place * 4;
          if (elect_lane()) {
            mbar_expect_at(bar, 2 * bytes);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (j < here) {
                tma_load_4d_at(dst + j * page_bytes, &P.latent_map, 0, d, id[j], bar);
                tma_load_4d_at(dst + kBlock + j * page_bytes, &P.latent_map, 0, d + 1, id[j], bar);
              }
          }
          __syncwarp();
          place += 2;
          if (place == kLatent) { place = 0; phase ^= 1; }
        }
        if (static_cast<int>(k) >= kRopes + freed) {
          wait_for<N != 64>(&S.done[freed % kSlots], (freed / kSlots) & 1, &S.abort, err);
          ++freed;
        }
        if (elect_lane()) {
          mbar_expect_at(rope_full0 + rope_at * 8, bytes);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j < here) tma_load_4d_at(rope0 + rope_at * kBlock + j * page_bytes, &P.rope_map, 0, blocks, id[j], rope_full0 + rope_at * 8);
        }
        __syncwarp();
      }
      if (++rope_at == kRopes) rope_at = 0;
      if (small) {
        pg += per_tile;
      } else {
        row += kTile;
        if (row == A.page_size) { row = 0; ++pg; }
      }
    }
  }
  // The copies in flight end before the CTA does: the MMAs of the last tile waited for them, unless a wait ran out.
  if (*reinterpret_cast<volatile int*>(&S.abort))
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
}

// S.  The whole warp runs the loop and one elected lane issues: descriptors stay in uniform registers.
template <typename T, int N>
__device__ __forceinline__ void score_tiles(Smem<N>& S, const Args& P, const Start& start, uint32_t tmem) {
  constexpr int kLatent = Ring<N>::kLatent, kRopes = Ring<N>::kRopes;
  const gemq_latent_decode_t& A = P.a;
  const int blocks = A.rank / 64;
  int* const err = A.err;
  Walk<N> walk(P, start);
  Piece p;
  const uint64_t q0 = umma_desc_k_sw128(smem_u32(S.q[0])), ring0 = umma_desc_k_sw128(smem_u32(S.ring[0])),
                 rope0 = umma_desc_k_sw128(smem_u32(S.rope[0]));
  uint32_t k = 0, phase = 0, rope_at = 0, rope_phase = 0;
  int place = 0;
  for (uint32_t piece = 0; walk.next(p); ++piece) {
    const uint32_t idesc = umma_idesc_f16(Pair<T>::kBf16, kTile, p.width());
    wait_for<N != 64>(&S.q_full, piece & 1, &S.abort, err);
    for (int i = 0; i < p.n; ++i, ++k) {
      wait_for<N != 64>(&S.s_free[k & 1], ((k >> 1) & 1) ^ 1, &S.abort, err);
      const uint32_t s = tmem + (k & 1) * N;
      for (int d = 0; d < blocks; d += 2) {
        wait_for<N != 64>(&S.full[place >> 1], phase, &S.abort, err);
        tc_fence_after_sync();
        const uint64_t a = ring0 + place * (kBlock >> 4), b = q0 + d * (N * 128 >> 4);
        if (elect_lane()) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            umma_ss_f16(s, a + (j >> 2) * (kBlock >> 4) + (j & 3) * 2, b + (j >> 2) * (N * 128 >> 4) + (j & 3) * 2, idesc, d != 0 || j != 0);
        }
        __syncwarp();
        place += 2;
        if (place == kLatent) { place = 0; phase ^= 1; }
      }
      wait_for<N != 64>(&S.rope_full[rope_at], rope_phase, &S.abort, err);
      tc_fence_after_sync();
      const uint64_t a = rope0 + rope_at * (kBlock >> 4), b = q0 + blocks * (N * 128 >> 4);
      if (elect_lane()) {
#pragma unroll
        for (int j = 0; j < 4; ++j) umma_ss_f16(s, a + j * 2, b + j * 2, idesc, 1);
        umma_commit(&S.s_full[k & 1]);
        if (i == p.n - 1) umma_commit(&S.q_free);
      }
      __syncwarp();
      if (++rope_at == kRopes) { rope_at = 0; rope_phase ^= 1; }
    }
  }
}

// O.
template <typename T, int N>
__device__ __forceinline__ void sum_tiles(Smem<N>& S, const Args& P, const Start& start, uint32_t sums) {
  constexpr int kLatent = Ring<N>::kLatent, kOs = Smem<N>::kOs;
  const gemq_latent_decode_t& A = P.a;
  const int blocks = A.rank / 64;
  int* const err = A.err;
  Walk<N> walk(P, start);
  Piece p;
  const uint64_t p0 = umma_desc_k_sw128(smem_u32(S.p)), ring0 = umma_desc_mn_sw128(smem_u32(S.ring[0]), kBlock);
  uint32_t k = 0;
  int place = 0;
  for (uint32_t piece = 0; walk.next(p); ++piece) {
    const uint32_t idesc = umma_idesc_f16(Pair<T>::kBf16, 128, p.width()) | kUmmaTransposeA;
    const uint32_t acc = sums + piece % kOs * (4 * N);
    wait_for<N != 64>(&S.o_free[piece % kOs], ((piece / kOs) & 1) ^ 1, &S.abort, err);
    for (int i = 0; i < p.n; ++i, ++k) {
      const int steps = cdiv(min(p.x.len - (p.t0 + i) * kTile, kTile), 16);  // of 16 positions
      wait_for<N != 64>(&S.p_full, k & 1, &S.abort, err);
      tc_fence_after_sync();
      // a pair of blocks is free behind its MMAs: S of the tile is complete
      for (int m = 0; m < blocks / 2; ++m) {
        const uint64_t a = ring0 + place * (kBlock >> 4);
        const uint32_t o = acc + m * N;
        if (elect_lane()) {
          umma_ss_f16(o, a, p0, idesc, i != 0);
          if (steps == 4) {
#pragma unroll
            for (int s = 1; s < 4; ++s) umma_ss_f16(o, a + s * (2048 >> 4), p0 + s * (32 >> 4), idesc, 1);
          } else {
            for (int s = 1; s < steps; ++s) umma_ss_f16(o, a + s * (2048 >> 4), p0 + s * (32 >> 4), idesc, 1);
          }
          umma_commit(&S.empty[place >> 1]);
        }
        __syncwarp();
        place = place + 2 == kLatent ? 0 : place + 2;
      }
      if (elect_lane()) {
        umma_commit(&S.done[k % kSlots]);
        if (i == p.n - 1) umma_commit(&S.o_full[piece % kOs]);
      }
      __syncwarp();
    }
  }
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads, 1) latent_decode_kernel(const __grid_constant__ Args P) {
  constexpr int kLatent = Ring<N>::kLatent, kRopes = Ring<N>::kRopes;
  constexpr uint32_t kTmemCols = N == 16 ? 256 : 512;
  constexpr uint32_t kTmemO = 2 * N;
  constexpr int kOs = Smem<N>::kOs;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  Smem<N>& S = *reinterpret_cast<Smem<N>*>(smem_raw);
  const gemq_latent_decode_t& A = P.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kLatent / 2; ++i) { mbar_init(&S.full[i], 1); mbar_init(&S.empty[i], 1); }
    for (int i = 0; i < kRopes; ++i) mbar_init(&S.rope_full[i], 1);
    for (int i = 0; i < kSlots; ++i) { mbar_init(&S.done[i], 1); mbar_init(&S.told[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&S.s_full[i], 1); mbar_init(&S.s_free[i], 4); }
    mbar_init(&S.p_full, 4);
    mbar_init(&S.q_full, 4);
    mbar_init(&S.q_free, 1);
    for (int i = 0; i < kOs; ++i) { mbar_init(&S.o_full[i], 1); mbar_init(&S.o_free[i], 4); }
    mbar_init(&S.r_full, 4);
    mbar_init(&S.r_free, 4);
    S.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&S.tmem_base, kTmemCols);
  if (warp == 0 && lane < 2) prefetch_map(lane ? &P.rope_map : &P.latent_map);
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // Every CTA adds up the list.  Up to 32 entries each warp does, a lane an entry, and knows the CTA's share without another word.  More: a thread
  // has a run of them and the sums meet in shared memory (one sequence of 700 rows: 13.1 us that way, 11.4 this way; 37 sequences with two
  // entries a lane: no gain).
  const int entries = A.groups + A.batch, c = blockIdx.x;
  Start start = {0, 0, 0, 0, 0, 0, {0, 0, 0, 0, 0, 0}};
  auto share = [&](int total, bool wrong) {
    const Cut cut(wrong ? 0 : total, gridDim.x);
    if (c < cut.ctas) {
      start.from = cut.from(c);
      start.to = cut.from(c + 1);
    }
    if (c == 0 && threadIdx.x == 0) {
      P.ctl[0] = wrong ? -1 : total;
      if (wrong) atomicExch(A.err, GEMQ_LATENT_BAD_LENGTH);
    }
  };
  constexpr int kFew = 32;
  if (entries <= kFew) {
    Entry x = start.x;
    if (lane < entries) x = entry_here(P, lane);
    const int n = cdiv(x.rows, N);
    int upto = n * x.cost, rts = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, upto, d), b = __shfl_up_sync(0xffffffffu, rts, d);
      if (lane >= d) { upto += a; rts += b; }
    }
    share(__shfl_sync(0xffffffffu, upto, 31), A.groups > 0 && __any_sync(0xffffffffu, lane < A.groups && start_wrong(A, lane)));
    const int begin = upto - n * x.cost;
    rts -= n;
    if (c == 0 && warp == 0 && lane < entries) {
      P.ctl[2 + 2 * lane] = begin;
      P.ctl[3 + 2 * lane] = rts;
    }
    if (start.from < start.to) {
      const int who = __ffs(__ballot_sync(0xffffffffu, start.from >= begin && start.from < upto)) - 1;
      auto of = [&](int v) { return __shfl_sync(0xffffffffu, v, who); };
      start.x = {of(x.len), of(x.tiles), of(x.row0), of(x.rows), of(x.piece), of(x.cost)};
      start.e = who;
      start.base = of(begin);
      start.rto = of(rts);
      if (start.x.rows > N) {
        start.rt = (start.from - start.base) / start.x.cost;
        start.base += start.rt * start.x.cost;
      }
    }
  }
  int cost = 0, rts = 0, before = 0, rts_before = 0;
  bool wrong = false;
  const int run = cdiv(entries, kThreads);
  if (entries > kFew) {
    for (int k = 0; k < run; ++k) {
      const int e = static_cast<int>(threadIdx.x) * run + k;
      if (e >= entries) break;
      if (e < A.groups) wrong = wrong || start_wrong(A, e);
      const Entry x = entry_of(P, e);
      const int n = cdiv(x.rows, N);
      cost += n * x.cost;
      rts += n;
    }
    before = cost;
    rts_before = rts;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, before, d), b = __shfl_up_sync(0xffffffffu, rts_before, d);
      if (lane >= d) { before += a; rts_before += b; }
    }
    if (lane == 31) { S.sums[warp][0] = before; S.sums[warp][1] = rts_before; }
  }
  tc_fence_before_sync();
  if (entries <= kFew || A.groups == 0) __syncthreads();
  else wrong = __syncthreads_or(wrong);
  tc_fence_after_sync();
  // Only now: a CTA of the next kernel must not take this SM's tensor memory first.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (entries > kFew) {
    before -= cost;
    rts_before -= rts;
    int total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) { before += S.sums[w][0]; rts_before += S.sums[w][1]; }
      total += S.sums[w][0];
    }
    share(total, wrong);
    if (c == 0 || (start.from >= before && start.from < before + cost)) {
      int at = before, rto = rts_before;
      for (int k = 0; k < run; ++k) {
        const int e = static_cast<int>(threadIdx.x) * run + k;
        if (e >= entries) break;
        const Entry x = entry_of(P, e);
        const int n = cdiv(x.rows, N), all = n * x.cost;
        if (c == 0) {
          P.ctl[2 + 2 * e] = at;
          P.ctl[3 + 2 * e] = rto;
        }
        if (start.from >= at && start.from < at + all) {
          const int rt = (start.from - at) / x.cost;
          S.start = {e, rt, at + rt * x.cost, start.from, start.to, rto, x};
        }
        at += all;
        rto += n;
      }
    }
    __syncthreads();
    if (start.from < start.to) start = S.start;
  }
  const uint32_t tmem = S.tmem_base;
  // 64 rows of queries: 240 registers for the softmax warps; with the others' 88 and 168 below the launch's 3 x 168
  if (warp < kSoftWarp) {
    if (N == 64) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 0) load_tiles<N>(S, P, start);
    else if (warp == 1) score_tiles<T, N>(S, P, start, tmem);
    else if (warp == 2) sum_tiles<T, N>(S, P, start, tmem + kTmemO);
  } else if (warp >= kEdgeWarp) {
    Walk<N> ahead(P, start), walk(P, start);
    Piece q, p;
    uint32_t loads = 0;
    if (ahead.next(q)) load_queries<T, N>(S, P, q, loads++);
    for (uint32_t piece = 0; walk.next(p); ++piece) {
      if (ahead.next(q)) load_queries<T, N>(S, P, q, loads++);
      finish_piece<T, N>(S, P, p, piece, tmem + kTmemO + piece % kOs * (4 * N));
    }
  } else {
    if (N == 64) asm volatile("setmaxnreg.inc.sync.aligned.u32 240;");
    Walk<N, N != 64> walk(P, start);
    Piece p;
    uint32_t k = 0;
    for (uint32_t piece = 0; walk.next(p); ++piece) {
      const uint32_t acc = tmem + kTmemO + piece % kOs * (4 * N);
      if (N == 16 || p.rows <= 16) softmax_piece<T, N, 16>(S, P, p, k, piece, tmem, acc);
      else if (N == 32 || p.rows <= 32) softmax_piece<T, N, N < 32 ? 16 : 32>(S, P, p, k, piece, tmem, acc);
      else if (p.rows <= 48) softmax_piece<T, N, N < 64 ? 16 : 48>(S, P, p, k, piece, tmem, acc);
      else softmax_piece<T, N, N < 64 ? 16 : 64>(S, P, p, k, piece, tmem, acc);
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
// A warp has 128 numbers of a row, eight pieces in flight.  Many rows have few pieces each (W = 1): a CTA has a row, and its warps all pieces of
// their numbers.  Few rows may have a piece from every CTA (W = 8): a CTA has 128 numbers, its warps take every eighth piece and keep a maximum
// of their own; the eight are added in a fixed order.  What decides is the pieces a row, which only the device knows; the rows of the batch stand in
// for it: up to two a CTA take W = 8.  Measured, the call in a graph, 16 heads, W = 8 against W = 1: one sequence of 200,000 positions 52 and 81 us;
// 20,000 positions in 4 equal ones 14.6 and 22.2, in 9 17.8 and 19.5, in 18 22.1 and 17.7, in 37 30.6 and 17.5; one of 131,072 beside 19 of 200
// 43 and 70.  Equal lengths alone would put the line at 10 sequences; it stands where a batch of 18 loses 4 us if they are equal and gains 27 if one
// of them is long.
constexpr int kJoinAhead = 8;

template <typename T, int W>
__global__ void __launch_bounds__(W == 1 ? 128 : 32 * W, W == 1 ? 6 : 2) latent_join_kernel(const __grid_constant__ Args P, int N, int sms) {
  __shared__ float4 part[W][32];
  __shared__ float2 part_ml[W];
  const gemq_latent_decode_t& A = P.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, cuts = A.rank / 128;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // Ahead of every read, those of the inputs too: what kernels before have written is visible behind a wait of the reader.  (Lengths and starts
  // read ahead of it: 0.3 us less, 0.6 with prefixes.)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int total = P.ctl[0];
  const bool sound = total >= 0;
  const int per_row = W == 1 ? 1 : cuts, bits = 31 - __clz(N);
  const Find cut(total, sms);
  for (int job = blockIdx.x; job < A.batch * A.steps * A.heads * per_row; job += gridDim.x) {
    const int row = W == 1 ? job : cuts == 4 ? job >> 2 : job / cuts, at4 = (W == 1 ? warp : job - row * cuts) * 32 + lane;
    const Row q(P, row);
    const int b = q.b, hidden = A.steps - 1 - q.i;
    const int2 own = *reinterpret_cast<const int2*>(P.ctl + 2 + 2 * (A.groups + b));  // asked for beside the length
    int g = -1, len = 0;
    Entry x[2];
    x[0] = {0, 0, 0, 0, 0, 0};
    if (A.groups > 0) {
      int hi = A.groups;  // the last group that begins at b or before (g < hi)
      for (g = 0; hi - g > 1;) {
        const int mid = (g + hi) >> 1;
        if (start_of(A, mid) <= b) g = mid;
        else hi = mid;
      }
      x[0] = entry_here(P, g);
      if (row < x[0].row0 || row >= x[0].row0 + x[0].rows) x[0].tiles = 0;
      else len = x[0].len;
    }
    x[1] = entry_here(P, A.groups + b);
    len += x[1].len;
    int rt[2] = {0, 0}, first[2] = {0, 0}, count[2] = {0, 0}, at[2] = {0, 0};  // runs of pieces: of the group's prefix, of the sequence's own tiles
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (x[k].tiles > 0 && sound) {
        const int2 list = k ? own : *reinterpret_cast<const int2*>(P.ctl + 2 + 2 * g);
        const int r = row - x[k].row0, base = list.x + (r >> bits) * x[k].cost;
        const int c0 = cut.cta_of(base + x[k].piece), c1 = cut.cta_of(base + x[k].piece + 4 * (x[k].tiles - 1));
        rt[k] = list.y + (r >> bits);
        first[k] = c0;
        count[k] = c1 - c0 + 1;
        at[k] = r & (N - 1);
      }
    }
    if (A.groups == 0 && count[1] == 1) continue;  // written already
    const int pieces = count[0] + count[1];
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = sound ? 0.f : __int_as_float(0x7fc00000), top = -INFINITY;
    if (W == 1 && warp >= cuts) continue;
    for (int i0 = W == 1 ? 0 : warp; i0 < pieces; i0 += W * kJoinAhead) {
      float4 v[kJoinAhead];
      float2 ml[kJoinAhead];
#pragma unroll
      for (int k = 0; k < kJoinAhead; ++k) {
        const int i = i0 + W * k;
        const int s = i < count[0] ? slot_of(true, rt[0], first[0] + i, false)
                                   : slot_of(A.groups > 0, rt[1], first[1] + i - count[0], i == pieces - 1);
        ml[k] = make_float2(-INFINITY, 0.f);
        v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < pieces && static_cast<unsigned>(s) < static_cast<unsigned>(P.slots)) {
          const long long from = static_cast<long long>(s) * N + (i < count[0] ? at[0] : at[1]);
          ml[k] = P.part_ml[from];
          v[k] = reinterpret_cast<const float4*>(P.part_o + from * A.rank)[at4];
        }
      }
      float now = top;
#pragma unroll
      for (int k = 0; k < kJoinAhead; ++k) now = fmaxf(now, ml[k].x);
      const float base = now == -INFINITY ? 0.f : now, f0 = exp2_fast(top - base);
      top = now;
      l *= f0;
      o = make_float4(o.x * f0, o.y * f0, o.z * f0, o.w * f0);
#pragma unroll
      for (int k = 0; k < kJoinAhead; ++k) {
        const float f = exp2_fast(ml[k].x - base);
        l = fmaf(ml[k].y, f, l);
        o.x = fmaf(v[k].x, f, o.x);
        o.y = fmaf(v[k].y, f, o.y);
        o.z = fmaf(v[k].z, f, o.z);
        o.w = fmaf(v[k].w, f, o.w);
      }
    }
    if (W > 1) {
      part[warp][lane] = o;
      if (lane == 0) part_ml[warp] = make_float2(top, l);
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int w = 1; w < W; ++w) top = fmaxf(top, part_ml[w].x);
        const float base = top == -INFINITY ? 0.f : top;
        o = make_float4(0.f, 0.f, 0.f, 0.f);
        l = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float4 v = part[w][lane];
          const float f = exp2_fast(part_ml[w].x - base);
          l = fmaf(part_ml[w].y, f, l);
          o.x = fmaf(v.x, f, o.x);
          o.y = fmaf(v.y, f, o.y);
          o.z = fmaf(v.z, f, o.z);
          o.w = fmaf(v.w, f, o.w);
        }
      }
    }
    if (W == 1 || warp == 0) {
      const bool empty = len - hidden <= 0 && sound;
      const float f = 1.f / l;
      reinterpret_cast<uint2*>(static_cast<T*>(A.out) + static_cast<long long>(row) * A.rank)[at4] =
          empty ? make_uint2(0, 0) : make_uint2(Pair<T>::r(o.x * f, o.y * f), Pair<T>::r(o.z * f, o.w * f));
      if (at4 == 0) A.lse[row] = empty ? -INFINITY : (top + log2f(l)) * kLn2;
    }
    if (W > 1) __syncthreads();
  }
}

int check(const gemq_latent_decode_t* A) {
  if (!A || !A->q_latent || !A->q_rope || !A->cache || !A->table || !A->lens || !A->out || !A->lse || !A->err) return GEMQ_ERR_BAD_ARG;
  if (A->batch < 0 || A->steps <= 0 || A->heads <= 0 || A->n_pages <= 0 || A->table_pitch < 0 || A->groups < 0) return GEMQ_ERR_BAD_ARG;
  if (A->groups && (!A->prefix_table || !A->prefix_lens || !A->starts || A->prefix_pitch < 0)) return GEMQ_ERR_BAD_ARG;
  if (!rank_ok(A->rank) || !page_ok(A->page_size)) return GEMQ_ERR_BAD_SHAPE;
  const long long rows = static_cast<long long>(A->batch) * A->steps * A->heads;
  if (rows > (1 << 28) || A->groups > (1 << 24)) return GEMQ_ERR_BAD_SHAPE;
  // the list of work is counted in 32 bits
  const long long own = static_cast<long long>(A->table_pitch) * A->page_size, pre = static_cast<long long>(A->prefix_pitch) * A->page_size;
  const long long tiles = (rows / 16 + A->batch) * (own / kTile + 2) + (A->groups ? (rows / 16 + A->groups) * (pre / kTile + 2) : 0);
  if (own > 0x7fffff00 || pre > 0x7fffff00 || tiles > 0x7fffffff / 8) return GEMQ_ERR_BAD_SHAPE;
  if (!aligned16(A->q_latent) || !aligned16(A->q_rope) || !aligned16(A->cache) || !aligned16(A->out) || (A->page_stride & 7))
    return GEMQ_ERR_ALIGN;
  for (int i = 0; i < 3; ++i)
    if ((A->q_latent_stride[i] | A->q_rope_stride[i]) & 7) return GEMQ_ERR_ALIGN;
  if (A->n_pages > 1 && A->page_stride < static_cast<int64_t>(A->page_size) * (A->rank + kRope)) return GEMQ_ERR_BAD_SHAPE;
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
  s.slots = static_cast<int>(A->groups ? rts + sm_count_or_default() : 2 * sm_count_or_default());
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
  const long long rows = static_cast<long long>(P.a.batch) * P.a.steps * P.a.heads, most = 16ll * ctas;
  const bool few = rows <= 2 * ctas;
  const long long jobs = few ? rows * (P.a.rank / 128) : rows;
  cfg.gridDim = dim3(static_cast<unsigned>(jobs < most ? jobs : most));
  cfg.blockDim = dim3(few ? 256 : 128);
  cfg.dynamicSmemBytes = 0;
  const cudaError_t e = few ? cudaLaunchKernelEx(&cfg, latent_join_kernel<T, 8>, P, N, ctas) : cudaLaunchKernelEx(&cfg, latent_join_kernel<T, 1>, P, N, ctas);
  return e == cudaSuccess ? GEMQ_OK : GEMQ_ERR_LAUNCH;
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
  P.per = div_by(A->steps * A->heads);
  P.heads = div_by(A->heads);
  const int rows = A->page_size < kTile ? A->page_size : kTile;
  const int blocks = A->rank / 64 + 1;
  if (!tensor_map_pages(&P.latent_map, A->cache, blocks, A->page_size, A->page_stride, A->n_pages, rows, A->page_size < kTile ? 1 : 2) ||
      !tensor_map_pages(&P.rope_map, A->cache, blocks, A->page_size, A->page_stride, A->n_pages, rows, 1))
    return GEMQ_ERR_LAUNCH;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int N = row_tile(A);
  return A->is_bf16 ? launch<__nv_bfloat16>(P, N, sms, st) : launch<__half>(P, N, sms, st);
}
