// What the attention kernels with a window and sinks share (gdn_window.hip: whole sequences with their backward;
// gdn_paged.hip: a paged cache): which keys a query sees, the walk of sequences in tiles, tiles of rows in LDS, the
// softmax of a block, and the rows that are computed one by one where infinities or NaN lie in places they must not see.
//
//   A query at place i of its sequence sees key j iff j <= i and (i - j < window or j < sinks).
//
// v_mfma_f32_32x32x16 layouts (lane = 32 hh + li): A lane holds row li, k = 8 hh .. 8 hh + 7; B lane column li, same k;
// the accumulator's element e of a lane is column li, row 8 (e / 4) + 4 hh + e % 4.
#pragma once

#include "gdn_mfma.h"

namespace gdn {

// lift: the weights' exponent at the running maximum. fp16's lie 2^7 higher, so that those as far as 2^8 above the maximum still
// fit: below 2^-14 a weight keeps fewer bits, and a row that gives most of its sum to one key has many small ones.
template <typename E> struct Pack;
template <> struct Pack<bf16> { using x8 = bf16x8; using x4 = bf16x4; static constexpr float lift = 0.f; static constexpr uint16_t infinity = 0x7f80; };
template <> struct Pack<f16> { using x8 = f16x8; using x4 = f16x4; static constexpr float lift = 7.f; static constexpr uint16_t infinity = 0x7c00; };

__device__ __forceinline__ f32x16 mma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ int64_t uniform64(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)x), hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)((uint64_t)x >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}
template <typename F>
__device__ __forceinline__ int lanes_of(F yes) {
  return __popcll(__ballot(yes((int)(threadIdx.x % kWave))));
}

}  // namespace gdn

#include "gdn_flash_walk.h"

namespace gdn {

constexpr int64_t kMaxRowBytes = 1 << 24;  // bytes between two tokens of an operand read through 32-bit offsets inside a block

// ------------------------------------------------------------------------------------------------ tiles in LDS
// Rows of D elements lie unpadded (a load straight into LDS fills 1 KB contiguously); the 16-byte chunk c of row r is stored
// at chunk c ^ swz(r), which keeps both the row fragments' and the transposed reads free of bank conflicts.
template <int D>
__device__ __forceinline__ int swz(int r) {
  return D == 128 ? (((r & 3) << 2) | ((r >> 2) & 3)) : (((r & 3) << 1) | ((r >> 2) & 1));
}

// Where a lane reads a tile: the XOR of a chunk number is the XOR of the address, so that three registers hold all of them.
template <int D>
struct TileReads {
  int row, tr0, tr1;
  __device__ __forceinline__ void init(int lane) {
    const int hh = lane >> 5, li = lane & 31, gsub = (lane >> 4) & 1, lm = (lane & 15) >> 2, lq = lane & 3;
    row = li * D + ((hh ^ swz<D>(li)) << 3);
    const int r = 4 * hh + lm, ch = 2 * gsub + (lq >> 1);
    tr0 = r * D + ((ch ^ swz<D>(r)) << 3) + 4 * (lq & 1);
    tr1 = (r + 8) * D + ((ch ^ swz<D>(r + 8)) << 3) + 4 * (lq & 1);
  }
  // the same, with the addresses made where they are used instead of being kept in registers over a loop
  __device__ __forceinline__ TileReads here() const { return TileReads{opaque_int(row), opaque_int(tr0), opaque_int(tr1)}; }
};

// A operand: row li of the 32 from `tile`, k-step st
template <int D, typename E>
__device__ __forceinline__ typename Pack<E>::x8 row_frag(const E* tile, const TileReads<D>& rd, int st) {
  return *reinterpret_cast<const typename Pack<E>::x8*>(tile + (rd.row ^ (16 * st)));
}
// A operand of the transposed 16 rows from `tile`: lane li holds column 32 d + li, k in the order 4 hh + r, 8 + 4 hh + r, which
// is the accumulator's own row order
template <int D, typename E>
__device__ __forceinline__ typename Pack<E>::x8 tr_frag(const E* tile, const TileReads<D>& rd, int d) {
  const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(tile + (rd.tr0 ^ (32 * d))));
  const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(tile + (rd.tr1 ^ (32 * d))));
  return __builtin_bit_cast(typename Pack<E>::x8, bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
}

// 16 accumulator elements as the two B operands of their 32 rows
template <typename E>
__device__ __forceinline__ void pack16(const f32x16& s, typename Pack<E>::x8 (&out)[2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 8; ++e) out[h][e] = (E)s[8 * h + e];
}

// One 16-byte load a lane straight into LDS (lane l's at `to` + 16 l bytes).
__device__ __forceinline__ void load_lds16(__amdgpu_buffer_rsrc_t r, void* to, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)to, 16, off, 0, 0, 0);
}
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0F70); }  // vmcnt(0)

// ------------------------------------------------------------------------------------------------ softmax
// Online softmax of KT x 32 keys of the wave's 32 queries (raw scores s, masked ones -inf) and O^T += V^T P^T.
// p = 2^(s c - m c + lift), c = scale log2(e) > 0. The row's m moves only when a block's maximum exceeds it by more than `slack` =
// 8 / c: p <= 2^(8 + lift) meanwhile, which costs no precision, and O^T is rescaled rarely. A row that saw no key yet keeps
// m = -inf and uses 0. P is rounded to the inputs' type for the product: off by half a step of it a term, as the output itself is,
// or in fp16 by 2^-32 of the row's sum. The row sum adds p in fp32, so that the backward's logarithm of it is exact to fp32. The
// sum of a row that saw a key whose score is above -inf is 2^lift at least.
template <int KT, int D, typename E>
__device__ __forceinline__ void softmax_step(f32x16 (&s)[KT], f32x16 (&acc)[D / 32], float& m, float& l, float c, float slack,
                                             const E* vb, const TileReads<D>& rd) {
  float mx = -INFINITY;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[kt][e]);
  mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
  const bool grow = mx > m + slack;
  if (!__all(!grow)) {
    const float alpha = grow ? __builtin_amdgcn_exp2f((m - mx) * c) : 1.f;  // 0 while no key was seen
    m = grow ? mx : m;
    l *= alpha;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) acc[d] *= alpha;
  }
  const float nmc = m == -INFINITY ? 0.f : Pack<E>::lift - m * c;
  float sum = 0.f;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[kt][e] = __builtin_amdgcn_exp2f(fmaf(s[kt][e], c, nmc));
      sum += s[kt][e];
    }
  }
  l += sum;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    typename Pack<E>::x8 pb[2];
    pack16<E>(s[kt], pb);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int d = 0; d < D / 32; ++d) acc[d] = mma32(tr_frag(vb + (2 * kt + h) * 16 * D, rd, d), pb[h], acc[d]);
  }
  __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);  // the fragments' reads two products ahead
#pragma unroll
  for (int i = 0; i < 2 * KT * (D / 32) - 2; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
}

// ------------------------------------------------------------------------------------------------ sums that are not finite
// The matrix products multiply a masked place's weight, 0, with what lies there: an infinity or NaN among the values would
// reach rows that do not see it. And weights of up to 2^8, of any number of keys, times finite values may pass fp32's range before
// they are divided by the row's sum. (Masked scores take part in nothing: the row's maximum and sum are right, and where the sum
// is NaN the row is.) Rows whose sums are not finite are taken again, without the infinities and NaN, which are then added to the
// rows that see them.
__device__ __forceinline__ bool finite_f(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// whether a lane's accumulators are all finite: 0 x stays 0 unless x is not
template <int N>
__device__ __forceinline__ bool finite_all(const f32x16 (&a)[N]) {
  float z = 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int e = 0; e < 16; ++e) z = fmaf(a[n][e], 0.f, z);
  return z == 0.f;
}

// Entries of an A operand that are not finite: x keeps 0 in their place, `up` and `down` hold a 1 where +inf and -inf were, and both
// where NaN was.
template <typename E>
__device__ __forceinline__ void split_infinite(typename Pack<E>::x8& x, typename Pack<E>::x8& up, typename Pack<E>::x8& down) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const bool fine = (__builtin_bit_cast(uint16_t, (E)x[e]) & Pack<E>::infinity) != Pack<E>::infinity;
    up[e] = (E)(fine || x[e] < (E)0.f ? 0.f : 1.f);
    down[e] = (E)(fine || x[e] > (E)0.f ? 0.f : 1.f);
    x[e] = fine ? x[e] : (E)0.f;
  }
}
// They reach the columns of acc that see their rows (`ones`: 1 where seen, a B operand).
template <typename E>
__device__ __forceinline__ void add_infinite(f32x16& acc, typename Pack<E>::x8 up, typename Pack<E>::x8 down, typename Pack<E>::x8 ones) {
  bool any = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) any |= up[e] != (E)0.f || down[e] != (E)0.f;
  if (!__any(any)) return;
  const f32x16 n = mma32(up, ones, f32x16{}), m = mma32(down, ones, f32x16{});
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] += (n[e] > 0.f ? INFINITY : 0.f) - (m[e] > 0.f ? INFINITY : 0.f);
}

// The product with the values again for the wave's rows whose sums are not finite, a block of KT x 32 keys at a time, with weights
// that are divided by the row's sum first (`by`; the maximum is the final one). `seen`: the block's keys that the lane's row sees.
// key(j), val(j): rows of key j of the block, null: none. `tile`: LDS of the wave's own for the values. acc: O^T times 2^raise<E>.
template <typename E>
constexpr float raise = Pack<E>::lift > 0.f ? 14.f : 0.f;  // weights of 1 at most: fp16's are raised as far as they fit
template <int KT, int D, typename E, typename Key, typename Val>
__device__ __forceinline__ void again_block(f32x16 (&acc)[D / 32], const typename Pack<E>::x8 (&qf)[D / 16], uint64_t seen, Key key,
                                            Val val, E* tile, float c, float nmc, float by, const TileReads<D>& rd) {
  using X8 = typename Pack<E>::x8;
  constexpr int CPR = D / 8, RPL = 512 / D;
  const int lane = threadIdx.x % kWave, hh = lane >> 5, li = lane & 31;
#pragma unroll 4
  for (int u = 0; u < KT * 32 / RPL; ++u) {
    const int r = u * RPL + lane / CPR, ch = lane % CPR;
    const E* const v = val(r);
    *reinterpret_cast<X8*>(tile + r * D + ((ch ^ swz<D>(r)) << 3)) = v ? *reinterpret_cast<const X8*>(v + 8 * ch) : X8{};
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    f32x16 s{}, one;
    const E* const k = key(32 * kt + li);
#pragma unroll
    for (int st = 0; st < D / 16; ++st) s = mma32(k ? *reinterpret_cast<const X8*>(k + 16 * st + 8 * hh) : X8{}, qf[st], s);
    const uint32_t bits = (uint32_t)(seen >> 32 * kt) >> 4 * hh;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const bool see = bits >> (8 * (e >> 2) + (e & 3)) & 1;
      s[e] = see ? __builtin_amdgcn_exp2f(fmaf(s[e], c, nmc)) * by : 0.f;
      one[e] = see ? 1.f : 0.f;
    }
    X8 pb[2], ones[2];
    pack16<E>(s, pb);
    pack16<E>(one, ones);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int d = 0; d < D / 32; ++d) {
        X8 x = tr_frag(tile + (2 * kt + h) * 16 * D, rd, d), up, down;
        split_infinite<E>(x, up, down);
        acc[d] = mma32(x, pb[h], acc[d]);
        add_infinite<E>(acc[d], up, down, ones[h]);
      }
  }
  __builtin_amdgcn_wave_barrier();  // the tile is read before the next block's is written
}

// ------------------------------------------------------------------------------------------------ parameters and plans
// Strides in elements; k and v of a paged cache: between pages, tokens of a page, heads.
struct FlashParams {
  const void *q, *k, *v;
  int64_t qsb, qst, qsh, ksb, kst, ksh, vsb, vst, vsh;
  void* o;       // [B, T, HQ, D]
  void* o_rest;  // like o, or null: what o's rounding left, rounded in its turn
  float* lse;    // [HQ, B T] or null: log2 of the sum of 2^(c s)
  Packed seqs;   // cu null: batch rows of T tokens
  int64_t B, tiles;
  int HQ, HKV, parts, window, sinks;
  float scale_log2;
  // paged: the table, the sequences' lengths, and how the work on their keys is cut
  const int* table;
  int64_t table_stride;
  const void* lengths;
  int len_i32, width, shift, pages;
  const int64_t* tree;  // [B, T] bits of the sequence's drafted tokens that each sees, or null
  int64_t tb, tt;
  int splits;
  float* part;          // [tiles HKV][splits][rows a tile][D], then [tiles HKV][splits][2][rows a tile]: O (divided), maximum, sum
};

// Entry `at` of a row of a page table, `at` the same in every lane: through the scalar cache, apart from the vector loads that
// are under way.
__device__ __forceinline__ int page_at(const int* table, int at) {
  typedef const __attribute__((address_space(4))) int* Constant;
  return ((Constant)(uintptr_t)table)[__builtin_amdgcn_readfirstlane(at)];
}

// the sequence's length in the cache, within what its row of the table can hold
__device__ __forceinline__ int cache_length(const void* lengths, int i32, int seq, int width, int shift) {
  const int64_t x = uniform64(load_index(lengths, i32, seq)), most = (int64_t)width << shift;
  return (int)(x < 0 ? 0 : x > most ? most : x);
}

// A tile of ROWS rows (token, q head of the group) of a sequence's new tokens over a kv head of the cache: the blocks of BK
// keys that they see, cut into runs.
struct PagedPlan {
  Seq sq;
  int hkv, row0, rows;     // rows of this tile
  int klen, base;          // keys; place of the first new token
  int first, last;         // places that its rows see from: all of them lie between
  Blocks bl;
  int per, used;           // blocks a run, runs with any
  int64_t job;
};
template <int ROWS, int BK>
__device__ __forceinline__ bool paged_plan(const FlashParams& p, int64_t t, int hkv, PagedPlan& f) {
  const int rep = p.HQ / p.HKV;
  f.job = t * p.HKV + hkv;
  f.hkv = hkv;
  if (p.seqs.cu) {
    f.sq = packed_tile(p.seqs, t, rep, ROWS);
  } else {
    const int64_t per = (p.seqs.T * rep + ROWS - 1) / ROWS, row = t / per;
    f.sq = Seq{row, 0, (int)p.seqs.T, (int)row, (int)(t - row * per)};
  }
  if (f.sq.tile >= kFar / ROWS) return false;
  f.row0 = f.sq.tile * ROWS;
  const int64_t left = (int64_t)f.sq.len * rep - f.row0;
  f.rows = (int)(left < ROWS ? left : ROWS);
  if (f.rows <= 0) return false;
  f.klen = f.sq.num < 0 ? 0 : cache_length(p.lengths, p.len_i32, f.sq.num, p.width, p.shift);
  f.base = f.klen - f.sq.len;
  // a drafted token stands behind as many others as it sees; one that sees none at the committed tokens' end
  f.first = p.tree ? f.base - 1 : f.base + f.row0 / rep;
  f.last = p.tree ? f.klen - 1 : f.base + (f.row0 + f.rows - 1) / rep;
  f.bl = blocks_of<BK>(f.first, f.last, p.window, p.sinks);
  if (f.sq.num < 0) f.bl.count = 0;
  f.per = imax((f.bl.count + p.splits - 1) / p.splits, 4);
  f.used = imax((f.bl.count + f.per - 1) / f.per, 1);
  return true;
}

// bits 0 .. n - 1
__device__ __forceinline__ uint64_t bits_below(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0 : (1ull << n) - 1; }

// What the rounding of x to E left, in 16 bits: with o it is x to 16 bits and more, a 2^-8th of the step that delta is to be free of.
template <typename E>
__device__ __forceinline__ E rest_of(float x) {
  const float r = x - (float)(E)x;
  return (E)(finite_f(r) ? r : 0.f);
}

// What one row sees: a place in the sequence and, for a tree, the drafted tokens' bits.
struct RowView {
  int place, base;  // base: the first drafted token's place; without a tree behind every place
  uint64_t bits;
  __device__ __forceinline__ bool operator()(int j, int window, int sinks) const {
    const int n = j - base;
    const bool by_place = (j <= place) & ((place - j < window) | (j < sinks));
    return ((n < 0) & by_place) | ((n >= 0) & (n < 64) & ((bits >> (n & 63) & 1) != 0));
  }
  // bit x: whether key k0 + x is seen, x = 0 .. 63
  __device__ __forceinline__ uint64_t block(int k0, int window, int sinks) const {
    const int n = k0 - base, at = place - k0;
    const uint64_t by_place = bits_below(at + 1) & (~bits_below(at - window + 1) | bits_below(sinks - k0)) & bits_below(-n);
    const uint64_t drafted = n >= 64 || n <= -64 ? 0 : n >= 0 ? bits >> n : bits << -n;
    return by_place | drafted;
  }
};
__device__ __forceinline__ RowView row_view(const FlashParams& p, const PagedPlan& f, int row) {
  const int token = row / (p.HQ / p.HKV);
  RowView v{f.base + token, kFar, 0};
  if (p.tree) {
    v.base = f.base;
    v.bits = (uint64_t)p.tree[f.sq.row * p.tb + (f.sq.start + token) * p.tt];
    if (f.sq.len < 64) v.bits &= (1ull << f.sq.len) - 1;
    v.place = f.base + __popcll(v.bits) - 1;
  }
  return v;
}

// Whether a row sees any key of the cache. Asked of rows whose sum is 0: with a key all their scores are -inf, and their softmax
// is 0 / 0.
template <int BK>
__device__ __forceinline__ bool sees_any(const FlashParams& p, const PagedPlan& f, const RowView& v) {
  if (f.sq.num < 0) return false;
  const int* const table = p.table + f.sq.num * p.table_stride;
  for (int n = 0; n < f.bl.count; ++n) {
    const int k0 = f.bl.at(n) * BK;
    const uint64_t seen = v.block(k0, p.window, p.sinks) & bits_below(f.klen - k0);
    for (int g = 0; g < BK / 16; ++g) {
      if (!(seen >> 16 * g & 0xffff)) continue;
      const int id = table[(k0 + 16 * g) >> p.shift];
      if (id >= 0 && id < p.pages) return true;
    }
  }
  return false;
}

// ------------------------------------------------------------------------------------------------ forward over whole tiles
constexpr int kBQ = 128;  // rows a workgroup: 32 a wave
constexpr int kBK = 64;   // keys a block

// O = softmax(scale Q K^T) V over the keys that a row sees. A workgroup of 4 waves takes 128 rows, a wave 32 of them in
// registers: queries of one head, or of a paged cache new tokens with the heads of a group. Blocks of 64 keys pass through LDS,
// loaded straight from memory one block ahead. S^T = K Q^T puts one row into each lane's column: maximum, sum and rescaling
// are a lane's own, and P^T is the next product's operand as it is. Bound by the matrix and vector units in turn (its kernels
// give times). Left out after measuring, prompt of 8,192 tokens / piece of 4 x 512: no maximum a block, the sum telling when one is
// needed (93 -> 98, 172 -> 221 us: the whole sum has to be there before the first product with V); the second half's scores
// under the first half's exponentials, and other orders of the instructions (no change); comparisons instead of a word of
// mask bits a lane (256 registers against 196, training step 408 against 391 us).
template <int D, typename E, bool PAGED>
__device__ __forceinline__ void flash_forward(const FlashParams& p, E* Ks0, E* Ks1, E* Vs0, E* Vs1) {
  using X8 = typename Pack<E>::x8;
  using X4 = typename Pack<E>::x4;
  constexpr int DS = D / 16, DT = D / 32, CPR = D / 8, RPL = 512 / D, LPT = kBK / (4 * RPL);
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), hh = lane >> 5, li = lane & 31;
  const int rep = p.HQ / p.HKV;
  Job job;
  PagedPlan f;
  Seq sq;
  int row0, rows, klen, split = 0, n0 = 0, n1;
  Blocks bl;
  const int* table = nullptr;
  RowView view;
  int wq0, wq1;  // places of the wave's first and last row
  if constexpr (PAGED) {
    const int64_t jobs = gridDim.x / p.splits;
    split = (int)(blockIdx.x / jobs);
    if (!job_of(blockIdx.x - split * jobs, p.HKV, 1, p.parts, p.tiles, job)) return;
    // odd runs from the last tile on: workgroups are dealt out in order, so a CU's second one is of another sequence than its
    // first (4 sequences of 2,964 to 8,192 tokens, 512 new ones each: 157 us with the merge, 168 without this)
    const int64_t tile = split & 1 ? p.tiles - 1 - job.tile : job.tile;
    if (!paged_plan<kBQ, kBK>(p, tile, job.hkv, f) || split >= f.used) return;
    sq = f.sq;
    row0 = f.row0;
    rows = f.rows;
    klen = f.klen;
    bl = f.bl;
    n0 = split * f.per;
    n1 = imin(n0 + f.per, bl.count);
    if (sq.num >= 0) table = p.table + sq.num * p.table_stride;
    view = row_view(p, f, row0 + imin(32 * w + li, rows - 1));
    wq0 = p.tree ? f.first : f.base + (row0 + 32 * w) / rep;
    wq1 = p.tree ? f.last : f.base + (row0 + imin(32 * w + 31, rows - 1)) / rep;
  } else {
    if (!job_of(blockIdx.x, p.HKV, rep, p.parts, p.tiles, job)) return;
    if (p.seqs.cu) {
      sq = packed_tile(p.seqs, job.tile, 1, kBQ);
    } else {  // the last tiles, which see most, first
      const int64_t per = (p.seqs.T + kBQ - 1) / kBQ;
      sq = Seq{job.tile % p.B, 0, (int)p.seqs.T, 0, (int)(per - 1 - job.tile / p.B)};
    }
    row0 = sq.tile * kBQ;
    rows = imin(kBQ, sq.len - row0);
    if (rows <= 0) return;
    klen = sq.num < 0 ? 0 : sq.len;
    wq0 = row0 + 32 * w;
    wq1 = row0 + imin(32 * w + 31, rows - 1);
    view = RowView{row0 + imin(32 * w + li, rows - 1), kFar, 0};
    bl = blocks_of<kBK>(row0, row0 + rows - 1, p.window, p.sinks);
    if (sq.num < 0) bl.count = 0;
    n1 = bl.count;
  }
  const bool wave_live = 32 * w < rows, row_ok = 32 * w + li < rows;
  // row r of the tile: which token and q head
  auto token_of = [&](int r) { return PAGED ? (row0 + r) / rep : row0 + r; };
  auto head_of = [&](int r) { return job.hkv * rep + (PAGED ? (row0 + r) % rep : job.hm); };
  auto q_at = [&](int r) {
    return static_cast<const E*>(p.q) + sq.row * p.qsb + (sq.start + token_of(r)) * p.qst + head_of(r) * p.qsh;
  };
  auto o_at = [&](int r) {
    return static_cast<E*>(p.o) + ((sq.row * p.seqs.T + sq.start + token_of(r)) * p.HQ + head_of(r)) * D;
  };
  X8 qf[DS];
  {
    const E* q = q_at(imin(32 * w + li, rows - 1));
#pragma unroll
    for (int s = 0; s < DS; ++s) qf[s] = *reinterpret_cast<const X8*>(q + 16 * s + 8 * hh);
  }

  // load u of wave w fills LDS bytes [(w + 4u) KB, + 1 KB) of a block: rows (w + 4u) RPL + lane / CPR. The lane's chunk does not
  // depend on u.
  const char* const kbase = reinterpret_cast<const char*>(static_cast<const E*>(p.k) + (PAGED ? 0 : sq.row * p.ksb + sq.start * p.kst) + job.hkv * p.ksh);
  const char* const vbase = reinterpret_cast<const char*>(static_cast<const E*>(p.v) + (PAGED ? 0 : sq.row * p.vsb + sq.start * p.vst) + job.hkv * p.vsh);
  const int kst = (int)p.kst * 2, vst = (int)p.vst * 2;  // bytes
  const int drow = w * RPL + lane / CPR, dch = (lane % CPR) ^ swz<D>(drow);
  const int grow = PAGED ? drow & 15 : drow;  // paged: the row inside its 16 keys, which share a page
  const uint32_t koff = (uint32_t)(grow * kst + dch * 16), voff = (uint32_t)(grow * vst + dch * 16);
  int pid[4];  // paged: pages of a block's four groups of 16 keys, -1: none
  auto look_up = [&](int jb) {
    if (!PAGED) return;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int key = jb * kBK + 16 * g, at = key >> p.shift;
      const int id = key < klen ? page_at(table, at) : -1;
      pid[g] = id >= 0 && id < p.pages ? id : -1;
    }
  };
  auto ok_bits = [&]() {
    int b = 15;
    if (PAGED) {
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (pid[g] < 0) b &= ~(1 << g);
    }
    return b;
  };
  auto fetch = [&](int jb, E* kd, E* vd) {
    const int key0 = jb * kBK;
    if (PAGED) {
#pragma unroll
      for (int u = 0; u < LPT; ++u) {
        const int g = D == 128 ? u : 2 * u + (w >> 1), id = D == 128 ? pid[u] : (w >> 1) ? pid[2 * u + 1] : pid[2 * u];
        const int key = key0 + 16 * g, left = imin(16, klen - key), in = key & ((1 << p.shift) - 1);
        const bool any = id >= 0 && left > 0;
        const int64_t page = any ? id : 0;
        const auto rk = make_rsrc(kbase + page * p.ksb * 2 + (int64_t)in * kst, any ? (uint32_t)((left - 1) * kst + 2 * D) : 0u);
        const auto rv = make_rsrc(vbase + page * p.vsb * 2 + (int64_t)in * vst, any ? (uint32_t)((left - 1) * vst + 2 * D) : 0u);
        load_lds16(rk, kd + (w + 4 * u) * 512, koff);
        load_lds16(rv, vd + (w + 4 * u) * 512, voff);
      }
    } else {
      const int left = imin(kBK, klen - key0);
      const auto rk = make_rsrc(kbase + (int64_t)key0 * kst, (uint32_t)((left - 1) * kst + 2 * D));
      const auto rv = make_rsrc(vbase + (int64_t)key0 * vst, (uint32_t)((left - 1) * vst + 2 * D));
#pragma unroll
      for (int u = 0; u < LPT; ++u) {
        load_lds16(rk, kd + (w + 4 * u) * 512, koff + u * 4 * RPL * kst);
        load_lds16(rv, vd + (w + 4 * u) * 512, voff + u * 4 * RPL * vst);
      }
    }
  };
  // rows of a block behind the sequence's end or on no page: zeros among the values (their weight is 0, and 0 times whatever
  // lies there has to be 0). The wave's own loads have landed.
  auto clean = [&](int jb, int ok, E* vd) {
    if ((jb + 1) * kBK <= klen && ok == 15) return;
#pragma unroll
    for (int u = 0; u < LPT; ++u) {
      const int row = (w + 4 * u) * RPL + lane / CPR;
      if (jb * kBK + row >= klen || !(ok >> (row >> 4) & 1)) *reinterpret_cast<X8*>(vd + (w + 4 * u) * 512 + lane * 8) = X8{};
    }
  };

  TileReads<D> rd;
  rd.init(lane);
  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
  float m = -INFINITY, l = 0.f;
  const float c = p.scale_log2, slack = fminf(8.f / c, 3e38f);  // finite: a first maximum is always taken

  auto block = [&](bool masked, int ok, const E* kb, const E* vb, int k0) {
    f32x16 s[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      s[kt] = f32x16{};
#pragma unroll
      for (int st = 0; st < DS; ++st) s[kt] = mma32(row_frag(kb + 32 * kt * D, rd, st), qf[st], s[kt]);
    }
    // the fragments' reads two products ahead
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
    for (int i = 0; i < 2 * DS - 2; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
    if (masked) {  // selects, from one word of bits a lane: branches a lane apart cost more
      uint64_t seen = view.block(k0, p.window, p.sinks);
      if (PAGED) {
        seen &= bits_below(klen - k0);
#pragma unroll
        for (int g = 0; g < 4; ++g) seen &= ok >> g & 1 ? ~0ull : ~(0xffffull << 16 * g);
      }
      seen >>= 4 * hh;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s[kt][e] = (uint32_t)(seen >> 32 * kt) >> (8 * (e >> 2) + (e & 3)) & 1 ? s[kt][e] : -INFINITY;
    }
    softmax_step<2, D, E>(s, acc, m, l, c, slack, vb, rd);
  };
  int ok = 15, ok_next = 15;  // of the block being used and of the one being loaded
  auto step = [&](int n, const E* kc, const E* vc, E* kn, E* vn) {
    const int jb = bl.at(n), next = bl.at(n + 1);
    const bool more = n + 1 < n1;
    if (more) {
      ok_next = ok_bits();
      fetch(next, kn, vn);
      if (n + 2 < n1) look_up(bl.at(n + 2));
    }
    const int k0 = jb * kBK, k1 = k0 + kBK - 1;
    if (wave_live && !none_sees(wq0, wq1, k0, k1, p.window, p.sinks))
      block(ok != 15 || !all_see(wq0, wq1, k0, k1, p.window, p.sinks), ok, kc, vc, k0);
    wait_loads();
    if (more) clean(next, ok_next, vn);
    ok = ok_next;
    __syncthreads();
  };
  if (n0 < n1) {
    look_up(bl.at(n0));
    ok = ok_bits();
    fetch(bl.at(n0), Ks0, Vs0);
    if (n0 + 1 < n1) look_up(bl.at(n0 + 1));
    wait_loads();
    clean(bl.at(n0), ok, Vs0);
    __syncthreads();
    for (int n = n0; n < n1; n += 2) {
      step(n, Ks0, Vs0, Ks1, Vs1);
      if (n + 1 < n1) step(n + 1, Ks1, Vs1, Ks0, Vs0);
    }
  }

  // O = O^T / l; the lane holds its row's columns 32 d + 8 j + 4 hh + r. Of several runs each leaves O, m and l.
  const bool whole = !PAGED || f.used == 1;
  float *po = nullptr, *pml = nullptr;
  if constexpr (PAGED) {
    po = p.part + (f.job * p.splits + split) * kBQ * D;
    pml = p.part + p.tiles * p.HKV * p.splits * kBQ * D + (f.job * p.splits + split) * 2 * kBQ;
  }
  l += __shfl_xor(l, 32, kWave);
  if (whole && row_ok && l == 0.f) {  // NaN where keys were seen, all with scores of -inf
    if constexpr (PAGED) l = sees_any<kBK>(p, f, view) ? NAN : 0.f;
    else l = sq.num >= 0 ? NAN : 0.f;
  }
  bool fine = finite_all(acc);
  fine = l != l || (__shfl_xor((int)fine, 32, kWave) && fine);
  const int64_t all = p.B * p.seqs.T, tok = sq.row * p.seqs.T + sq.start;
  const int r = 32 * w + li;
  auto write = [&](float inv) {
    if (whole) {
      E* const to = o_at(r);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          X4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = (E)(acc[d][4 * j + e] * inv);
          *reinterpret_cast<X4*>(to + 32 * d + 8 * j + 4 * hh) = x;
          if (!PAGED && p.o_rest) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = rest_of<E>(acc[d][4 * j + e] * inv);
            *reinterpret_cast<X4*>(static_cast<E*>(p.o_rest) + (to - static_cast<E*>(p.o)) + 32 * d + 8 * j + 4 * hh) = x;
          }
        }
    } else {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<f32x4*>(po + r * D + 32 * d + 8 * j + 4 * hh) =
              f32x4{acc[d][4 * j] * inv, acc[d][4 * j + 1] * inv, acc[d][4 * j + 2] * inv, acc[d][4 * j + 3] * inv};
    }
  };
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (row_ok) {
    write(inv);
    if (whole) {
      if (!PAGED && p.lse && hh == 0)
        p.lse[head_of(r) * all + tok + token_of(r)] = l == 0.f ? INFINITY : m * c + (__builtin_amdgcn_logf(l) - Pack<E>::lift);
    } else if (hh == 0) {
      pml[r] = m;
      pml[kBQ + r] = l;
    }
  }
  if (!__any(row_ok && !fine)) return;
  wait_loads();  // what was written above is there before rows are written again
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
  E* const tile = w == 0 ? Ks0 : w == 1 ? Ks1 : w == 2 ? Vs0 : Vs1;  // all waves are behind their last block
  const float nmc = m == -INFINITY ? 0.f : Pack<E>::lift - m * c, by = exp2f(raise<E>) * inv;
  for (int n = n0; n < n1; ++n) {
    const int k0 = bl.at(n) * kBK;
    if (none_sees(wq0, wq1, k0, k0 + kBK - 1, p.window, p.sinks)) continue;
    auto row_of = [&](const char* base, int64_t page_bytes, int64_t row_bytes, int j) {
      if (k0 + j >= klen) return static_cast<const E*>(nullptr);
      if (!PAGED) return reinterpret_cast<const E*>(base + (k0 + j) * row_bytes);
      const int id = table[(k0 + j) >> p.shift];
      return id < 0 || id >= p.pages ? static_cast<const E*>(nullptr)
                                     : reinterpret_cast<const E*>(base + id * page_bytes + ((k0 + j) & ((1 << p.shift) - 1)) * row_bytes);
    };
    auto key = [&](int j) { return row_of(kbase, p.ksb * 2, kst, j); };
    uint64_t seen = view.block(k0, p.window, p.sinks) & bits_below(klen - k0);
    if (PAGED) {
      look_up(bl.at(n));
#pragma unroll
      for (int g = 0; g < 4; ++g) seen &= pid[g] >= 0 ? ~0ull : ~(0xffffull << 16 * g);
    }
    again_block<2, D, E>(acc, qf, seen, key, [&](int j) { return row_of(vbase, p.vsb * 2, vst, j); }, tile, c, nmc, by, rd);
  }
  if (row_ok && !fine) write(exp2f(-raise<E>));
}

}  // namespace gdn
