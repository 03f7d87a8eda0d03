// Which sequence, tile and keys a workgroup of the attention kernels takes: index arithmetic alone, which also compiles for the
// host. load_index, uniform64 (a value that is the same in every lane) and lanes_of (how many lanes say yes) come from outside.
#pragma once

namespace gdn {

constexpr int kFar = 1 << 29;  // no window; also the bound on a sequence's length, so that places and their differences fit 32 bits

__device__ __forceinline__ int imin(int a, int b) { return a < b ? a : b; }
__device__ __forceinline__ int imax(int a, int b) { return a > b ? a : b; }

// ------------------------------------------------------------------------------------------------ sequences in tiles
// Tokens of a packed axis, cut where a sequence ends: N sequences and, for bounds that nobody checked, the tokens before
// the first and behind the last as sequences 0 and N + 1 that see nothing. Bounds are taken as between 0 and T: whatever they
// hold, no token outside is touched.
struct Packed {
  const void* cu;
  int cu_i32;
  int64_t N, T;
  __device__ __forceinline__ int64_t bound(int64_t j) const {
    if (j <= 0) return 0;
    if (j > N + 1) return T;
    const int64_t x = load_index(cu, cu_i32, j - 1);
    return x < 0 ? 0 : x > T ? T : x;
  }
};

// Tile `t` of rows of the sequences, `mul` rows a token and M rows a tile. A sequence from row b0 to row b1 has the tiles
// b0 / M + j to b1 / M + j of the list, j its number: as many as it can need, without a scan of the lengths. One wave reads
// 64 bounds at a time.
struct Seq {
  int64_t row;   // the batch row
  int64_t start; // first token inside it
  int len;       // tokens
  int num;       // number of the sequence, -1: tokens that belong to none
  int tile;      // tile of the sequence
};
__device__ __forceinline__ Seq packed_tile(const Packed& s, int64_t t, int mul, int M) {
  int64_t count = 0;  // sequences whose tiles begin at t or before: as the bounds ascend, the first ones
  for (int64_t base = 0; base < s.N + 2; base += 64) {
    const int below = lanes_of([&](int lane) { return base + lane < s.N + 2 && s.bound(base + lane) * mul / M + base + lane <= t; });
    count += below;
    if (below < 64) break;
  }
  const int64_t j = count > 0 ? count - 1 : 0, b0 = uniform64(s.bound(j)), b1 = uniform64(s.bound(j + 1));
  Seq r;
  r.row = 0;
  r.start = b0;
  r.len = (int)(b1 > b0 ? b1 - b0 : 0);
  r.num = j == 0 || j == s.N + 1 ? -1 : (int)(j - 1);
  const int64_t tile = t - (b0 * mul / M + j);
  r.tile = tile < 0 || tile > kFar / M ? kFar / M : (int)tile;  // of bounds out of order: none
  return r;
}
__host__ __device__ inline int64_t packed_tiles(int64_t T, int64_t N, int mul, int M) { return T * mul / M + N + 2; }

// Workgroup `idx` of a flat grid as (kv head, q head of it, tile). Workgroup i runs on XCD i % 8: the q heads of one kv head
// and neighbouring tiles share an XCD and its L2 as far as the heads divide over the eight; the tiles are dealt out in turn
// among the `parts` XCDs that share a head.
struct Job {
  int hkv, hm;
  int64_t tile;
};
__device__ __forceinline__ bool job_of(int64_t idx, int hkv, int rep, int parts, int64_t tiles, Job& job) {
  const int x = (int)(idx & 7), per = hkv * parts / 8 * rep;
  const int64_t j = idx >> 3, rank = j / per;
  const int m = (int)(j - rank * per), vg = x + 8 * (m / rep);
  job.hm = m % rep;
  job.hkv = vg % hkv;
  job.tile = rank * parts + vg / hkv;
  return job.tile < tiles;
}
__host__ __device__ inline int job_parts(int64_t hkv) { return hkv % 8 == 0 ? 1 : hkv % 4 == 0 ? 2 : hkv % 2 == 0 ? 4 : 8; }
__host__ __device__ inline int64_t job_groups(int64_t hkv, int64_t rep, int64_t tiles) {
  const int64_t parts = job_parts(hkv);
  return hkv * parts * rep * ((tiles + parts - 1) / parts);
}

// The blocks of BK keys that queries at places first .. last see: those with sinks before the window's, then the window's.
struct Blocks {
  int sinks, from, count;  // block n is n < sinks ? n : n - sinks + from
  __device__ __forceinline__ int at(int n) const { return n < sinks ? n : n - sinks + from; }
};
template <int BK>
__device__ __forceinline__ Blocks blocks_of(int first, int last, int window, int sinks) {
  Blocks b;
  const int lo = imax(0, first - window + 1);
  b.from = lo / BK;
  b.sinks = imin((sinks + BK - 1) / BK, b.from);
  const int end = last >= 0 ? last / BK + 1 : 0;
  b.count = imax(0, b.sinks + end - b.from);
  return b;
}

__device__ __forceinline__ bool sees(int q, int k, int window, int sinks) { return k <= q && (q - k < window || k < sinks); }
// of keys k0 .. k1 and queries q0 .. q1: all see all; none sees any
__device__ __forceinline__ bool all_see(int q0, int q1, int k0, int k1, int window, int sinks) {
  return k1 <= q0 && (q1 - k0 < window || k1 < sinks);
}
__device__ __forceinline__ bool none_sees(int q0, int q1, int k0, int k1, int window, int sinks) {
  return k0 > q1 || (q0 - k1 >= window && k0 >= sinks);
}

// Queries from here on see keys of the tile of 128 only as sinks; those before see them through the window.
__device__ __forceinline__ int near_end(int tile, int window, int len) { return imin(len, tile * 128 + 127 + window); }

// Far queries of a sequence's sinks, in pieces: work on (tile of 128 sinks, piece), with a slot of partial sums each, and a slot for
// the near queries of each such tile. Two layouts of both lists:
//   by number (by_start 0): every sequence has slots, as in packed_tile's list of tiles of `far` rows times `tiles`.
//   by start: only sequences with far queries have any, those of `reach` = window + 128 tokens and more. One of len tokens has
//   n = min(tiles, 1 + (len - reach) / 128) tiles and 1 + (len - reach) / far pieces, n times that at most len / by_start in all,
//   so that the slots from start / by_start on are its own.
struct FarList {
  int far, tiles;       // queries a piece, tiles of sinks at most
  int by_start, reach;
  __host__ __device__ int first_query() const { return by_start ? reach - 1 : 0; }  // where a sequence's pieces begin
};
__host__ __device__ inline int far_tiles_of(const FarList& f, int len) {
  if (len < f.reach) return 0;
  const int n = 1 + (len - f.reach) / 128;
  return n < f.tiles ? n : f.tiles;
}
// the largest by_start: (reach + x) / (tiles and pieces of x more tokens) is least where the last tile begins (x = 128 (tiles - 1)),
// or the second piece (x = 256 tiles), or where pieces are many, with 256 tiles queries each
__host__ __device__ inline int far_by_start(int reach, int tiles) {
  const int a = (reach - 128) / tiles + 128, b = (reach / tiles + 256) / 2;
  const int m = a < b ? a : b;
  return m < 256 ? m : 256;
}

// The sequence whose slots from start / by_start on hold `t`: the last that begins before; its own number of slots says whether
// `t` is one of them.
__device__ __forceinline__ Seq far_sequence(const Packed& s, int64_t t, int by_start) {
  int64_t count = 0;
  for (int64_t base = 0; base < s.N + 2; base += 64) {
    const int below = lanes_of([&](int lane) { return base + lane < s.N + 2 && s.bound(base + lane) / by_start <= t; });
    count += below;
    if (below < 64) break;
  }
  const int64_t j = count > 0 ? count - 1 : 0, b0 = uniform64(s.bound(j)), b1 = uniform64(s.bound(j + 1));
  return Seq{0, b0, (int)(b1 > b0 ? b1 - b0 : 0), j == 0 || j == s.N + 1 ? -1 : (int)(j - 1), 0};
}

// Job `t` of the far queries: the sequence with its piece as `tile`, and the tile of sinks, -1: none.
struct FarWork {
  Seq sq;
  int sink_tile;
};
__device__ __forceinline__ FarWork far_work(const Packed& s, const FarList& f, int64_t B, int64_t t) {
  FarWork w;
  if (f.by_start) {
    w.sq = far_sequence(s, t, f.by_start);
    const int64_t y = t - w.sq.start / f.by_start;
    const int n = w.sq.num < 0 ? 0 : far_tiles_of(f, w.sq.len);
    w.sink_tile = y >= 0 && n && y < (int64_t)n * (1 + (w.sq.len - f.reach) / f.far) ? (int)(y % n) : -1;
    w.sq.tile = n ? (int)(y / n) : 0;
    return w;
  }
  const int64_t slot = t / f.tiles;
  w.sink_tile = (int)(t - slot * f.tiles);
  if (s.cu) w.sq = packed_tile(s, slot, 1, f.far);
  else w.sq = Seq{slot % B, 0, (int)s.T, 0, (int)(slot / B)};
  if (w.sq.num < 0 || w.sq.tile > w.sq.len / f.far) w.sink_tile = -1;
  return w;
}
// Near slot `x`: the sequence and the tile of sinks, -1: none.
__device__ __forceinline__ FarWork near_work(const Packed& s, const FarList& f, int64_t x) {
  FarWork w;
  if (f.by_start) {
    w.sq = far_sequence(s, x, f.by_start);
    const int64_t y = x - w.sq.start / f.by_start;
    w.sink_tile = y >= 0 && w.sq.num >= 0 && y < far_tiles_of(f, w.sq.len) ? (int)y : -1;
    return w;
  }
  const int num = (int)(x / f.tiles);
  w.sink_tile = (int)(x - (int64_t)num * f.tiles);
  w.sq = Seq{num, 0, (int)s.T, num, 0};
  if (s.cu) {
    const int64_t b0 = s.bound(num + 1), b1 = s.bound(num + 2);
    w.sq.row = 0, w.sq.start = b0, w.sq.len = (int)(b1 > b0 ? b1 - b0 : 0);
  }
  return w;
}
// The slots of a sequence's tile of sinks: of its near queries, and of its piece 0, with `far_step` from one piece to the next.
__device__ __forceinline__ int64_t near_slot(const FarList& f, const Seq& sq, int sink_tile) {
  return (f.by_start ? sq.start / f.by_start : (int64_t)sq.num * f.tiles) + sink_tile;
}
__device__ __forceinline__ int64_t far_slot(const Packed& s, const FarList& f, const Seq& sq, int sink_tile) {
  if (f.by_start) return sq.start / f.by_start + sink_tile;
  return (s.cu ? sq.start / f.far + sq.num + 1 : sq.row) * f.tiles + sink_tile;
}
__device__ __forceinline__ int64_t far_step(const Packed& s, const FarList& f, const Seq& sq, int64_t B) {
  return f.by_start ? far_tiles_of(f, sq.len) : (s.cu ? 1 : B) * f.tiles;
}

}  // namespace gdn
