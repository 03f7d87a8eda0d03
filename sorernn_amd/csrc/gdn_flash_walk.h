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

}  // namespace gdn
