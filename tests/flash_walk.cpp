// The attention kernels' index arithmetic (gdn_flash_walk.h) compiled for the host.
#include <stdint.h>

#define __device__
#define __host__
#define __forceinline__ inline

namespace gdn {

static int64_t g_outside, g_entries;  // reads outside the bounds' entries, and how many there are

inline int64_t load_index(const void* p, int is_i32, int64_t i) {
  if (i < 0 || i >= g_entries) {
    ++g_outside;
    return 0;
  }
  return is_i32 ? static_cast<const int32_t*>(p)[i] : static_cast<const int64_t*>(p)[i];
}
inline int64_t uniform64(int64_t x) { return x; }
template <typename F>
inline int lanes_of(F yes) {
  int n = 0;
  for (int lane = 0; lane < 64; ++lane) n += yes(lane);
  return n;
}

}  // namespace gdn

#include "../sorernn_amd/csrc/gdn_flash_walk.h"

using namespace gdn;

// Tiles of packed sequences: out[t] = start, len, num, tile. Returns their number, -1 after a read outside.
extern "C" int64_t flash_tiles(const int64_t* cu, int64_t n, int64_t tokens, int mul, int rows, int64_t* out, int64_t room) {
  g_outside = 0;
  g_entries = n + 1;
  const Packed s{cu, 0, n, tokens};
  const int64_t count = packed_tiles(tokens, n, mul, rows);
  if (count > room) return -2;
  for (int64_t t = 0; t < count; ++t) {
    const Seq q = packed_tile(s, t, mul, rows);
    out[4 * t] = q.start;
    out[4 * t + 1] = q.len;
    out[4 * t + 2] = q.num;
    out[4 * t + 3] = q.tile;
  }
  return g_outside ? -1 : count;
}

// Jobs of a flat grid: out[i] = kv head, head of the group, tile, or -1s.
extern "C" int64_t flash_jobs(int hkv, int rep, int64_t tiles, int64_t* out, int64_t room) {
  const int64_t n = job_groups(hkv, rep, tiles);
  if (n > room) return -2;
  for (int64_t i = 0; i < n; ++i) {
    Job j;
    const bool ok = job_of(i, hkv, rep, job_parts(hkv), tiles, j);
    out[3 * i] = ok ? j.hkv : -1;
    out[3 * i + 1] = ok ? j.hm : -1;
    out[3 * i + 2] = ok ? j.tile : -1;
  }
  return n;
}

// Blocks that queries at places first .. last see; and, of queries q0 .. q1 and keys k0 .. k1, bits: all see all, none sees any.
extern "C" int flash_blocks(int size, int first, int last, int window, int sinks, int* out) {
  const Blocks b = size == 32 ? blocks_of<32>(first, last, window, sinks) : blocks_of<64>(first, last, window, sinks);
  for (int n = 0; n < b.count; ++n) out[n] = b.at(n);
  return b.count;
}
extern "C" int flash_sees(int q0, int q1, int k0, int k1, int window, int sinks) {
  return (all_see(q0, q1, k0, k1, window, sinks) ? 1 : 0) | (none_sees(q0, q1, k0, k1, window, sinks) ? 2 : 0);
}
extern "C" int flash_near_end(int tile, int window, int len) { return near_end(tile, window, len); }
