// Which far queries and sinks the workgroups of attention's key gradients take (gdn_flash_walk.h), compiled for the host.
#include <stdint.h>

#define __device__
#define __host__
#define __forceinline__ inline

namespace gdn {

static int64_t g_outside, g_entries;  // reads outside the bounds' entries, and how many there are

inline int64_t load_index(const void* p, int, int64_t i) {
  if (i < 0 || i >= g_entries) {
    ++g_outside;
    return 0;
  }
  return static_cast<const int64_t*>(p)[i];
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

extern "C" int far_start(int reach, int tiles) { return far_by_start(reach, tiles); }

// A sequence's tiles of sinks with far queries.
extern "C" int far_tiles(int reach, int tiles, int len) { return far_tiles_of(FarList{256 * tiles, tiles, 1, reach}, len); }

// The far jobs: out[t] = row, start, len, number, piece, tile of sinks (-1: none), the slot and step that the sums are looked for at.
extern "C" int64_t far_jobs(const int64_t* cu, int64_t n, int64_t B, int64_t tokens, int far, int tiles, int by_start, int reach, int64_t jobs,
                            int64_t* out) {
  g_outside = 0;
  g_entries = n + 1;
  const Packed s{cu, 0, n, tokens};
  const FarList f{far, tiles, by_start, reach};
  for (int64_t t = 0; t < jobs; ++t) {
    const FarWork w = far_work(s, f, B, t);
    int64_t* o = out + 8 * t;
    o[0] = w.sq.row, o[1] = w.sq.start, o[2] = w.sq.len, o[3] = w.sq.num, o[4] = w.sq.tile, o[5] = w.sink_tile;
    Seq q = w.sq;
    if (!cu) q.num = (int)q.row;
    o[6] = w.sink_tile < 0 ? 0 : far_slot(s, f, q, w.sink_tile);
    o[7] = w.sink_tile < 0 ? 0 : far_step(s, f, q, B);
  }
  return g_outside;
}

// The near slots: out[x] = row, start, len, number, tile of sinks (-1: none), the slot that its sums are put at.
extern "C" int64_t near_slots(const int64_t* cu, int64_t n, int64_t tokens, int far, int tiles, int by_start, int reach, int64_t slots,
                              int64_t* out) {
  g_outside = 0;
  g_entries = n + 1;
  const Packed s{cu, 0, n, tokens};
  const FarList f{far, tiles, by_start, reach};
  for (int64_t x = 0; x < slots; ++x) {
    const FarWork w = near_work(s, f, x);
    int64_t* o = out + 6 * x;
    o[0] = w.sq.row, o[1] = w.sq.start, o[2] = w.sq.len, o[3] = w.sq.num, o[4] = w.sink_tile;
    o[5] = w.sink_tile < 0 ? 0 : near_slot(f, w.sq, w.sink_tile);
  }
  return g_outside;
}

extern "C" int far_first(int by_start, int reach) { return FarList{256, 1, by_start, reach}.first_query(); }
