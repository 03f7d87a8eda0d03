// The walk's index arithmetic (gdn_linear_walk.h) compiled for the host: the chunks of one segment, as a wave sees them.
#include <stdint.h>

#define __device__
#define __forceinline__ inline

namespace gdn {

struct Bounds {
  const void* cu;
  int cu_i32, T, N, tokens;
};

static int g_outside;  // reads outside the bounds' N + 1 entries
static int g_entries;

inline int64_t load_index(const void* p, int is_i32, int64_t i) {
  if (i < 0 || i >= g_entries) {
    ++g_outside;
    return 0;
  }
  return is_i32 ? static_cast<const int32_t*>(p)[i] : static_cast<const int64_t*>(p)[i];
}

inline int uniform(int x) { return x; }

inline int starts_up_to(const Bounds& p, int lo, int hi, int step, int t) {
  int count = 0;
  for (int lane = 0; lane < 64; ++lane) {
    const int i = lo + lane * step;
    count += i < hi && load_index(p.cu, p.cu_i32, i) <= t;
  }
  return count;
}

}  // namespace gdn

#include "../sorernn_amd/csrc/gdn_linear_walk.h"

template <bool REV>
static int walk(const gdn::Bounds& p, int lo, int hi, int* out, int most, int* ends) {
  gdn::ChunkWalk<REV> it;
  it.start(p, lo, hi);
  ends[0] = it.t;
  int count = 0;
  for (gdn::Chunk c = it.next(p); c.len > 0 && count < most; c = it.next(p), ++count) {
    const int row[] = {c.t, c.len, c.n, c.fresh, c.done};
    for (int i = 0; i < 5; ++i) out[5 * count + i] = row[i];
  }
  ends[1] = it.t;
  return count;
}

// Chunks (t, len, n, fresh, done) of tokens [lo, hi) into out, and where they begin and end in walking order; their number,
// or -1 after a read outside the bounds.
extern "C" int linear_walk(const int64_t* cu, int n, int tokens, int seq, int rev, int lo, int hi, int* out, int most, int* ends) {
  const gdn::Bounds p{cu, 0, seq, n, tokens};
  gdn::g_outside = 0;
  gdn::g_entries = n + 1;
  const int count = rev ? walk<true>(p, lo, hi, out, most, ends) : walk<false>(p, lo, hi, out, most, ends);
  return gdn::g_outside ? -1 : count;
}

// The tokens among [lo, hi) that belong to documents, and the first and last document: t0, t1, first, last into out.
extern "C" int linear_span(const int64_t* cu, int n, int tokens, int seq, int lo, int hi, int* out) {
  const gdn::Bounds p{cu, 0, seq, n, tokens};
  gdn::g_outside = 0;
  gdn::g_entries = n + 1;
  const gdn::Span s = gdn::span_of(p, lo, hi);
  out[0] = s.t0;
  out[1] = s.t1;
  out[2] = s.first;
  out[3] = s.last;
  return gdn::g_outside ? -1 : 0;
}
