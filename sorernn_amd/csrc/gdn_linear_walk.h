// Which tokens a workgroup of the decay linear attention walks, in chunks: index arithmetic only, the same on the host.
// Included after the definitions of load_index, uniform and starts_up_to.
//
// P has cu, cu_i32, T, N and tokens. starts_up_to(p, lo, hi, step, t) counts the lanes i of a wave with
// lo + i step < hi and start of sequence lo + i step <= t.
#pragma once

#include <stdint.h>

namespace gdn {

constexpr int kLinChunk = 64, kLinLanes = 64;

// First token of sequence n; of n = N the number of tokens. Captured and compiled calls do not check the bounds: whatever
// they hold, nothing outside the tensors is touched, and tokens of no sequence are left out.
template <typename P>
__device__ __forceinline__ int seq_start(const P& p, int n) {
  if (!p.cu) return n * p.T;
  const int64_t x = load_index(p.cu, p.cu_i32, n);
  return x < 0 ? 0 : x > p.tokens ? p.tokens : (int)x;
}

// The sequence of token t. All lanes of a wave search together.
template <typename P>
__device__ __forceinline__ int seq_of(const P& p, int t) {
  if (!p.cu) return (unsigned)t / (unsigned)p.T;
  int lo = 0, hi = p.N;  // start of lo <= t < start of hi
  while (hi - lo > 1) {
    const int step = (hi - lo + kLinLanes - 1) / kLinLanes;
    const int cnt = starts_up_to(p, lo, hi, step, t);  // one at least: lane 0's
    lo += (cnt > 1 ? cnt - 1 : 0) * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  return uniform(lo);
}

// The tokens among [lo, hi) that belong to sequences, [t0, t1), and the first and the last of these sequences, neither of
// them empty; t0 >= t1: none. The sequence found for a token is empty where the token belongs to none: behind the last
// sequence with tokens, or before the first.
struct Span {
  int t0, t1, first, last;
};
template <typename P>
__device__ __forceinline__ int span_front(const P& p, int& t0, int hi) {
  int n = seq_of(p, t0);
  const int bos = seq_start(p, n);
  if (bos > t0) {
    t0 = bos;
    if (t0 < hi) n = seq_of(p, t0);
  }
  return n;
}
template <typename P>
__device__ __forceinline__ int span_back(const P& p, int& t1, int lo) {
  int n = seq_of(p, t1 - 1);
  const int eos = seq_start(p, n + 1);
  if (eos < t1) {
    t1 = eos;
    if (t1 > lo) n = seq_of(p, t1 - 1);
  }
  return n;
}
template <typename P>
__device__ __forceinline__ Span span_of(const P& p, int lo, int hi) {
  Span s{lo, hi, 0, 0};
  s.first = span_front(p, s.t0, hi);
  s.last = span_back(p, s.t1, lo);
  return s;
}

// Up to 64 tokens of sequence n in walking order: fresh, the walk of the sequence begins with them; done, it ends.
struct Chunk {
  int t, len, n;  // len 0: none
  bool fresh, done;
};

// The chunks of tokens [lo, hi) in walking order. Chunks begin where a sequence or the segment does. The first is not fresh
// only if it lies at a border inside the token axis. They cover all tokens from t after start() to t after the last of them;
// the others of [lo, hi) belong to no sequence.
template <bool REV>
struct ChunkWalk {
  int lo, hi, n, bos, eos, t;  // t: REV, the end of what is left; else its start
  template <typename P>
  __device__ __forceinline__ void start(const P& p, int from, int to) {
    lo = from;
    hi = to;
    t = REV ? hi : lo;
    n = REV ? span_back(p, t, lo) : span_front(p, t, hi);
    t = t < lo ? lo : t > hi ? hi : t;
    bos = seq_start(p, n);
    eos = seq_start(p, n + 1);
    if (REV && t < hi) eos = t;
    if (!REV && t > lo) bos = t;
    // next() goes over empty sequences one by one: not over those that a call of a fixed number is filled up with
    const int end = seq_start(p, REV ? 0 : p.N);
    if (REV && end > lo) lo = end;
    if (!REV && end < hi) hi = end;
  }
  template <typename P>
  __device__ __forceinline__ Chunk next(const P& p) {
    Chunk c{0, 0, n, false, false};
    if (REV) {
      const int first = bos > lo ? bos : lo;
      if (t <= first) return c;
      c.t = first + ((t - 1 - first) & ~(kLinChunk - 1));
      c.len = t - c.t;
      c.fresh = t == eos;
      c.done = c.t == bos;
      t = c.t;
      if (t == bos && t > lo) {
        eos = t;
        while (bos >= t && --n >= 0) bos = seq_start(p, n);
      }
    } else {
      const int end = eos < hi ? eos : hi;
      if (t >= end) return c;
      c.t = t;
      c.len = end - t < kLinChunk ? end - t : kLinChunk;
      c.fresh = t == bos;
      c.done = t + c.len == eos;
      t += c.len;
      if (t == eos && t < hi) {
        bos = t;
        while (eos <= t && ++n < p.N) eos = seq_start(p, n + 1);
      }
    }
    return c;
  }
};

}  // namespace gdn
