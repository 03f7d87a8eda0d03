// Linear attention with a decay for each head (the gated delta rule's recurrence without its correction term):
// chunked forward and backward for gfx950.
//
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t
//
// Over a chunk of 64 tokens, with b_i the sum of g up to token i and b_C that of the whole chunk:
//   o_i   = scale (exp(b_i) S_in^T q_i + sum_{j <= i} exp(b_i - b_j) (q_i . k_j) v_j)
//   S_out = exp(b_C) S_in + sum_j exp(b_C - b_j) k_j v_j^T
//
// One walker kernel computes the forward and the three gradients, as all of them are this recurrence:
//   dq_i = scale S_i do_i              the walk itself with (q, k, v) = (do, v, k): its state is S^T
//   dv_j = R_j^T k_j, dk_j = R_j v_j   R_j = exp(g_{j+1}) R_{j+1} + scale q_j do_j^T: the walk from the end with
//                                      (k, q, do) and (v, do, q)
//   dg_t = exp(g_t) <S_{t-1}, R_t> = sum over i >= t of (q_i . dq_i - k_i . dk_i), plus <S_T, dS_T>
//
// The state stays in fp32 MFMA accumulators, a wave holding all K rows of its columns; it is the A operand of S^T Q^T as it
// stands, split into bf16 parts in registers. A workgroup walks one segment of the flat token axis for one value head,
// over the sequences' borders, so that 256 workgroups have the same number of tokens whatever the sequences' lengths are.
// For the sequence that a segment's border cuts, a first kernel walks the segment for its own contribution to the state
// (k and v only), a scan over the segments turns these into the states at the borders, and the walkers run side by side.
//
// Rounding: q, k, v and do are bf16 operands as they come. What is computed is split into bf16 parts that are multiplied
// one by one: three (24 bits, as fp32 holds) where the result is an fp32 output (the state, and what dg sums), two
// where the outputs are rounded to bf16 (scores, and the state under o): a single part's 2^-9 would be as large as the
// rounding of the output itself. The decays are summed in 64 bits: a difference of two sums in 32 would carry the
// rounding of the sums into every weight.

#include <stddef.h>

#include <type_traits>

#include "gdn_mfma.h"

namespace gdn {

// In place of a segment's decay: the sequence that goes on in the next segment begins in this one, or none does. No decay is
// negative.
constexpr float kBegins = -1.f;

struct LinParams {
  const bf16 *q, *k, *v, *e;    // [tokens][heads][K or V]: the walk's q, k, v and the rows of the gate's dot products
  int64_t qs, ks, vs, es;       // elements between tokens
  unsigned rq, rk, rv, re;      // value heads that share a head of each
  const void* g;                // log decays, or null: no decay
  int dg;
  int64_t gb, gt, gh;           // element strides of batch row, token and value head
  const float* init;            // [N][HV][K][V] state before the walk, or null: zeros
  float* entry;                 // [segments][HV][K][V] states entering the segments, or null where no border cuts a sequence
  float* decay;                 // [segments][HV] decay of the sequence that goes on in the next segment, or kBegins
  int transposed;               // init and entry are read as [V][K]
  float* fin;                   // [N][HV][K][V] state after the walk, or null
  void* o;                      // [tokens][HV][V]
  float* dot;                   // [HV][tokens] with DOT
  const void* cu;
  int cu_i32, T, N, tokens, L;  // segments of L tokens; without cu sequences of T
  int zero_rest;                // write zeros to the rows of o whose tokens belong to no sequence
  unsigned HV;
  float scale;
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

__device__ __forceinline__ int starts_up_to(const LinParams& p, int lo, int hi, int step, int t) {
  const int i = lo + (int)(threadIdx.x % kWave) * step;
  return __popcll(__ballot(i < hi && load_index(p.cu, p.cu_i32, i < hi ? i : lo) <= t));
}

}  // namespace gdn

#include "gdn_linear_walk.h"

namespace gdn {

static_assert(kLinChunk == kC && kLinLanes == kWave, "the walk's chunks and lanes");

// Decay terms of a chunk, base-2 logarithms: b = h + l in two floats, the weight of a token in the state's update and
// that of the state in a token's output (each with the factor it carries), and the decay of the whole chunk.
struct alignas(16) Decays {
  float h[kC], l[kC], wst[kC], win[kC];
  float all;
};
static_assert(sizeof(Decays) % 16 == 0, "arrays of it are read 16 bytes at a time");

template <int CTRL, int ROW_MASK>
__device__ __forceinline__ double dpp_scan_step(double v) {
  const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROW_MASK, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROW_MASK, 0xf, false);
  return v + __hiloint2double(hi, lo);
}

__device__ __forceinline__ double wave_inclusive_sum64(double x) {
  x = dpp_scan_step<0x111, 0xf>(x);
  x = dpp_scan_step<0x112, 0xf>(x);
  x = dpp_scan_step<0x114, 0xf>(x);
  x = dpp_scan_step<0x118, 0xf>(x);
  x = dpp_scan_step<0x142, 0xa>(x);
  return dpp_scan_step<0x143, 0xc>(x);
}
__device__ __forceinline__ double last_lane(double x) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), kWave - 1),
                          __builtin_amdgcn_readlane(__double2loint(x), kWave - 1));
}

// Log decays below -100 (exp of it is 0 beside any weight that counts) are taken as -100: a reset of -inf leaves the
// differences of sums behind it finite.
__device__ __forceinline__ double log2_decay(uint32_t raw, int dtype) {
  const float x = raw32_to_f32(raw, dtype);
  return (double)(x < -100.f ? -100.f : x) * 1.4426950408889634;
}

// One wave, lane = token.
template <bool REV>
__device__ __forceinline__ void chunk_decays(Decays& d, double x, float scale, int lane) {
  x = wave_inclusive_sum64(x);
  const double all = last_lane(x);
  const float head = __builtin_amdgcn_exp2f((float)x), tail = __builtin_amdgcn_exp2f((float)(all - x));
  d.h[lane] = (float)x;
  d.l[lane] = (float)(x - (double)(float)x);
  d.wst[lane] = REV ? scale * head : tail;
  d.win[lane] = REV ? tail : scale * head;
  if (lane == 0) d.all = __builtin_amdgcn_exp2f((float)all);
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// A pair of bf16 as bits, kept in a scalar register: as a literal -1 the pair (-1, 0) is encoded as an inline constant,
// which the dot product takes for (0, -1).
__device__ __forceinline__ bf16x2 scalar_pair(uint32_t bits) {
  asm("" : "+s"(bits));
  return __builtin_bit_cast(bf16x2, bits);
}

// The next bf16 part of 8 fp32 values: rounds them, and leaves in x what the rounding left out. x - part is exact; as a
// product with (-1, 0) or (0, -1) it needs no unpacking of the pair.
__device__ __forceinline__ bf16x8 next_part(float (&x)[8], bool more) {
  const bf16x2 lo = scalar_pair(0x0000bf80u), hi = scalar_pair(0xbf800000u);
  bf16x8 r;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const bf16x2 h = {(bf16)x[e], (bf16)x[e + 1]};
    r[e] = h[0];
    r[e + 1] = h[1];
    if (more) {
      x[e] = __builtin_amdgcn_fdot2_f32_bf16(h, lo, x[e], false);
      x[e + 1] = __builtin_amdgcn_fdot2_f32_bf16(h, hi, x[e + 1], false);
    }
  }
  return r;
}

// Tiles in LDS: rows of D elements without padding, the 16-byte piece c of row r at piece c ^ swz(r). A row fragment
// (16 rows, one piece) then falls on all 64 banks, and so do 8 rows of two neighbouring pieces (the transposed reads of
// 16 columns); the transposed reads of 32 columns, half a piece each, take two turns.
template <int D>
__device__ __forceinline__ int swz(int r) {
  return D == 128 ? ((r & 3) << 2 | ((r >> 2) & 1) << 1 | ((r >> 3) & 1))
                  : (((r >> 2) & 1) << 2 | ((r >> 1) & 1) << 1 | ((r >> 3) & 1));
}
template <int D>
__device__ __forceinline__ bf16x8 ld_row(const bf16* tile, int row, int piece) {
  return ld8(tile + row * D + ((piece ^ swz<D>(row)) << 3));
}
// Rows r0 + 4g + m and r0 + 16 + 4g + m, m = 0..3, of one column: c0 + STEP (i / 4) + i % 4.
template <int D, int STEP>
__device__ __forceinline__ bf16x8 ld_cols(const bf16* tile, int r0, int c0, int lane) {
  const int g = lane >> 4, li = lane & 15, row = r0 + 4 * g + (li >> 2), col = c0 + STEP * (li & 3);
  const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
      (lds_bf16x4*)(tile + row * D + (((col >> 3) ^ swz<D>(row)) << 3) + (col & 7)));
  const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
      (lds_bf16x4*)(tile + (row + 16) * D + (((col >> 3) ^ swz<D>(row + 16)) << 3) + (col & 7)));
  return bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// A chunk's rows on their way to LDS: thread t of 256 holds the 16-byte pieces t, t + 256, ... of the 64 x D tile, RP rows
// apart. Whole chunks are read at a scalar address plus the thread's offset; in a sequence's last chunk the rows past its
// end re-read its first row and are written as zeros.
template <int D>
struct Tile {
  static constexpr int NP = kC * D / 8 / 256, RP = 256 / (D / 8);
  static_assert(RP % 16 == 0, "the swizzle has a period of 16 rows");
  bf16x8 r[NP];
  __device__ __forceinline__ static int row0() { return threadIdx.x % 256 / (D / 8); }
  __device__ __forceinline__ static int piece() { return threadIdx.x % (D / 8); }
  __device__ __forceinline__ static uint32_t offset(int64_t stride) {
    return (uint32_t)(row0() * (int)stride + piece() * 8) * 2u;
  }
  __device__ __forceinline__ void fetch(const bf16* base, int64_t stride, uint32_t off, int len) {
    if (len == kC) {
#pragma unroll
      for (int n = 0; n < NP; ++n)
        r[n] = *reinterpret_cast<const bf16x8*>(reinterpret_cast<const char*>(base + n * RP * stride) + off);
    } else {
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        const int row = row0() + n * RP;
        r[n] = *reinterpret_cast<const bf16x8*>(base + (row < len ? row : 0) * stride + piece() * 8);
      }
    }
  }
  __device__ __forceinline__ void put(bf16* tile, int len) {
    if (len < kC) {
#pragma unroll
      for (int n = 0; n < NP; ++n)
        if (row0() + n * RP >= len) r[n] = bf16x8{};
    }
#pragma unroll
    for (int n = 0; n < NP; ++n)
      *reinterpret_cast<bf16x8*>(tile + (row0() + n * RP) * D + ((piece() ^ swz<D>(row0())) << 3)) = r[n];
  }
};

// The state's columns of wave w of NW: accumulator tiles s[2u + c][ct], rows 32u + 8g + 4c + r, columns
// 16 NCT w + 4 NCT (i / 4) + 4 ct + i % 4, so that 4 NCT neighbouring columns of O^T fall on a lane.
template <int KD, int VD, int NW>
struct State {
  static constexpr int NA = KD / 16, NCT = VD / 16 / NW;
  f32x4 s[NA][NCT];

  __device__ __forceinline__ static int row0(int a, int g) { return 32 * (a >> 1) + 8 * g + 4 * (a & 1); }
  __device__ __forceinline__ static int col(int w, int ct, int i) {
    return 16 * NCT * w + 4 * NCT * (i >> 2) + 4 * ct + (i & 3);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) s[a][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // The addresses of load and store are computed where they are used, not kept in registers over the walk.
  __device__ __forceinline__ void load(const float* src, int pitch, bool transposed, int w, int lane) {
    lane = opaque_int(lane);
    const int g = lane >> 4, i = lane & 15;
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
        if (transposed) {
          s[a][ct] = *reinterpret_cast<const f32x4*>(src + col(w, ct, i) * KD + row0(a, g));
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) s[a][ct][r] = src[(row0(a, g) + r) * pitch + col(w, ct, i)];
        }
      }
  }
  __device__ __forceinline__ void store(float* dst, int pitch, int w, int lane) const {
    lane = opaque_int(lane);
    const int g = lane >> 4, i = lane & 15;
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
        for (int r = 0; r < 4; ++r) dst[(row0(a, g) + r) * pitch + col(w, ct, i)] = s[a][ct][r];
  }
  // The wave's columns of 32 rows of V from r0 on, as the accumulators' token order has them.
  __device__ __forceinline__ static void columns(const bf16* Vs, int r0, int w, int lane, bf16x8 (&vf)[NCT]) {
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct) vf[ct] = ld_cols<VD, 4 * NCT>(Vs, r0, 16 * NCT * w + 4 * ct, lane);
  }
  // S = all S + K^T (wst V): V weighted in fp32 and split into three bf16 parts (K is exact)
  __device__ __forceinline__ void update(const Decays& d, const bf16* Ks, const bf16x8 (&vf)[2][NCT], int lane) {
    const int g = lane >> 4;
    const float all = d.all;
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) s[a][ct] *= all;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const f32x4 w0 = *reinterpret_cast<const f32x4*>(d.wst + 32 * ks + 4 * g);
      const f32x4 w1 = *reinterpret_cast<const f32x4*>(d.wst + 32 * ks + 16 + 4 * g);
      bf16x8 part[NCT][3];
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)vf[ks][ct][e] * (e < 4 ? w0[e & 3] : w1[e & 3]);
#pragma unroll
        for (int n = 0; n < 3; ++n) part[ct][n] = next_part(x, n < 2);
      }
      constexpr int AB = 4 / NCT;  // rows of tiles whose products run side by side
#pragma unroll
      for (int a0 = 0; a0 < NA; a0 += AB) {
        bf16x8 kf[AB];
#pragma unroll
        for (int a = 0; a < AB; ++a)
          kf[a] = ld_cols<KD, 8>(Ks, 32 * ks, 32 * ((a0 + a) >> 1) + 4 * ((a0 + a) & 1), lane);
#pragma unroll
        for (int n = 2; n >= 0; --n)
#pragma unroll
          for (int a = 0; a < AB; ++a)
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct) s[a0 + a][ct] = mma(kf[a], part[ct][n], s[a0 + a][ct]);
      }
    }
  }
};

// Raw gate values of a chunk's tokens, a lane each, read ahead of their use.
struct GateRow {
  uint32_t raw = 0;
  __device__ __forceinline__ void fetch(const LinParams& p, unsigned hv, const Chunk& c, int lane) {
    const int64_t row = p.cu ? c.t * p.gt : c.n * p.gb + (c.t - c.n * p.T) * p.gt;
    raw = p.g && lane < c.len ? load_raw32(p.g, p.dg, row + lane * p.gt + hv * p.gh) : 0u;
  }
  __device__ __forceinline__ double value(const LinParams& p) const { return p.g ? log2_decay(raw, p.dg) : 0.; }
};

// ------------------------------------------------------------------------------------------------
// What a segment adds to the state of the sequence that its border cuts: the walk without outputs, from where the sequence
// begins (with its initial state) or from the segment's other border (from zero). Forward walks leave it in the next
// segment's place, walks from the end in that of the segment before. Two workgroups share 128 columns, which doubles the
// waves in flight: at 4 x 4,096 tokens, 16 heads of 128, 37.5 us, 40.7 with eight waves of one workgroup for all columns.
template <int KD, bool REV>
__global__ __launch_bounds__(256, 3) void gated_deltaless_segment_kernel(LinParams p, int VD) {
  __shared__ __align__(16) bf16 Ks[2][kC * KD], Vs[2][kC * 64];
  __shared__ __align__(16) Decays d[2];
  const int lane = threadIdx.x % kWave, w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const unsigned hv = blockIdx.x % p.HV;
  const int seg = blockIdx.x / p.HV + (REV ? 1 : 0);  // without the last (first), whose border cuts nothing
  int lo = seg * p.L, hi = lo + p.L < p.tokens ? lo + p.L : p.tokens;
  const int n = seq_of(p, REV ? lo - 1 : hi), bos = seq_start(p, n), eos = seq_start(p, n + 1);
  const bool whole = REV ? eos <= hi : bos >= lo;  // the sequence's walk begins in this segment
  if (REV ? bos >= lo || eos <= lo : bos >= hi || eos <= hi) {  // no sequence is cut
    if (threadIdx.x == 0 && blockIdx.y == 0) p.decay[(int64_t)seg * p.HV + hv] = kBegins;
    return;
  }
  if (REV) hi = whole ? eos : hi;
  else lo = whole ? bos : lo;
  const bf16* k0 = p.k + lo * p.ks + hv / p.rk * KD;
  const bf16* v0 = p.v + lo * p.vs + hv / p.rv * VD + blockIdx.y * 64;
  const int nc = (hi - lo + kC - 1) / kC;
  auto chunk = [&](int ci) {
    Chunk c{lo + (REV ? nc - 1 - ci : ci) * kC, 0, n, false, false};
    c.len = ci >= nc ? 0 : hi - c.t < kC ? hi - c.t : kC;
    return c;
  };
  Tile<KD> kt;
  Tile<64> vt;
  GateRow gate;
  const uint32_t koff = kt.offset(p.ks), voff = vt.offset(p.vs);
  auto fetch = [&](int ci) {
    const Chunk c = chunk(ci);
    kt.fetch(k0 + (c.t - lo) * p.ks, p.ks, koff, c.len);
    vt.fetch(v0 + (c.t - lo) * p.vs, p.vs, voff, c.len);
  };
  if (w == 0) gate.fetch(p, hv, chunk(0), lane);
  fetch(0);
  State<KD, 64, 4> st;
  if (whole && p.init) st.load(p.init + ((int64_t)n * p.HV + hv) * (KD * VD) + blockIdx.y * 64, VD, false, w, lane);
  else st.zero();
  double total = 0.;
  auto bring = [&](int ci) {  // chunk ci, on its way, into LDS, and the next one's loads
    if (ci >= nc) return;
    const int len = chunk(ci).len;
    const double x = w == 0 ? gate.value(p) : 0.;  // ahead of the next loads: the wait for it would be for them too
    kt.put(Ks[ci & 1], len);
    vt.put(Vs[ci & 1], len);
    if (w == 0) gate.fetch(p, hv, chunk(ci + 1), lane);
    if (ci + 1 < nc) fetch(ci + 1);
    if (w == 0) {
      total += x;
      chunk_decays<REV>(d[ci & 1], x, p.scale, lane);
    }
  };
  bring(0);
  __syncthreads();
  for (int ci = 0; ci < nc; ++ci) {
    bring(ci + 1);
    bf16x8 vf[2][1];
    st.columns(Vs[ci & 1], 0, w, lane, vf[0]);
    st.columns(Vs[ci & 1], 32, w, lane, vf[1]);
    st.update(d[ci & 1], Ks[ci & 1], vf, lane);
    __syncthreads();
  }
  st.store(p.entry + ((int64_t)(seg + (REV ? -1 : 1)) * p.HV + hv) * (KD * VD) + blockIdx.y * 64, VD, w, lane);
  if (w == 0 && blockIdx.y == 0) {
    for (int m = 1; m < kWave; m <<= 1) total += __shfl_xor(total, m, kWave);
    if (lane == 0) p.decay[(int64_t)seg * p.HV + hv] = whole ? kBegins : __builtin_amdgcn_exp2f((float)total);
  }
}

// The segments' contributions into the states entering them, in place: entry[s] += decay[s - 1] entry[s - 1] (from the
// end: decay[s + 1] entry[s + 1]), four neighbouring elements a thread. Where a decay is kBegins nothing of the other is
// taken: it may not have been written. A decay that is 0 is multiplied: 0 times an infinity or NaN is NaN, as in a walk.
template <bool REV>
__global__ __launch_bounds__(256) void gated_deltaless_scan_kernel(LinParams p, int elems, int segs) {
  const unsigned per = elems / 1024, hv = blockIdx.x / per;
  const int at = (blockIdx.x % per) * 1024 + threadIdx.x * 4;
  const int64_t step = (int64_t)p.HV * elems;
  float* e = p.entry + (int64_t)hv * elems + at;
  const float* dc = p.decay + hv;
  f32x4 run = {0.f, 0.f, 0.f, 0.f};
  constexpr int U = 8;  // loads in flight
  for (int s0 = 0; s0 < segs - 1; s0 += U) {
    f32x4 x[U];
    float c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u < segs - 1 ? s0 + u : segs - 2;
      x[u] = *reinterpret_cast<const f32x4*>(e + (REV ? segs - 2 - s : s + 1) * step);
      c[u] = dc[(int64_t)(REV ? segs - 1 - s : s) * p.HV];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u >= segs - 1) break;
      run = c[u] == kBegins ? x[u] : run * c[u] + x[u];
      *reinterpret_cast<f32x4*>(e + (REV ? segs - 2 - s0 - u : s0 + u + 1) * step) = run;
    }
  }
}

// ------------------------------------------------------------------------------------------------
// The walk. One workgroup a CU: waves 0-3 hold the state and make the outputs of chunk c, waves 4-7 meanwhile bring the
// tiles of chunks c + 1 and c + 2 into LDS and make the scores of chunk c + 1; one barrier a chunk. At 4 x 4,096 tokens,
// 16 heads of 128, 79 us; its loads and stores alone take 59, the state's waves alone 64. With eight waves for the state the
// scores' waves are what a chunk waits for: 80 us.
// DOT 1 also gives e_i . (the state's share of o_i) for every token; DOT 2 adds the scores' share, the row sums less the
// column sums of W_ij = P_ij (e_i . v_j), exact bf16 products summed in fp32.
//
// Scores are kept for the tiles that are not masked, in blocks of 16 queries x 32 keys (tok_col order): queries 0-15 and
// 16-31 have one block, the others two (walks from the end: mirrored).
constexpr int kStateWaves = 4, kScoreWaves = 4, kWalkThreads = (kStateWaves + kScoreWaves) * kWave;

template <int KD, int VD, int DOT>
struct WalkLds {
  bf16 q[3][kC * KD], k[3][kC * KD], v[2][kC * VD];
  bf16 ps[2][2][6 * 512];  // [slot][part]
  Decays d[3];
  float dots[DOT ? 2 : 1][kStateWaves][DOT ? kC : 1];
  float rows[DOT == 2 ? 2 : 1][10][DOT == 2 ? 16 : 1], cols[DOT == 2 ? 2 : 1][10][DOT == 2 ? 16 : 1];
};

// Zeros in rows [t0, t1) of o (pitch in elements), by the 256 threads of the scores' waves.
template <int VD, typename OT>
__device__ __forceinline__ void zero_rows(OT* o, int64_t pitch, int t0, int t1) {
  constexpr int PER = 16 / sizeof(OT), LPR = VD / PER, RP = kScoreWaves * kWave / LPR;
  const int at = threadIdx.x % (kScoreWaves * kWave);
  for (int t = t0 + at / LPR; t < t1; t += RP) *reinterpret_cast<f32x4*>(o + t * pitch + at % LPR * PER) = f32x4{0.f, 0.f, 0.f, 0.f};
}

// The states of sequences without tokens go through a walk as they are. One wave; the segments take the sequences in turn.
template <int KD, int VD>
__device__ __forceinline__ void pass_states(const LinParams& p, unsigned hv, int seg, int segs, int lane) {
  for (int64_t n0 = seg; n0 < p.N; n0 += (int64_t)segs * kWave) {
    const int64_t n = n0 + (int64_t)lane * segs;
    const bool empty = n < p.N && seq_start(p, (int)n) >= seq_start(p, (int)n + 1);
    for (uint64_t m = __ballot(empty); m; m &= m - 1) {
      const int64_t at = ((n0 + (int64_t)(__ffsll((unsigned long long)m) - 1) * segs) * p.HV + hv) * (KD * VD) + lane * 4;
      for (int i = 0; i < KD * VD; i += 4 * kWave)
        *reinterpret_cast<f32x4*>(p.fin + at + i) =
            p.init ? *reinterpret_cast<const f32x4*>(p.init + at + i) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
}

template <int KD, int VD, bool REV, int DOT, typename OT>
__device__ __forceinline__ void walk_segment(const LinParams& p, WalkLds<KD, VD, DOT>& lds) {
  constexpr int NCT = VD / 16 / kStateWaves, NU = KD / 32;
  constexpr int NS = DOT ? 3 : 2;  // parts of the state under o
  using Lds = WalkLds<KD, VD, DOT>;
  static_assert(offsetof(Lds, ps) % 16 == 0 && offsetof(Lds, d) % 16 == 0 && (DOT < 2 || offsetof(Lds, cols) % 16 == 0),
                "accessed 16 bytes at a time");
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int g = lane >> 4, i = lane & 15;
  const unsigned hv = blockIdx.x % p.HV, seg = blockIdx.x / p.HV;
  const int seg0 = seg * p.L, seg1 = p.tokens - seg0 < p.L ? p.tokens : seg0 + p.L;
  const bf16* e0 = DOT ? p.e + hv / p.re * VD : nullptr;
  ChunkWalk<REV> it;
  it.start(p, seg0, seg1);
  const int first = it.t;  // with REV the end of the first chunk

  if (wave < kStateWaves) {  // ------------------------------------------------------------------ the state's waves
    const int w = wave;
    OT* o0 = static_cast<OT*>(p.o) + (int64_t)hv * VD;
    State<KD, VD, kStateWaves> st;
    auto begin = [&](const Chunk& c) {
      const float* src = !c.fresh ? p.entry + ((int64_t)seg * p.HV + hv) * (KD * VD)
                                  : (p.init ? p.init + ((int64_t)c.n * p.HV + hv) * (KD * VD) : nullptr);
      if (src) st.load(src, VD, p.transposed, w, lane);
      else st.zero();
    };
    Chunk now = it.next(p), then = it.next(p);
    if (now.len > 0) begin(now);
    __syncthreads();
    __syncthreads();
    for (int c = 0; now.len > 0; ++c) {
      const int t0 = now.t, len = now.len;
      const Decays& d = lds.d[c % 3];
      const bf16 *Qs = lds.q[c % 3], *Ks = lds.k[c % 3], *Vs = lds.v[c & 1];
      bf16x4 ev[4][NCT];
      if (DOT) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int row = 16 * t + i;
          const bf16* er = e0 + (int64_t)(t0 + (row < len ? row : 0)) * p.es + 16 * NCT * w + 4 * NCT * g;
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) ev[t][ct] = *reinterpret_cast<const bf16x4*>(er + 4 * ct);
        }
      }
      // the state's share: O^T = S^T Q^T, columns = tokens
      f32x4 acc[4][NCT];
      f32x4 low[DOT ? 4 : 1][DOT ? NCT : 1] = {};  // the small parts' products apart: fewer roundings of the whole
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) acc[t][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        bf16x8 part[NCT][NS], qf[4];
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = st.s[2 * u + (e >> 2)][ct][e & 3];
#pragma unroll
          for (int n = 0; n < NS; ++n) part[ct][n] = next_part(x, n + 1 < NS);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) qf[t] = ld_row<KD>(Qs, 16 * t + i, 4 * u + g);
#pragma unroll
        for (int n = NS - 1; n >= 0; --n)
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct) {
              if (DOT && n > 0) low[DOT ? t : 0][DOT ? ct : 0] = mma(part[ct][n], qf[t], low[DOT ? t : 0][DOT ? ct : 0]);
              else acc[t][ct] = mma(part[ct][n], qf[t], acc[t][ct]);
            }
      }
      if (DOT) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) acc[t][ct] += low[DOT ? t : 0][DOT ? ct : 0];
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float wi = d.win[16 * t + i];
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) acc[t][ct] *= wi;
      }
      if (DOT) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          double x = 0.;  // dg sums thousands of these, which mostly cancel
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
            for (int r = 0; r < 4; ++r) x += (double)acc[t][ct][r] * (double)(float)ev[t][ct][r];
          x += __shfl_xor(x, 16);
          x += __shfl_xor(x, 32);
          if (g == 0) lds.dots[DOT ? c & 1 : 0][w][DOT ? 16 * t + i : 0] = (float)x;
        }
      }
      // the scores' share: O^T += V^T P^T
      bf16x8 vf[2][NCT];
      float bad = 0.f;  // NaN where the wave's columns of v hold an infinity or NaN: a sum of products with zero
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        State<KD, VD, kStateWaves>::columns(Vs, 32 * k2, w, lane, vf[k2]);
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
          for (int e = 0; e < 8; e += 2)
            bad = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{vf[k2][ct][e], vf[k2][ct][e + 1]}, scalar_pair(0u), bad, false);
      }
      const auto* ps = lds.ps[c & 1];
      if (__ballot(!(bad == 0.f)) == 0) {
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
          for (int n = 1; n >= 0; --n)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const int ta = REV ? 3 - t : t, ka = REV ? 1 - k2 : k2;
              if (ta < 2 && ka == 1) continue;  // all masked
              const int block = ta < 2 ? ta : 2 * ta - 2 + ka;
              const bf16x8 pf = ld8(ps[n] + block * 512 + i * 32 + ((g ^ (i >> 2)) << 3));
#pragma unroll
              for (int ct = 0; ct < NCT; ++ct) acc[t][ct] = mma(vf[k2][ct], pf, acc[t][ct]);
            }
      } else {  // they reach the tokens that see them, not those whose score is masked
        for (int j = 0; j < len; ++j) {
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            if (REV ? j < 16 * t + i : j > 16 * t + i) continue;
            const int ta = REV ? 3 - t : t, ka = REV ? 1 - (j >> 5) : j >> 5, col = tok_col(j & 31);
            const int at = (ta < 2 ? ta : 2 * ta - 2 + ka) * 512 + i * 32 + (((col >> 3) ^ (i >> 2)) << 3) + (col & 7);
            const float x = (float)ps[0][at] + (float)ps[1][at];
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const int vc = 16 * NCT * w + 4 * NCT * g + 4 * ct + r;
                acc[t][ct][r] += x * (float)Vs[j * VD + (((vc >> 3) ^ swz<VD>(j)) << 3) + (vc & 7)];
              }
          }
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int row = 16 * t + i;
        if (row >= len) continue;
        OT* dst = o0 + (int64_t)(t0 + row) * p.HV * VD + 16 * NCT * w + 4 * NCT * g;
        if constexpr (sizeof(OT) == 4) {
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) *reinterpret_cast<f32x4*>(dst + 4 * ct) = acc[t][ct];
        } else if constexpr (NCT == 2) {
          *reinterpret_cast<bf16x8*>(dst) = pack8(acc[t][0], acc[t][NCT - 1]);
        } else {
          *reinterpret_cast<bf16x4*>(dst) = to_bf16x4(acc[t][0][0], acc[t][0][1], acc[t][0][2], acc[t][0][3]);
        }
      }
      if (now.done ? p.fin != nullptr : then.len > 0) st.update(d, Ks, vf, lane);
      if (now.done && p.fin) st.store(p.fin + ((int64_t)now.n * p.HV + hv) * (KD * VD), VD, w, lane);
      __syncthreads();
      now = then;
      then = it.next(p);
      if (now.len > 0 && now.fresh) begin(now);
    }
    return;
  }

  // ------------------------------------------------------------------------------------ the scores' waves
  const int w = wave - kStateWaves;
  const bf16* q0 = p.q + hv / p.rq * KD;
  const bf16* k0 = p.k + hv / p.rk * KD;
  const bf16* v0 = p.v + hv / p.rv * VD;
  Tile<KD> qt, kt;
  Tile<VD> vt;
  const uint32_t qoff = qt.offset(p.qs), koff = kt.offset(p.ks), voff = vt.offset(p.vs);
  auto fetch_qk = [&](const Chunk& c) {
    if (c.len == 0) return;
    qt.fetch(q0 + c.t * p.qs, p.qs, qoff, c.len);
    kt.fetch(k0 + c.t * p.ks, p.ks, koff, c.len);
  };
  auto fetch_v = [&](const Chunk& c) {
    if (c.len) vt.fetch(v0 + c.t * p.vs, p.vs, voff, c.len);
  };
  auto put_qk = [&](const Chunk& c, int slot) {
    if (c.len == 0) return;
    qt.put(lds.q[slot], c.len);
    kt.put(lds.k[slot], c.len);
  };
  auto put_v = [&](const Chunk& c, int half) {
    if (c.len) vt.put(lds.v[half], c.len);
  };
  GateRow gate;
  // The gate's values and the rows of score_dots are taken before new loads are issued: a wait for them would be for
  // those too.
  auto gate_value = [&](const Chunk& c, const Chunk& after) {  // of c, which has been fetched; then the next one's loads
    const double x = w == 0 && c.len ? gate.value(p) : 0.;
    if (w == 0) gate.fetch(p, hv, after, lane);
    return x;
  };
  auto decays = [&](const Chunk& c, int slot, double x) {
    if (w == 0 && c.len) chunk_decays<REV>(lds.d[slot], x, p.scale, lane);
  };
  // 12 tiles of 16 keys x 16 queries are written (2 of zeros), 3 a wave: P^T, rows = keys j, column = query
  f32x4 pv[3];
  auto tile_of = [&](int n, int& ta, int& ja) {
    const int sl = w + 4 * n;
    ta = n == 0 ? sl >> 1 : 1 + n;
    ja = n == 0 ? sl & 1 : w;
  };
  auto scores = [&](const Chunk& c, int slot, int half) {  // half: the chunk's number & 1
    if (c.len == 0) return;
    const bf16 *Qs = lds.q[slot], *Ks = lds.k[slot];
    const Decays& d = lds.d[slot];
    auto* ps = lds.ps[half];
    // the three tiles side by side, also where all of one is masked; tiles 1 and 2 have the same keys
    bf16x8 kf[2][NU], qf[3][NU];
#pragma unroll
    for (int n = 0; n < 3; ++n) {
      int ta, ja;
      tile_of(n, ta, ja);
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        qf[n][u] = ld_row<KD>(Qs, 16 * (REV ? 3 - ta : ta) + i, 4 * u + g);
        if (n < 2) kf[n][u] = ld_row<KD>(Ks, 16 * (REV ? 3 - ja : ja) + i, 4 * u + g);
      }
      pv[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int n = 0; n < 3; ++n) pv[n] = mma(kf[n > 0][u], qf[n][u], pv[n]);
#pragma unroll
    for (int n = 0; n < 3; ++n) {
      int ta, ja;
      tile_of(n, ta, ja);
      const int t = REV ? 3 - ta : ta, jt = REV ? 3 - ja : ja, iq = 16 * t + i;
      const float bh = d.h[iq], bl = d.l[iq];
      const f32x4 jh = *reinterpret_cast<const f32x4*>(d.h + 16 * jt + 4 * g);
      const f32x4 jl = *reinterpret_cast<const f32x4*>(d.l + 16 * jt + 4 * g);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 16 * jt + 4 * g + r;
        const float diff = REV ? (jh[r] - bh) + (jl[r] - bl) : (bh - jh[r]) + (bl - jl[r]);
        const float x = pv[n][r] * (p.scale * __builtin_amdgcn_exp2f(diff));
        pv[n][r] = (REV ? j >= iq : j <= iq) ? x : 0.f;
      }
      const f32x4 x = pv[n];
      const bf16x4 hi = to_bf16x4(x[0], x[1], x[2], x[3]);
      const bf16x4 lo = to_bf16x4(x[0] - (float)hi[0], x[1] - (float)hi[1], x[2] - (float)hi[2], x[3] - (float)hi[3]);
      const int block = ta < 2 ? ta : 2 * ta - 2 + (ja >> 1);
      const int at = block * 512 + i * 32 + ((g ^ (i >> 2)) << 3) + 4 * (jt & 1);
      *reinterpret_cast<bf16x4*>(ps[0] + at) = hi;
      *reinterpret_cast<bf16x4*>(ps[1] + at) = lo;
    }
  };
  // DOT 2: the sums of W over the tiles whose scores this wave holds (pv, of the chunk before the one just scored)
  bf16x8 er[DOT == 2 ? 3 : 1][DOT == 2 ? VD / 32 : 1];
  auto dot_rows = [&](const Chunk& c) {
    if (DOT != 2 || c.len == 0) return;
#pragma unroll
    for (int n = 0; n < 3; ++n) {
      int ta, ja;
      tile_of(n, ta, ja);
      const int iq = 16 * (REV ? 3 - ta : ta) + i;
      const bf16* src = e0 + (int64_t)(c.t + (iq < c.len ? iq : 0)) * p.es + 8 * g;
#pragma unroll
      for (int u = 0; u < VD / 32; ++u) er[DOT == 2 ? n : 0][DOT == 2 ? u : 0] = ld8(src + 32 * u);
    }
  };
  auto score_dots = [&](const Chunk& c, int half, const f32x4 (&x)[3]) {
    const int len = c.len;
    const bf16* Vs = lds.v[half];
#pragma unroll
    for (int n = 0; n < 3; ++n) {
      int ta, ja;
      tile_of(n, ta, ja);
      if (ja > ta) continue;
      const int t = REV ? 3 - ta : ta, jt = REV ? 3 - ja : ja, iq = 16 * t + i;
      f32x4 a = {0.f, 0.f, 0.f, 0.f}, cs;
#pragma unroll
      for (int u = 0; u < VD / 32; ++u)
        a = mma(ld_row<VD>(Vs, 16 * jt + i, 4 * u + g), er[DOT == 2 ? n : 0][DOT == 2 ? u : 0], a);
      float rs = 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 16 * jt + 4 * g + r;
        const float ww = (REV ? j >= iq : j <= iq) && iq < len && j < len ? x[n][r] * a[r] : 0.f;
        rs += ww;
        cs[r] = group_sum<16>(ww);
      }
      rs = xor32_sum(xor16_sum(rs));
      const int idx = ta * (ta + 1) / 2 + ja, sl = DOT == 2 ? half : 0;
      if (g == 0) lds.rows[sl][idx][DOT == 2 ? i : 0] = rs;
      if (i == 0) *reinterpret_cast<f32x4*>(&lds.cols[sl][idx][DOT == 2 ? 4 * g : 0]) = cs;
    }
  };
  // the gate's dot products of a chunk, all of whose shares are in LDS
  auto finish_dots = [&](const Chunk& c, int half) {
    if (!DOT || w != 1 || lane >= c.len) return;
    const int sl = DOT ? half : 0;
    double x = 0.;
#pragma unroll
    for (int ww = 0; ww < kStateWaves; ++ww) x += lds.dots[sl][ww][DOT ? lane : 0];
    if (DOT == 2) {
      const int ta = REV ? 3 - g : g;  // the token's tile, as query and as key
#pragma unroll
      for (int o = 0; o < 4; ++o) {
        if (o <= ta) x += lds.rows[DOT == 2 ? sl : 0][ta * (ta + 1) / 2 + o][DOT == 2 ? i : 0];
        if (o >= ta) x -= lds.cols[DOT == 2 ? sl : 0][o * (o + 1) / 2 + ta][DOT == 2 ? i : 0];
      }
    }
    p.dot[(int64_t)hv * p.tokens + c.t + lane] = (float)x;
  };
  // chunk c is at[1] in step c, and at[0] the one before
  Chunk at[5] = {};
#pragma unroll
  for (int n = 1; n < 5; ++n) at[n] = it.next(p);
  if (w == 0) gate.fetch(p, hv, at[1], lane);
  fetch_qk(at[1]);
  fetch_v(at[1]);
  if (w == 3 && p.fin && p.cu) pass_states<KD, VD>(p, hv, seg, gridDim.x / p.HV, lane);
  const double x0 = gate_value(at[1], at[2]);
  put_qk(at[1], 0);
  fetch_qk(at[2]);
  put_v(at[1], 0);
  fetch_v(at[2]);
  decays(at[1], 0, x0);
  const double x1 = gate_value(at[2], at[3]);
  put_qk(at[2], 1);
  fetch_qk(at[3]);
  decays(at[2], 1, x1);
  __syncthreads();
  scores(at[1], 0, 0);
  __syncthreads();
  int slot = 0, half = 0;  // c % 3, c & 1
  while (at[1].len > 0) {
    const int s1 = slot == 2 ? 0 : slot + 1, s2 = slot == 0 ? 2 : slot - 1;  // of chunks c + 1 and c + 2
    dot_rows(at[1]);
    const double x = gate_value(at[3], at[4]);
    put_v(at[2], half ^ 1);
    put_qk(at[3], s2);
    fetch_v(at[3]);
    fetch_qk(at[4]);
    decays(at[3], s2, x);
    f32x4 held[3];
    if (DOT == 2) {
#pragma unroll
      for (int n = 0; n < 3; ++n) held[n] = pv[n];
    }
    scores(at[2], s1, half ^ 1);
    if (DOT == 2) score_dots(at[1], half, held);
    finish_dots(at[0], half ^ 1);
    __syncthreads();
    slot = s1;
    half ^= 1;
#pragma unroll
    for (int n = 0; n < 4; ++n) at[n] = at[n + 1];
    at[4] = it.next(p);
  }
  finish_dots(at[0], half ^ 1);
  if (p.zero_rest) {
    OT* o = static_cast<OT*>(p.o) + (int64_t)hv * VD;
    zero_rows<VD>(o, (int64_t)p.HV * VD, seg0, REV ? it.t : first);
    zero_rows<VD>(o, (int64_t)p.HV * VD, REV ? first : it.t, seg1);
  }
}

template <int KD, int VD>
__global__ __launch_bounds__(kWalkThreads, 2) void gated_deltaless_chunk_kernel(LinParams p) {
  __shared__ __align__(16) WalkLds<KD, VD, 0> lds;
  walk_segment<KD, VD, false, 0, bf16>(p, lds);
}

// The backward's three walks in one launch (K, V: those of the forward): y = 0 dq, 1 dk, 2 dv. OT: of dq and dk. At
// 4 x 4,096 tokens, 16 heads of 128, 271 us; without the gate's gradient each walk is the forward's.
template <int K, int V, bool GATE, typename OT>
__global__ __launch_bounds__(kWalkThreads, 2) void gated_deltaless_chunk_bwd_kernel(LinParams dq, LinParams dk, LinParams dv) {
  using Q = WalkLds<V, K, GATE ? 2 : 0>;
  using R = WalkLds<V, K, GATE ? 1 : 0>;
  using S = WalkLds<K, V, 0>;
  constexpr size_t qr = sizeof(Q) > sizeof(R) ? sizeof(Q) : sizeof(R);
  __shared__ __align__(16) char lds[qr > sizeof(S) ? qr : sizeof(S)];
  if (blockIdx.y == 0) walk_segment<V, K, false, GATE ? 2 : 0, OT>(dq, *reinterpret_cast<Q*>(lds));
  else if (blockIdx.y == 1) walk_segment<V, K, true, GATE ? 1 : 0, OT>(dk, *reinterpret_cast<R*>(lds));
  else walk_segment<K, V, true, 0, bf16>(dv, *reinterpret_cast<S*>(lds));
}

// ------------------------------------------------------------------------------------------------
// dg of a segment: what lies behind each of its sequences is <S, R> at the segment's border (the state entering the next
// segment with what the walk from the end brings there) or <S_T, dS_T> at the sequence's end, then the sum from the end
// of q . dq - k . dk. The sum over a whole piece is known as well, from <S, R> at the border before it or <S_0, dS_0>: what
// it misses, the rounding of all the dot products, is spread over the piece in proportion to |q . dq| + |k . dk|, which
// leaves 1/sqrt(3) of the error of a plain sum. The waves take the sequences in turn; the one at the border is the last.
// 22 us at 4 x 4,096 tokens, 16 heads of 128, most of it for the states' products (14 with one border's instead of both).
struct LinFinish {
  const float *x, *y;              // [HV][tokens] q . dq and k . dk
  const float *entry, *rentry;     // the states at the segments' borders, or null
  const float *fin, *dfin;         // at the sequences' ends; either may be null (dfin: a zero gradient)
  const float *init, *dinit;       // at their beginnings, or null (init: zeros)
  void* dg;                        // [tokens][HV], or null
  int dtype, elems, segs;          // elems: K V
  // dq and dk of the value heads that share a head, [tokens][HV][K] fp32, into [tokens][HV / rep][K]; or null
  const float *dq_heads, *dk_heads;
  bf16 *dq, *dk;
  int rep, K;
};

// Sum over the threads of `of` (a wave's 64 or a workgroup's 256) of the products of 4,096 m elements.
__device__ __forceinline__ double state_product(const float* s, const float* r, int elems, int at, int of) {
  double sum = 0.;
  for (int at0 = at * 4; at0 < elems; at0 += 16 * of) {
    f32x4 u[4], v[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      u[n] = *reinterpret_cast<const f32x4*>(s + at0 + 4 * of * n);
      v[n] = *reinterpret_cast<const f32x4*>(r + at0 + 4 * of * n);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n)
      sum += (double)(u[n][0] * v[n][0] + u[n][1] * v[n][1]) + (double)(u[n][2] * v[n][2] + u[n][3] * v[n][3]);
  }
  for (int m = 1; m < kWave; m <<= 1) sum += __shfl_xor(sum, m, kWave);
  return sum;
}

__global__ __launch_bounds__(256) void gated_deltaless_finish_kernel(LinParams p, LinFinish a) {
  __shared__ double part[2][4];
  const unsigned gates = a.dg ? (unsigned)a.segs * p.HV : 0u;
  if (blockIdx.x >= gates) {  // the sums over the value heads that share a q/k head
    const int64_t at = ((int64_t)(blockIdx.x - gates) * 256 + threadIdx.x) * 4, all = (int64_t)p.tokens * (p.HV / a.rep) * a.K;
    if (at >= all) return;
    const float* src = (blockIdx.y ? a.dk_heads : a.dq_heads) + at / a.K * a.rep * a.K + at % a.K;
    f32x4 sum = *reinterpret_cast<const f32x4*>(src);
    for (int r = 1; r < a.rep; ++r) sum += *reinterpret_cast<const f32x4*>(src + (int64_t)r * a.K);
    *reinterpret_cast<bf16x4*>((blockIdx.y ? a.dk : a.dq) + at) = to_bf16x4(sum[0], sum[1], sum[2], sum[3]);
    return;
  }
  if (blockIdx.y) return;
  const int lane = threadIdx.x % kWave, w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const unsigned hv = blockIdx.x % p.HV, seg = blockIdx.x / p.HV;
  const int seg0 = seg * p.L, seg1 = p.tokens - seg0 < p.L ? p.tokens : seg0 + p.L;
  const Span span = span_of(p, seg0, seg1);
  if (p.zero_rest)  // tokens of no sequence
    for (int t = seg0 + threadIdx.x; t < seg1; t += 256)
      if (t < span.t0 || t >= span.t1) store_from_f32(a.dg, a.dtype, (int64_t)t * p.HV + hv, 0.f);
  if (span.t0 >= span.t1) return;
  const int first = span.first, last = span.last;
  const bool cut = seq_start(p, last + 1) > seg1;  // the last sequence goes on in the next segment
  const bool begun = seq_start(p, first) < seg0;   // the first one began in an earlier segment
  const int64_t next = (int64_t)p.HV * a.elems, at0 = ((int64_t)seg * p.HV + hv) * a.elems;
  double border = 0., before = 0.;
  if (cut || begun) {
    double r = 0., l = 0.;
    if (cut) r = state_product(a.entry + at0 + next, a.rentry + at0, a.elems, threadIdx.x, 256);
    if (begun) l = state_product(a.entry + at0, a.rentry + at0 - next, a.elems, threadIdx.x, 256);
    if (lane == 0) {
      part[0][w] = r;
      part[1][w] = l;
    }
    __syncthreads();
    border = part[0][0] + part[0][1] + part[0][2] + part[0][3];
    before = part[1][0] + part[1][1] + part[1][2] + part[1][3];
  }
  for (int n = last - w; n >= first; n -= 4) {
    const int bos = seq_start(p, n), eos = seq_start(p, n + 1);
    const int lo = bos > seg0 ? bos : seg0, hi = eos < seg1 ? eos : seg1;
    double sum = 0.;
    if (eos > seg1) sum = border;
    else if (a.fin && a.dfin) {
      const int64_t at = ((int64_t)n * p.HV + hv) * a.elems;
      sum = state_product(a.fin + at, a.dfin + at, a.elems, lane, kWave);
    }
    const float *xs = a.x + (int64_t)hv * p.tokens, *ys = a.y + (int64_t)hv * p.tokens;
    // what the sum over the piece misses, for a unit of |x| + |y|
    double first_sum = before;
    bool known = true;
    if (bos >= seg0) {
      first_sum = 0.;
      known = !a.init || a.dinit;
      if (a.init && a.dinit) {
        const int64_t at = ((int64_t)n * p.HV + hv) * a.elems;
        first_sum = state_product(a.init + at, a.dinit + at, a.elems, lane, kWave);
      }
    }
    double all = 0., weight = 0.;
    constexpr int U = 8;  // loads in flight
    for (int t0 = known ? lo + lane : hi; t0 < hi; t0 += U * kWave) {
      float x[U], y[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u * kWave;
        x[u] = xs[t < hi ? t : lo];
        y[u] = ys[t < hi ? t : lo];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (t0 + u * kWave >= hi) break;
        all += (double)x[u] - (double)y[u];
        weight += fabs((double)x[u]) + fabs((double)y[u]);
      }
    }
    for (int m = 1; m < kWave; m <<= 1) {
      all += __shfl_xor(all, m, kWave);
      weight += __shfl_xor(weight, m, kWave);
    }
    double miss = known && weight > 0. ? (first_sum - sum - all) / weight : 0.;
    if (!(fabs(miss) < 1e30)) miss = 0.;  // infinities and NaN stay with the tokens before them
    for (int end0 = hi; end0 > lo; end0 -= U * kWave) {
      float x[U], y[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {  // lane 0 the last of 64 tokens
        const int t = end0 - u * kWave - 1 - lane;
        x[u] = xs[t >= lo ? t : lo];
        y[u] = ys[t >= lo ? t : lo];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = end0 - u * kWave - 1 - lane;
        if (end0 - u * kWave <= lo) break;
        const double xx = x[u], yy = y[u];
        const double run = wave_inclusive_sum64(t >= lo ? xx - yy + miss * (fabs(xx) + fabs(yy)) : 0.);
        if (t >= lo) store_from_f32(a.dg, a.dtype, (int64_t)t * p.HV + hv, (float)(sum + run));
        sum += last_lane(run);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------
// host
struct LinPlan {
  int64_t L, segs;  // segments of L tokens of the flat token axis
  bool split;       // a segment's border may cut a sequence
};

// Segments so that their number times the value heads is at most 256, a workgroup a CU (from 129 heads on one segment: more
// are uneven, up to 170 heads three are less so). Short sequences stay whole, several a segment: a cut costs two launches
// and a second pass over k and v, as much as walking 384 tokens (1 x 384 tokens, 4 heads of 64: 15.5 us whole; 448, the
// first length that is cut: 15.1, and about 5 us of the host's time for the launches).
constexpr int64_t kLinGroups = 256, kLinMinSegment = 128, kLinWhole = 384;

static LinPlan lin_plan(int64_t B, int64_t T, int64_t HV, bool varlen) {
  const int64_t tokens = B * T, most = HV <= 128 ? kLinGroups / HV : HV <= 170 ? 3 : 1;
  LinPlan pl{};
  int64_t L = ((tokens + most - 1) / most + kC - 1) / kC * kC;
  if (L < kLinMinSegment) L = kLinMinSegment;
  if (!varlen && T <= (L > kLinWhole ? L : kLinWhole)) {
    pl.L = (L + T - 1) / T * T;
  } else if (tokens <= kLinWhole) {
    pl.L = tokens;
  } else {
    pl.L = L;
  }
  pl.segs = (tokens + pl.L - 1) / pl.L;
  pl.split = pl.segs > 1 && (varlen || T > pl.L);
  return pl;
}

static int64_t align256l(int64_t b) { return (b + 255) / 256 * 256; }
static int64_t lin_states_bytes(const LinPlan& pl, int64_t HV, int64_t K, int64_t V) {
  return pl.split ? align256l(pl.segs * HV * K * V * 4) + align256l(pl.segs * HV * 4) : 0;
}

template <typename F>
static void lin_by_dims(int64_t K, int64_t V, F go) {
  using C64 = std::integral_constant<int, 64>;
  using C128 = std::integral_constant<int, 128>;
  if (K == 128 && V == 128) go(C128{}, C128{});
  else if (K == 64 && V == 64) go(C64{}, C64{});
  else if (K == 128) go(C128{}, C64{});
  else go(C64{}, C128{});
}

template <bool REV>
static void launch_segments(const LinParams& p, const LinPlan& pl, int64_t K, int64_t V, hipStream_t s) {
  const dim3 grid((unsigned)((pl.segs - 1) * p.HV), (unsigned)(V / 64));
  if (K == 128) hipLaunchKernelGGL((gated_deltaless_segment_kernel<128, REV>), grid, dim3(256), 0, s, p, (int)V);
  else hipLaunchKernelGGL((gated_deltaless_segment_kernel<64, REV>), grid, dim3(256), 0, s, p, (int)V);
  if (pl.segs > 2)
    hipLaunchKernelGGL((gated_deltaless_scan_kernel<REV>), dim3((unsigned)(p.HV * (K * V / 1024))), dim3(256), 0, s, p,
                       (int)(K * V), (int)pl.segs);
}

static int lin_check(const char* name, int64_t B, int64_t T, int64_t H, int64_t HV, int64_t K, int64_t V, int64_t N,
                     bool varlen, int g_dtype, const void* const* ptrs, int nptrs) {
  if (B <= 0 || T < 0 || H <= 0 || HV <= 0 || HV % H || N <= 0 || (varlen ? B != 1 : N != B)) {
    gdn_internal_set_error("%s: bad sizes B=%lld T=%lld H=%lld HV=%lld N=%lld (cu_seqlens requires B == 1, N == B without "
                           "it)", name, (long long)B, (long long)T, (long long)H, (long long)HV, (long long)N);
    return GDN_ERR_INVALID;
  }
  if ((K != 64 && K != 128) || (V != 64 && V != 128)) {
    gdn_internal_set_error("%s: head dims K=%lld V=%lld unsupported (each must be 64 or 128)", name, (long long)K,
                           (long long)V);
    return GDN_ERR_UNSUPPORTED;
  }
  if (g_dtype < GDN_DTYPE_F32 || g_dtype > GDN_DTYPE_F16) {
    gdn_internal_set_error("%s: unknown gate dtype %d", name, g_dtype);
    return GDN_ERR_INVALID;
  }
  for (int n = 0; n < nptrs; ++n)
    if (reinterpret_cast<uintptr_t>(ptrs[n]) & 15) {
      gdn_internal_set_error("%s: tensors must be 16-byte aligned", name);
      return GDN_ERR_INVALID;
    }
  if (HV > 65536 || N > 0x3fffffffLL || B > 0x3fffffffLL || T > 0x3fffffffLL || B * T > 0x3fffffffLL) {
    gdn_internal_set_error("%s: too many sequences, heads or tokens for one call", name);
    return GDN_ERR_UNSUPPORTED;
  }
  return GDN_OK;
}

static LinParams lin_params(const LinPlan& pl, const void* g, int g_dtype, int64_t gb, int64_t gt, int64_t gh, const void* cu,
                            unsigned flags, int64_t T, int64_t N, int64_t HV, float scale) {
  LinParams p{};
  p.g = g;
  p.dg = g_dtype;
  p.gb = gb;
  p.gt = gt;
  p.gh = gh;
  p.cu = cu;
  p.cu_i32 = (flags & GDN_FLAG_CU_INT32) ? 1 : 0;
  p.T = (int)T;
  p.N = (int)N;
  p.tokens = (int)(cu ? T : N * T);
  p.L = (int)pl.L;
  p.HV = (unsigned)HV;
  p.scale = scale;
  return p;
}

// The walk's q, k, v and e with the number of value heads that share a head of each.
static void lin_roles(LinParams& p, const void* q, int rq, const void* k, int rk, const void* v, int rv, const void* e,
                      int re, int64_t K, int64_t V) {
  p.q = static_cast<const bf16*>(q);
  p.k = static_cast<const bf16*>(k);
  p.v = static_cast<const bf16*>(v);
  p.e = static_cast<const bf16*>(e);
  p.rq = rq;
  p.rk = rk;
  p.rv = rv;
  p.re = re;
  p.qs = p.HV / rq * K;
  p.ks = p.HV / rk * K;
  p.vs = p.HV / rv * V;
  p.es = p.HV / re * V;
}

static void lin_states(LinParams& p, const LinPlan& pl, char* states, int64_t K, int64_t V) {
  p.entry = pl.split ? reinterpret_cast<float*>(states) : nullptr;
  p.decay = pl.split ? reinterpret_cast<float*>(states + align256l(pl.segs * p.HV * K * V * 4)) : nullptr;
}

}  // namespace gdn

using namespace gdn;

extern "C" size_t gdn_decay_attn_states_size(int64_t B, int64_t T, int64_t HV, int64_t K, int64_t V, int64_t N, int varlen) {
  if (B <= 0 || T <= 0 || HV <= 0 || K <= 0 || V <= 0 || N <= 0) return 0;
  return (size_t)lin_states_bytes(lin_plan(B, T, HV, varlen != 0), HV, K, V);
}

extern "C" int gdn_decay_attn_fwd(const void* q, const void* k, const void* v, const void* g, const float* initial_state,
                                  void* o, float* final_state, const void* cu_seqlens, int64_t B, int64_t T, int64_t H,
                                  int64_t HV, int64_t K, int64_t V, int64_t N, int g_dtype, int64_t g_batch_stride,
                                  int64_t g_token_stride, int64_t g_head_stride, float scale, unsigned flags, void* states,
                                  size_t states_bytes, void* stream) {
  if (!q || !k || !v || !o) {
    gdn_internal_set_error("gdn_decay_attn_fwd: null tensor pointer");
    return GDN_ERR_INVALID;
  }
  const void* ptrs[] = {q, k, v, o, initial_state, final_state, states};
  if (int rc = lin_check("gdn_decay_attn_fwd", B, T, H, HV, K, V, N, cu_seqlens != nullptr, g_dtype, ptrs, 7)) return rc;
  if (T == 0) return GDN_OK;
  const LinPlan pl = lin_plan(B, T, HV, cu_seqlens != nullptr);
  const size_t need = (size_t)lin_states_bytes(pl, HV, K, V);
  if (need && (!states || states_bytes < need)) {
    gdn_internal_set_error("gdn_decay_attn_fwd: states of %zu bytes needed", need);
    return GDN_ERR_INVALID;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int rep = (int)(HV / H);
  LinParams p = lin_params(pl, g, g_dtype, g_batch_stride, g_token_stride, g_head_stride, cu_seqlens, flags, T, N, HV, scale);
  lin_roles(p, q, rep, k, rep, v, 1, nullptr, 1, K, V);
  lin_states(p, pl, static_cast<char*>(states), K, V);
  p.init = initial_state;
  if (pl.split) launch_segments<false>(p, pl, K, V, s);
  p.fin = final_state;
  p.o = o;
  p.zero_rest = cu_seqlens && (flags & GDN_FLAG_ZERO_REST);
  lin_by_dims(K, V, [&](auto k_, auto v_) {
    hipLaunchKernelGGL((gated_deltaless_chunk_kernel<decltype(k_)::value, decltype(v_)::value>),
                       dim3((unsigned)(pl.segs * HV)), dim3(kWalkThreads), 0, s, p);
  });
  return gdn_internal_check_launch("gated_deltaless_chunk_kernel");
}

// Workspace of the backward: the states of the walk from the end, the gate's two dot products, and with shared q/k heads
// dq and dk of every value head in fp32.
namespace {
struct LinBwdSpace {
  int64_t states, dots, heads;
  int64_t bytes(bool shared) const { return states + 2 * dots + (shared ? 2 * heads : 0); }
};
LinBwdSpace lin_bwd_space(const LinPlan& pl, int64_t B, int64_t T, int64_t HV, int64_t K, int64_t V) {
  return {lin_states_bytes(pl, HV, K, V), align256l(B * T * HV * 4), align256l(B * T * HV * K * 4)};
}
}  // namespace

extern "C" size_t gdn_decay_attn_bwd_workspace_size(int64_t B, int64_t T, int64_t H, int64_t HV, int64_t K, int64_t V,
                                                    int64_t N, int varlen) {
  if (B <= 0 || T <= 0 || H <= 0 || HV <= 0 || HV % H || K <= 0 || V <= 0 || N <= 0) return 0;
  return (size_t)lin_bwd_space(lin_plan(B, T, HV, varlen != 0), B, T, HV, K, V).bytes(HV != H);
}

extern "C" int gdn_decay_attn_bwd(const void* q, const void* k, const void* v, const void* g, const float* initial_state,
                                  const float* final_state, const void* d_o, const float* d_final_state, const void* states,
                                  const void* cu_seqlens, int64_t B, int64_t T, int64_t H, int64_t HV, int64_t K, int64_t V,
                                  int64_t N, int g_dtype, int64_t g_batch_stride, int64_t g_token_stride,
                                  int64_t g_head_stride, float scale, unsigned flags, void* dq, void* dk, void* dv, void* dg,
                                  float* d_initial_state, void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !k || !v || !d_o || !dq || !dk || !dv || (dg && !g)) {
    gdn_internal_set_error("gdn_decay_attn_bwd: null tensor pointer");
    return GDN_ERR_INVALID;
  }
  if (dg && d_final_state && !final_state) {
    gdn_internal_set_error("gdn_decay_attn_bwd: dg with d_final_state needs final_state");
    return GDN_ERR_INVALID;
  }
  const void* ptrs[] = {q, k, v, d_o, dq, dk, dv, initial_state, final_state, d_final_state, d_initial_state, states,
                        workspace};
  if (int rc = lin_check("gdn_decay_attn_bwd", B, T, H, HV, K, V, N, cu_seqlens != nullptr, g_dtype, ptrs, 13)) return rc;
  if (T == 0) return GDN_OK;
  const LinPlan pl = lin_plan(B, T, HV, cu_seqlens != nullptr);
  const bool shared = H != HV;
  const LinBwdSpace sp = lin_bwd_space(pl, B, T, HV, K, V);
  if ((pl.split && !states) || (sp.bytes(shared) && (!workspace || workspace_bytes < (size_t)sp.bytes(shared)))) {
    gdn_internal_set_error("gdn_decay_attn_bwd: the forward's states and a workspace of %lld bytes are needed",
                           (long long)sp.bytes(shared));
    return GDN_ERR_INVALID;
  }
  // the last kernel's: the gate's segments, and dq and dk of shared heads
  const int64_t blocks = (dg ? pl.segs * HV : 0) + (shared ? (B * T * H * K / 4 + 255) / 256 : 0);
  if (blocks > kMaxGroups256) {
    gdn_internal_set_error("gdn_decay_attn_bwd: too many tokens and heads for one launch");
    return GDN_ERR_UNSUPPORTED;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int rep = (int)(HV / H);
  char* ws = static_cast<char*>(workspace);
  float* dot_q = reinterpret_cast<float*>(ws + sp.states);
  float* dot_k = reinterpret_cast<float*>(ws + sp.states + sp.dots);
  float* dq_heads = reinterpret_cast<float*>(ws + sp.states + 2 * sp.dots);
  float* dk_heads = reinterpret_cast<float*>(ws + sp.states + 2 * sp.dots + sp.heads);
  LinParams base = lin_params(pl, g, g_dtype, g_batch_stride, g_token_stride, g_head_stride, cu_seqlens, flags, T, N,
                                    HV, scale);
  base.zero_rest = cu_seqlens != nullptr;
  // from the end: the states R at the segments' borders, then dv and dk
  LinParams r = base;
  lin_roles(r, k, rep, q, rep, d_o, 1, nullptr, 1, K, V);
  lin_states(r, pl, ws, K, V);
  r.init = d_final_state;
  if (pl.split) launch_segments<true>(r, pl, K, V, s);
  LinParams v_ = r, k_ = r, q_ = base;
  v_.o = dv;
  v_.fin = d_initial_state;
  lin_roles(k_, v, 1, d_o, 1, q, rep, k, rep, V, K);
  k_.transposed = 1;
  k_.dot = dot_k;
  k_.o = shared ? static_cast<void*>(dk_heads) : dk;
  // from the start: dq
  lin_roles(q_, d_o, 1, v, 1, k, rep, q, rep, V, K);
  lin_states(q_, pl, static_cast<char*>(const_cast<void*>(states)), K, V);
  q_.init = initial_state;
  q_.transposed = 1;
  q_.dot = dot_q;
  q_.o = shared ? static_cast<void*>(dq_heads) : dq;
  const dim3 grid((unsigned)(pl.segs * HV), 3), nt(kWalkThreads);
  lin_by_dims(K, V, [&](auto kd, auto vd) {
    constexpr int KD = decltype(kd)::value, VD = decltype(vd)::value;
    if (dg && shared) hipLaunchKernelGGL((gated_deltaless_chunk_bwd_kernel<KD, VD, true, float>), grid, nt, 0, s, q_, k_, v_);
    else if (dg) hipLaunchKernelGGL((gated_deltaless_chunk_bwd_kernel<KD, VD, true, bf16>), grid, nt, 0, s, q_, k_, v_);
    else if (shared) hipLaunchKernelGGL((gated_deltaless_chunk_bwd_kernel<KD, VD, false, float>), grid, nt, 0, s, q_, k_, v_);
    else hipLaunchKernelGGL((gated_deltaless_chunk_bwd_kernel<KD, VD, false, bf16>), grid, nt, 0, s, q_, k_, v_);
  });
  if (dg || shared) {
    const LinFinish fin{dot_q, dot_k, q_.entry, r.entry, final_state, d_final_state, initial_state, d_initial_state, dg, g_dtype,
                        (int)(K * V), (int)pl.segs, dq_heads, dk_heads, static_cast<bf16*>(dq), static_cast<bf16*>(dk), rep,
                        (int)K};
    hipLaunchKernelGGL(gated_deltaless_finish_kernel, dim3((unsigned)blocks, shared ? 2 : 1), dim3(256), 0, s, base, fin);
  }
  return gdn_internal_check_launch("gated_deltaless_chunk_bwd_kernel");
}
