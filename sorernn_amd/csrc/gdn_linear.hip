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
// A workgroup of V / 16 waves walks one segment of a sequence for one value head. The state stays in fp32 MFMA
// accumulators, wave w holding all K rows of 16 columns; it is the A operand of S^T Q^T as it stands, split into
// bf16 parts in registers. Sequences are cut into segments so that few heads fill the chip: a first kernel walks
// the segments for their own contribution to the state (k and v only), a scan over the segments turns these into the
// states that enter them, and the walkers then run side by side.
//
// Rounding: q, k, v and do are bf16 operands as they come. What is computed is split into bf16 parts that are multiplied
// one by one: three (24 bits, as fp32 holds) where the result is an fp32 output (the state, and what dg sums), two
// where the outputs are rounded to bf16 (scores, and the state under o): a single part's 2^-9 would be as large as the
// rounding of the output itself. The decays are summed in 64 bits: a difference of two sums in 32 would carry the
// rounding of the sums into every weight.

#include <type_traits>

#include "gdn_mfma.h"

namespace gdn {

struct LinParams {
  const bf16 *q, *k, *v, *e;    // [tokens][heads][K or V]: the walk's q, k, v and the rows of the gate's dot products
  int64_t qs, ks, vs, es;       // elements between tokens
  unsigned rq, rk, rv, re;      // value heads that share a head of each
  const void* g;                // log decays, or null: no decay
  int dg;
  int64_t gb, gt, gh;           // element strides of batch row, token and value head
  const float* init;            // [N][HV][K][V] state before the walk, or null: zeros
  float* entry;                 // [slots][HV][K][V] states entering the segments, or null: one segment a sequence
  float* decay;                 // [slots][HV] decay of a whole segment
  int transposed;               // init and entry are read as [V][K]
  float* fin;                   // [N][HV][K][V] state after the walk, or null
  void* o;                      // [tokens][HV][V]
  float* dot;                   // [HV][tokens] with DOT
  const void* cu;
  int cu_i32, shift;            // segments of 1 << shift tokens
  int64_t T, N;
  unsigned HV, spq;             // spq: segments of a sequence without cu
  float scale;
};

// Where a workgroup works: sequence n, the segment's first token (flat) and length, and its place in the sequence.
struct Segment {
  int64_t n, slot, tok, row, col;  // row, col: batch row and first token in it (the gate's strides)
  int len;
  bool first, last, some;
};

// Slots of a sequence: with cu, sequence n has the slots from (cu[n] >> shift) + n on, which leaves room for its
// segments whatever the lengths are, so that the grid depends on T and N alone. All lanes of a wave search together.
__device__ __forceinline__ Segment find_segment(const LinParams& p, unsigned slot) {
  Segment s;
  int64_t bos, len, local;
  const int64_t L = (int64_t)1 << p.shift;
  if (p.cu) {
    const int lane = threadIdx.x % kWave;
    int64_t lo = 0, hi = p.N;  // first slot of sequence lo <= slot < that of sequence hi
    while (hi - lo > 1) {
      const int64_t step = (hi - lo + kWave - 1) / kWave, i = lo + lane * step;
      const bool in = i < hi && (load_index(p.cu, p.cu_i32, i < hi ? i : lo) >> p.shift) + i <= slot;
      const int cnt = __popcll(__ballot(in));  // one at least: lane 0's
      lo += (cnt > 1 ? cnt - 1 : 0) * step;
      hi = lo + step < hi ? lo + step : hi;
    }
    s.n = lo;
    bos = load_index(p.cu, p.cu_i32, lo);
    len = load_index(p.cu, p.cu_i32, lo + 1) - bos;
    local = slot - ((bos >> p.shift) + lo);
    s.row = 0;
    s.col = bos + local * L;
  } else {
    s.n = slot / p.spq;
    local = slot % p.spq;
    bos = s.n * p.T;
    len = p.T;
    s.row = s.n;
    s.col = local * L;
  }
  s.slot = slot;
  s.tok = bos + local * L;
  const int64_t left = len - local * L;
  s.some = left > 0;
  s.len = (int)(left < L ? left : L);
  s.first = local == 0;
  s.last = left <= L;
  return s;
}

// Decay terms of a chunk, base-2 logarithms: b = h + l in two floats, the weight of a token in the state's update and
// that of the state in a token's output (each with the factor it carries), and the decay of the whole chunk.
struct Decays {
  float h[kC], l[kC], wst[kC], win[kC];
  float all;
};

template <int CTRL, int ROW_MASK>
__device__ __forceinline__ double dpp_scan_step(double v) {
  const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROW_MASK, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROW_MASK, 0xf, false);
  return v + __hiloint2double(hi, lo);
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
  x = dpp_scan_step<0x111, 0xf>(x);
  x = dpp_scan_step<0x112, 0xf>(x);
  x = dpp_scan_step<0x114, 0xf>(x);
  x = dpp_scan_step<0x118, 0xf>(x);
  x = dpp_scan_step<0x142, 0xa>(x);
  x = dpp_scan_step<0x143, 0xc>(x);
  const double all = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), kWave - 1),
                                      __builtin_amdgcn_readlane(__double2loint(x), kWave - 1));
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
  __device__ __forceinline__ void load(const float* src, bool transposed, int w, int lane) {
    const int g = lane >> 4, i = lane & 15;
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
        if (transposed) {
          s[a][ct] = *reinterpret_cast<const f32x4*>(src + col(w, ct, i) * KD + row0(a, g));
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) s[a][ct][r] = src[(row0(a, g) + r) * VD + col(w, ct, i)];
        }
      }
  }
  __device__ __forceinline__ void store(float* dst, int pitch, int w, int lane) const {
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

__device__ __forceinline__ uint32_t gate_raw(const LinParams& p, const Segment& sg, unsigned hv, int t) {
  return load_raw32(p.g, p.dg, sg.row * p.gb + (sg.col + t) * p.gt + hv * p.gh);
}

// The gate of a segment's chunks in walking order, read by one wave: the raw values of the chunk after the next in flight.
template <bool REV>
struct GateWalk {
  uint32_t raw = 0;
  __device__ __forceinline__ void fetch(const LinParams& p, const Segment& sg, unsigned hv, int ci, int nc, int lane) {
    const int t = (REV ? nc - 1 - ci : ci) * kC + lane;
    raw = p.g && ci < nc && t < sg.len ? gate_raw(p, sg, hv, t) : 0u;
  }
  __device__ __forceinline__ double value(const LinParams& p) const { return p.g ? log2_decay(raw, p.dg) : 0.; }
};

// ------------------------------------------------------------------------------------------------
// A segment's own contribution to the state: the walk without outputs, from a zero state. Forward walks leave it in
// the next segment's slot, walks from the end in the one before; the sequence's last segment (first) has none to give.
// Two workgroups share 128 columns, which doubles the waves in flight.
template <int KD, bool REV>
__global__ __launch_bounds__(256, 3) void gated_deltaless_segment_kernel(LinParams p, int VD) {
  __shared__ __align__(16) bf16 Ks[kC * KD], Vs[kC * 64];
  __shared__ __align__(16) Decays d[2];
  const int lane = threadIdx.x % kWave, w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const unsigned hv = blockIdx.x % p.HV;
  const Segment sg = find_segment(p, blockIdx.x / p.HV);
  if (!sg.some || (REV ? sg.first : sg.last)) return;
  const bf16* k0 = p.k + sg.tok * p.ks + hv / p.rk * KD;
  const bf16* v0 = p.v + sg.tok * p.vs + hv / p.rv * VD + blockIdx.y * 64;
  const int nc = (sg.len + kC - 1) / kC;
  Tile<KD> kt;
  Tile<64> vt;
  GateWalk<REV> gate;
  const uint32_t koff = kt.offset(p.ks), voff = vt.offset(p.vs);
  auto fetch = [&](int ci) {
    const int t0 = (REV ? nc - 1 - ci : ci) * kC, len = sg.len - t0 < kC ? sg.len - t0 : kC;
    kt.fetch(k0 + t0 * p.ks, p.ks, koff, len);
    vt.fetch(v0 + t0 * p.vs, p.vs, voff, len);
  };
  State<KD, 64, 4> st;
  st.zero();
  double total = 0.;
  if (w == 0) gate.fetch(p, sg, hv, 0, nc, lane);
  fetch(0);
  if (w == 0) {
    total = gate.value(p);
    chunk_decays<REV>(d[0], total, p.scale, lane);
    gate.fetch(p, sg, hv, 1, nc, lane);
  }
  for (int ci = 0; ci < nc; ++ci) {
    const int t0 = (REV ? nc - 1 - ci : ci) * kC, len = sg.len - t0 < kC ? sg.len - t0 : kC;
    kt.put(Ks, len);
    vt.put(Vs, len);
    __syncthreads();
    if (ci + 1 < nc) fetch(ci + 1);
    if (w == 0 && ci + 1 < nc) {
      const double x = gate.value(p);
      total += x;
      chunk_decays<REV>(d[(ci + 1) & 1], x, p.scale, lane);
      gate.fetch(p, sg, hv, ci + 2, nc, lane);
    }
    bf16x8 vf[2][1];
    st.columns(Vs, 0, w, lane, vf[0]);
    st.columns(Vs, 32, w, lane, vf[1]);
    st.update(d[ci & 1], Ks, vf, lane);
    __syncthreads();
  }
  st.store(p.entry + ((sg.slot + (REV ? -1 : 1)) * p.HV + hv) * (KD * VD) + blockIdx.y * 64, VD, w, lane);
  if (w == 0 && blockIdx.y == 0) {
    for (int m = 1; m < kWave; m <<= 1) total += __shfl_xor(total, m, kWave);
    if (lane == 0) p.decay[sg.slot * p.HV + hv] = __builtin_amdgcn_exp2f((float)total);
  }
}

// The segments' contributions into the states entering them, in place: entry[s] += decay[s - 1] entry[s - 1] (from the
// end: decay[s + 1] entry[s + 1]), four neighbouring elements a thread.
template <bool REV>
__global__ __launch_bounds__(256) void gated_deltaless_scan_kernel(LinParams p, int64_t elems) {
  const unsigned per = (unsigned)elems / 1024, chain = blockIdx.x / per, hv = chain % p.HV, n = chain / p.HV;
  const int64_t at = (blockIdx.x % per) * 1024 + threadIdx.x * 4;
  int64_t slot0, cnt;
  if (p.cu) {
    const int64_t bos = load_index(p.cu, p.cu_i32, n), eos = load_index(p.cu, p.cu_i32, (int64_t)n + 1);
    slot0 = (bos >> p.shift) + n;
    cnt = (eos - bos + ((int64_t)1 << p.shift) - 1) >> p.shift;
  } else {
    slot0 = (int64_t)n * p.spq;
    cnt = p.spq;
  }
  if (cnt < 2) return;
  const int64_t step = (int64_t)p.HV * elems;
  float* e = p.entry + (slot0 * p.HV + hv) * elems + at;
  const float* dc = p.decay + slot0 * p.HV + hv;
  f32x4 run = {0.f, 0.f, 0.f, 0.f};
  if (p.init) run = *reinterpret_cast<const f32x4*>(p.init + chain * elems + at);
  constexpr int U = 4;  // loads in flight
  for (int64_t s0 = 0; s0 < cnt - 1; s0 += U) {
    f32x4 x[U];
    float c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t s = s0 + u < cnt - 1 ? s0 + u : cnt - 2;
      x[u] = *reinterpret_cast<const f32x4*>(e + (REV ? cnt - 2 - s : s + 1) * step);
      c[u] = dc[(REV ? cnt - 1 - s : s) * p.HV];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u >= cnt - 1) break;
      run = run * c[u] + x[u];
      *reinterpret_cast<f32x4*>(e + (REV ? cnt - 2 - s0 - u : s0 + u + 1) * step) = run;
    }
  }
}

// ------------------------------------------------------------------------------------------------
// The walk. One workgroup a CU: waves 0-3 hold the state and make the outputs of chunk c, waves 4-7 meanwhile bring the
// tiles of chunks c + 1 and c + 2 into LDS and make the scores of chunk c + 1; one barrier a chunk. At 4 x 4,096 tokens, 16 heads of 128, 82 us;
// its loads and stores alone 59 us, the state's waves alone 64 us.
// DOT 1 also gives e_i . (the state's share of o_i) for every token; DOT 2 adds the scores' share, the row sums less the
// column sums of W_ij = P_ij (e_i . v_j), exact bf16 products summed in fp32.
//
// Scores are kept for the tiles that are not masked, in blocks of 16 queries x 32 keys (tok_col order): queries 0-15 and
// 16-31 have one block, the others two (walks from the end: mirrored).
template <int KD, int VD, int DOT>
struct WalkLds {
  bf16 q[3][kC * KD], k[3][kC * KD], v[2][kC * VD];
  bf16 ps[2][2][6 * 512];  // [slot][part]
  Decays d[3];
  float dots[DOT ? 2 : 1][4][DOT ? kC : 1];
  float rows[DOT == 2 ? 2 : 1][10][DOT == 2 ? 16 : 1], cols[DOT == 2 ? 2 : 1][10][DOT == 2 ? 16 : 1];
};

template <int KD, int VD, bool REV, int DOT, typename OT>
__global__ __launch_bounds__(512, 2) void gated_deltaless_chunk_kernel(LinParams p) {
  constexpr int SW = 4, NCT = VD / 16 / SW, NU = KD / 32;
  constexpr int NS = DOT ? 3 : 2;  // parts of the state under o
  __shared__ __align__(16) WalkLds<KD, VD, DOT> lds;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int g = lane >> 4, i = lane & 15;
  const unsigned hv = blockIdx.x % p.HV;
  const Segment sg = find_segment(p, blockIdx.x / p.HV);
  if (!sg.some) return;
  const int nc = (sg.len + kC - 1) / kC;
  auto first_of = [&](int c) { return (REV ? nc - 1 - c : c) * kC; };  // first token of the walk's chunk c
  auto len_of = [&](int c) { return sg.len - first_of(c) < kC ? sg.len - first_of(c) : kC; };
  const bf16* e0 = DOT ? p.e + sg.tok * p.es + hv / p.re * VD : nullptr;

  if (wave < SW) {  // ------------------------------------------------------------------ the state's waves
    const int w = wave;
    OT* o0 = static_cast<OT*>(p.o) + (sg.tok * p.HV + hv) * VD;
    State<KD, VD, SW> st;
    const bool inner = REV ? !sg.last : !sg.first;  // a segment of this sequence comes before
    const float* src = inner ? p.entry + (sg.slot * p.HV + hv) * (KD * VD)
                             : (p.init ? p.init + (sg.n * p.HV + hv) * (KD * VD) : nullptr);
    if (src) st.load(src, p.transposed, w, lane);
    else st.zero();
    const bool wants_fin = p.fin && (REV ? sg.first : sg.last);
    __syncthreads();
    __syncthreads();
    for (int c = 0; c < nc; ++c) {
      const int t0 = first_of(c), len = len_of(c);
      const Decays& d = lds.d[c % 3];
      const bf16 *Qs = lds.q[c % 3], *Ks = lds.k[c % 3], *Vs = lds.v[c & 1];
      bf16x4 ev[4][NCT];
      if (DOT) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int row = 16 * t + i;
          const bf16* er = e0 + (t0 + (row < len ? row : 0)) * p.es + 16 * NCT * w + 4 * NCT * g;
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) ev[t][ct] = *reinterpret_cast<const bf16x4*>(er + 4 * ct);
        }
      }
      // the state's share: O^T = S^T Q^T, columns = tokens
      f32x4 acc[4][NCT];
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
            for (int ct = 0; ct < NCT; ++ct) acc[t][ct] = mma(part[ct][n], qf[t], acc[t][ct]);
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
          float x = 0.f;
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
            for (int r = 0; r < 4; ++r) x += acc[t][ct][r] * (float)ev[t][ct][r];
          x = xor32_sum(xor16_sum(x));
          if (g == 0) lds.dots[DOT ? c & 1 : 0][w][DOT ? 16 * t + i : 0] = x;
        }
      }
      // the scores' share: O^T += V^T P^T
      bf16x8 vf[2][NCT];
      float bad = 0.f;  // NaN where the wave's columns of v hold an infinity or NaN: a sum of products with zero
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        State<KD, VD, SW>::columns(Vs, 32 * k2, w, lane, vf[k2]);
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
      if (c + 1 < nc || wants_fin) st.update(d, Ks, vf, lane);
      __syncthreads();
    }
    if (wants_fin) st.store(p.fin + (sg.n * p.HV + hv) * (KD * VD), VD, w, lane);
    return;
  }

  // ------------------------------------------------------------------------------------ the scores' waves
  const int w = wave - SW;
  const bf16* q0 = p.q + sg.tok * p.qs + hv / p.rq * KD;
  const bf16* k0 = p.k + sg.tok * p.ks + hv / p.rk * KD;
  const bf16* v0 = p.v + sg.tok * p.vs + hv / p.rv * VD;
  // Two sets of tiles in flight: a chunk's loads are issued two steps before their rows go to LDS. With one step between
  // the two, a step lasted as long as the loads of all CUs took, and the memory had nothing to do meanwhile.
  Tile<KD> qt[2], kt[2];
  Tile<VD> vt[2];
  const uint32_t qoff = qt[0].offset(p.qs), koff = kt[0].offset(p.ks), voff = vt[0].offset(p.vs);
  auto fetch_qk = [&](int c, int set) {
    if (c >= nc) return;
    const int t0 = first_of(c), len = len_of(c);
    qt[set].fetch(q0 + t0 * p.qs, p.qs, qoff, len);
    kt[set].fetch(k0 + t0 * p.ks, p.ks, koff, len);
  };
  auto fetch_v = [&](int c, int set) {
    if (c < nc) vt[set].fetch(v0 + first_of(c) * p.vs, p.vs, voff, len_of(c));
  };
  auto put_qk = [&](int c, int set) {
    if (c >= nc) return;
    qt[set].put(lds.q[c % 3], len_of(c));
    kt[set].put(lds.k[c % 3], len_of(c));
  };
  auto put_v = [&](int c, int set) {
    if (c < nc) vt[set].put(lds.v[c & 1], len_of(c));
  };
  GateWalk<REV> gate;
  auto decays = [&](int c) {  // of chunk c, whose raw gate has been fetched; then the next chunk's
    if (w != 0 || c >= nc) return;
    chunk_decays<REV>(lds.d[c % 3], gate.value(p), p.scale, lane);
    gate.fetch(p, sg, hv, c + 1, nc, lane);
  };
  // 12 tiles of 16 keys x 16 queries are written (2 of zeros), 3 a wave: P^T, rows = keys j, column = query
  f32x4 pv[3];
  auto tile_of = [&](int n, int& ta, int& ja) {
    const int sl = w + 4 * n;
    ta = n == 0 ? sl >> 1 : 1 + n;
    ja = n == 0 ? sl & 1 : w;
  };
  auto scores = [&](int c) {
    if (c >= nc) return;
    const bf16 *Qs = lds.q[c % 3], *Ks = lds.k[c % 3];
    const Decays& d = lds.d[c % 3];
    auto* ps = lds.ps[c & 1];
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
  auto score_dots = [&](int c, const f32x4 (&x)[3]) {
    const int t0 = first_of(c), len = len_of(c);
    const bf16* Vs = lds.v[c & 1];
#pragma unroll
    for (int n = 0; n < 3; ++n) {
      int ta, ja;
      tile_of(n, ta, ja);
      if (ja > ta) continue;
      const int t = REV ? 3 - ta : ta, jt = REV ? 3 - ja : ja, iq = 16 * t + i;
      const bf16* er = e0 + (t0 + (iq < len ? iq : 0)) * p.es + 8 * g;
      f32x4 a = {0.f, 0.f, 0.f, 0.f}, cs;
#pragma unroll
      for (int u = 0; u < VD / 32; ++u) a = mma(ld_row<VD>(Vs, 16 * jt + i, 4 * u + g), ld8(er + 32 * u), a);
      float rs = 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 16 * jt + 4 * g + r;
        const float ww = (REV ? j >= iq : j <= iq) && iq < len && j < len ? x[n][r] * a[r] : 0.f;
        rs += ww;
        cs[r] = group_sum<16>(ww);
      }
      rs = xor32_sum(xor16_sum(rs));
      const int idx = ta * (ta + 1) / 2 + ja, sl = DOT == 2 ? c & 1 : 0;
      if (g == 0) lds.rows[sl][idx][DOT == 2 ? i : 0] = rs;
      if (i == 0) *reinterpret_cast<f32x4*>(&lds.cols[sl][idx][DOT == 2 ? 4 * g : 0]) = cs;
    }
  };
  // the gate's dot products of chunk c, all of whose shares are in LDS
  auto finish_dots = [&](int c) {
    if (!DOT || c < 0 || w != 1 || lane >= len_of(c)) return;
    const int sl = DOT ? c & 1 : 0;
    float x = 0.f;
#pragma unroll
    for (int ww = 0; ww < SW; ++ww) x += lds.dots[sl][ww][DOT ? lane : 0];
    if (DOT == 2) {
      const int ta = REV ? 3 - g : g;  // the token's tile, as query and as key
#pragma unroll
      for (int o = 0; o < 4; ++o) {
        if (o <= ta) x += lds.rows[DOT == 2 ? sl : 0][ta * (ta + 1) / 2 + o][DOT == 2 ? i : 0];
        if (o >= ta) x -= lds.cols[DOT == 2 ? sl : 0][o * (o + 1) / 2 + ta][DOT == 2 ? i : 0];
      }
    }
    const int64_t tokens = p.cu ? p.T : p.N * p.T;
    p.dot[hv * tokens + sg.tok + first_of(c) + lane] = x;
  };
  if (w == 0) gate.fetch(p, sg, hv, 0, nc, lane);
  fetch_qk(0, 0);
  fetch_v(0, 0);
  fetch_qk(1, 1);
  fetch_v(1, 1);
  decays(0);
  decays(1);
  put_qk(0, 0);
  fetch_qk(2, 0);
  put_v(0, 0);
  fetch_v(2, 0);
  put_qk(1, 1);
  fetch_qk(3, 1);
  __syncthreads();
  scores(0);
  __syncthreads();
  auto step = [&](int c, int set) {  // set: c & 1
    put_v(c + 1, 1 - set);
    fetch_v(c + 3, 1 - set);
    put_qk(c + 2, set);
    fetch_qk(c + 4, set);
    decays(c + 2);
    f32x4 held[3];
    if (DOT == 2) {
#pragma unroll
      for (int n = 0; n < 3; ++n) held[n] = pv[n];
    }
    scores(c + 1);
    if (DOT == 2) score_dots(c, held);
    finish_dots(c - 1);
    __syncthreads();
  };
  for (int c = 0; c < nc; c += 2) {
    step(c, 0);
    if (c + 1 < nc) step(c + 1, 1);
  }
  finish_dots(nc - 1);
}

// ------------------------------------------------------------------------------------------------
// dg of a segment: what lies behind it is <S, R> at its end (the state entering the next segment with what the walk from
// the end brings there; <S_T, dS_T> at the sequence's end), then the sum from the end of q . dq - k . dk.
struct LinGateGrad {
  const float *x, *y;              // [HV][tokens] q . dq and k . dk
  const float *entry, *rentry;     // the states at the segments' borders, or null
  const float *fin, *dfin;         // at the sequences' ends; either may be null (dfin: a zero gradient)
  void* out;                       // [tokens][HV]
  int dtype;
  int64_t elems;                   // K V
};

__global__ __launch_bounds__(256) void gated_deltaless_gate_grad_kernel(LinParams p, LinGateGrad a) {
  __shared__ double part[4];
  const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
  const unsigned hv = blockIdx.x % p.HV;
  const Segment sg = find_segment(p, blockIdx.x / p.HV);
  if (!sg.some) return;
  const float *s = nullptr, *r = nullptr;
  if (!sg.last) {
    s = a.entry + ((sg.slot + 1) * p.HV + hv) * a.elems;
    r = a.rentry + (sg.slot * p.HV + hv) * a.elems;
  } else if (a.fin && a.dfin) {
    s = a.fin + (sg.n * p.HV + hv) * a.elems;
    r = a.dfin + (sg.n * p.HV + hv) * a.elems;
  }
  double sum = 0.;
  if (s) {
    for (int64_t at = threadIdx.x * 4; at < a.elems; at += 1024) {
      const f32x4 u = *reinterpret_cast<const f32x4*>(s + at), v = *reinterpret_cast<const f32x4*>(r + at);
      sum += (double)(u[0] * v[0] + u[1] * v[1]) + (double)(u[2] * v[2] + u[3] * v[3]);
    }
    for (int m = 1; m < kWave; m <<= 1) sum += __shfl_xor(sum, m, kWave);
    if (lane == 0) part[w] = sum;
    __syncthreads();
    sum = part[0] + part[1] + part[2] + part[3];
    __syncthreads();
  }
  const int64_t tokens = p.cu ? p.T : p.N * p.T, base = hv * tokens + sg.tok;
  for (int hi = sg.len; hi > 0; hi -= 256) {  // 256 tokens a step: wave w those from hi - 64 (w + 1) on
    const int t = hi - kWave * (w + 1) + lane;
    const double x = t >= 0 ? (double)a.x[base + t] - (double)a.y[base + t] : 0.;
    double run = x;
    for (int m = 1; m < kWave; m <<= 1) {
      const double other = __shfl_down(run, m, kWave);
      if (lane + m < kWave) run += other;
    }
    if (lane == 0) part[w] = run;
    __syncthreads();
    for (int ww = 0; ww < 4; ++ww) {
      if (ww < w) run += part[ww];
    }
    if (t >= 0) store_from_f32(a.out, a.dtype, (sg.tok + t) * p.HV + hv, (float)(sum + run));
    sum += part[0] + part[1] + part[2] + part[3];
    __syncthreads();
  }
}

// Sums the gradients of the value heads that share a q/k head: [rows][rep][D] fp32 -> [rows][D] bf16.
__global__ __launch_bounds__(256) void gated_deltaless_head_sum_kernel(const float* x, bf16* y, int64_t rows, int rep, int D) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= rows * D) return;
  const float* src = x + at / D * rep * D + at % D;
  f32x4 sum = *reinterpret_cast<const f32x4*>(src);
  for (int r = 1; r < rep; ++r) sum += *reinterpret_cast<const f32x4*>(src + (int64_t)r * D);
  *reinterpret_cast<bf16x4*>(y + at) = to_bf16x4(sum[0], sum[1], sum[2], sum[3]);
}

// ------------------------------------------------------------------------------------------------
// host
struct LinPlan {
  int shift;
  int64_t spq, slots;  // segments of a sequence without cu, slots in all
  bool split;
};

// Segments of a power of two of tokens, as short as gives kLinGroups workgroups and no shorter than kLinMinSegment.
constexpr int64_t kLinGroups = 256, kLinMinSegment = 256;

static LinPlan lin_plan(int64_t B, int64_t T, int64_t HV, int64_t N, bool varlen) {
  LinPlan pl{};
  int64_t L = kLinMinSegment;
  pl.shift = 8;
  while (L < T && (B * T / L) * HV > kLinGroups) {
    L <<= 1;
    ++pl.shift;
  }
  pl.spq = T > L ? (T + L - 1) / L : 1;
  pl.slots = varlen ? (T >> pl.shift) + N : N * pl.spq;
  pl.split = T > L;
  return pl;
}

static int64_t align256l(int64_t b) { return (b + 255) / 256 * 256; }
static int64_t lin_states_bytes(const LinPlan& pl, int64_t HV, int64_t K, int64_t V) {
  return pl.split ? align256l(pl.slots * HV * K * V * 4) + align256l(pl.slots * HV * 4) : 0;
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
  const dim3 grid((unsigned)(pl.slots * p.HV), (unsigned)(V / 64));
  if (K == 128) hipLaunchKernelGGL((gated_deltaless_segment_kernel<128, REV>), grid, dim3(256), 0, s, p, (int)V);
  else hipLaunchKernelGGL((gated_deltaless_segment_kernel<64, REV>), grid, dim3(256), 0, s, p, (int)V);
  hipLaunchKernelGGL((gated_deltaless_scan_kernel<REV>), dim3((unsigned)(p.N * p.HV * (K * V / 1024))), dim3(256), 0, s, p,
                     K * V);
}

template <bool REV, int DOT, typename OT>
static void launch_walk(const LinParams& p, const LinPlan& pl, int64_t K, int64_t V, hipStream_t s) {
  lin_by_dims(K, V, [&](auto k, auto v) {
    hipLaunchKernelGGL((gated_deltaless_chunk_kernel<decltype(k)::value, decltype(v)::value, REV, DOT, OT>),
                       dim3((unsigned)(pl.slots * p.HV)), dim3(512), 0, s, p);
  });
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
  const LinPlan pl = lin_plan(B, T, HV, N, varlen);
  if (HV > 65536 || pl.slots * HV > 0x7fffffffLL || pl.spq > 0x7fffffffLL || N * HV * 16 > 0x7fffffffLL || B * T * HV > (1LL << 40)) {
    gdn_internal_set_error("%s: too many sequences, heads or tokens for one launch", name);
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
  p.shift = pl.shift;
  p.T = T;
  p.N = N;
  p.HV = (unsigned)HV;
  p.spq = (unsigned)pl.spq;
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
  p.decay = pl.split ? reinterpret_cast<float*>(states + align256l(pl.slots * p.HV * K * V * 4)) : nullptr;
}

}  // namespace gdn

using namespace gdn;

extern "C" size_t gdn_decay_attn_states_size(int64_t B, int64_t T, int64_t HV, int64_t K, int64_t V, int64_t N, int varlen) {
  if (B <= 0 || T < 0 || HV <= 0 || K <= 0 || V <= 0 || N <= 0) return 0;
  return (size_t)lin_states_bytes(lin_plan(B, T, HV, N, varlen != 0), HV, K, V);
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
  const LinPlan pl = lin_plan(B, T, HV, N, cu_seqlens != nullptr);
  const size_t need = (size_t)lin_states_bytes(pl, HV, K, V);
  if (need && (!states || states_bytes < need)) {
    gdn_internal_set_error("gdn_decay_attn_fwd: states of %zu bytes needed", need);
    return GDN_ERR_INVALID;
  }
  if (T == 0) return GDN_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int rep = (int)(HV / H);
  LinParams p = lin_params(pl, g, g_dtype, g_batch_stride, g_token_stride, g_head_stride, cu_seqlens, flags, T, N, HV, scale);
  lin_roles(p, q, rep, k, rep, v, 1, nullptr, 1, K, V);
  lin_states(p, pl, static_cast<char*>(states), K, V);
  p.init = initial_state;
  if (pl.split) launch_segments<false>(p, pl, K, V, s);
  p.fin = final_state;
  p.o = o;
  launch_walk<false, 0, bf16>(p, pl, K, V, s);
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
  if (B <= 0 || T < 0 || H <= 0 || HV <= 0 || HV % H || K <= 0 || V <= 0 || N <= 0) return 0;
  return (size_t)lin_bwd_space(lin_plan(B, T, HV, N, varlen != 0), B, T, HV, K, V).bytes(HV != H);
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
  const LinPlan pl = lin_plan(B, T, HV, N, cu_seqlens != nullptr);
  const bool shared = H != HV;
  const LinBwdSpace sp = lin_bwd_space(pl, B, T, HV, K, V);
  if ((pl.split && !states) || (sp.bytes(shared) && (!workspace || workspace_bytes < (size_t)sp.bytes(shared)))) {
    gdn_internal_set_error("gdn_decay_attn_bwd: the forward's states and a workspace of %lld bytes are needed",
                           (long long)sp.bytes(shared));
    return GDN_ERR_INVALID;
  }
  if (T == 0) return GDN_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int rep = (int)(HV / H);
  char* ws = static_cast<char*>(workspace);
  float* dot_q = reinterpret_cast<float*>(ws + sp.states);
  float* dot_k = reinterpret_cast<float*>(ws + sp.states + sp.dots);
  float* dq_heads = reinterpret_cast<float*>(ws + sp.states + 2 * sp.dots);
  float* dk_heads = reinterpret_cast<float*>(ws + sp.states + 2 * sp.dots + sp.heads);
  const LinParams base = lin_params(pl, g, g_dtype, g_batch_stride, g_token_stride, g_head_stride, cu_seqlens, flags, T, N,
                                    HV, scale);
  // from the end: R's segments, then dv and dk
  LinParams r = base;
  lin_roles(r, k, rep, q, rep, d_o, 1, nullptr, 1, K, V);
  lin_states(r, pl, ws, K, V);
  r.init = d_final_state;
  if (pl.split) launch_segments<true>(r, pl, K, V, s);
  LinParams a = r;
  a.o = dv;
  a.fin = d_initial_state;
  launch_walk<true, 0, bf16>(a, pl, K, V, s);
  a = r;
  lin_roles(a, v, 1, d_o, 1, q, rep, k, rep, V, K);
  a.transposed = 1;
  a.dot = dot_k;
  a.o = shared ? static_cast<void*>(dk_heads) : dk;
  if (shared) dg ? launch_walk<true, 1, float>(a, pl, V, K, s) : launch_walk<true, 0, float>(a, pl, V, K, s);
  else dg ? launch_walk<true, 1, bf16>(a, pl, V, K, s) : launch_walk<true, 0, bf16>(a, pl, V, K, s);
  // from the start: dq
  LinParams f = base;
  lin_roles(f, d_o, 1, v, 1, k, rep, q, rep, V, K);
  lin_states(f, pl, static_cast<char*>(const_cast<void*>(states)), K, V);
  f.init = initial_state;
  f.transposed = 1;
  f.dot = dot_q;
  f.o = shared ? static_cast<void*>(dq_heads) : dq;
  if (shared) dg ? launch_walk<false, 2, float>(f, pl, V, K, s) : launch_walk<false, 0, float>(f, pl, V, K, s);
  else dg ? launch_walk<false, 2, bf16>(f, pl, V, K, s) : launch_walk<false, 0, bf16>(f, pl, V, K, s);
  if (dg) {
    const LinGateGrad gg{dot_q, dot_k, f.entry, r.entry, final_state, d_final_state, dg, g_dtype, K * V};
    hipLaunchKernelGGL(gated_deltaless_gate_grad_kernel, dim3((unsigned)(pl.slots * HV)), dim3(256), 0, s, base, gg);
  }
  if (shared) {
    const int64_t rows = B * T * H, blocks = (rows * K / 4 + 255) / 256;
    hipLaunchKernelGGL(gated_deltaless_head_sum_kernel, dim3((unsigned)blocks), dim3(256), 0, s, dq_heads,
                       static_cast<bf16*>(dq), rows, rep, (int)K);
    hipLaunchKernelGGL(gated_deltaless_head_sum_kernel, dim3((unsigned)blocks), dim3(256), 0, s, dk_heads,
                       static_cast<bf16*>(dk), rows, rep, (int)K);
  }
  return gdn_internal_check_launch("gated_deltaless_chunk_kernel(bwd)");
}
