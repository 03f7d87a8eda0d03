// A paged cache of keys and values: new tokens' rows normed, rotated and put into their pages, and the attention that reads
// them: single tokens, pieces of a prompt, and trees of drafted tokens, causal at the cache's end, with a window and sinks.
//
//   cache [pages, HKV, page, D]; token s of sequence n lies at row s % page of page table[n][s / page]
//   lengths[n]: the sequence's tokens with the T_n new ones counted: new token t is at place lengths[n] - T_n + t
//
// Nothing that the table, the lengths or the bounds hold leads outside the tensors: a page number that is none is read as
// keys that nobody sees and is not written, a length as at most what a row of the table can hold.

#include <math.h>

#include <type_traits>

#include "gdn_flash.h"

namespace gdn {

// ------------------------------------------------------------------------------------------------ append
// k' = rotate(norm(k)) and v into their places, q' = rotate(norm(q)) beside them, fp32 with one rounding. Bound by the rows'
// bytes, or by the launch where tokens are few. A wave takes a token (with few tokens four share one) and its heads D / 16 lanes
// each; a lane holds two pieces of 8 elements that turn with one another. Angles are taken in turns in 64 bits,
// position * (theta^(-2f / rot) / 2 pi) less its whole part: at position 1,000,000 a 32-bit angle is off by 0.06 rad.
// Measured, 16 query and 4 kv heads of 128: 16,384 tokens 47 us a call, 4.3 TB/s (a large copy: 5.1); one token 4.4 us, 64 tokens
// 5.4 in the kernel.
struct AppendParams {
  const void* x[3];                // q (or null), k, v [B, T, heads, D] by strides (elements)
  int64_t sb[3], st[3], sh[3];
  const float* w[2];               // RMSNorm weights of q, k [D], null: not normed
  void* q_out;                     // [B, T, HQ, D]
  void* cache[2];                  // k, v
  int64_t cp[2], ch[2], ct[2];     // strides between pages, heads, tokens (elements)
  const int* table;
  int64_t table_stride;
  const void *lengths, *pos;       // pos: rotation's positions [B, T] by strides, or null: the tokens' places
  int64_t pb, pt;
  const void* cu;
  int len_i32, pos_i32, cu_i32, width, shift, pages;
  int64_t T, N, tokens;
  int HQ, HKV, rot, wpt;           // HQ 0 without q; wpt: waves that share a token
  float eps;
  double turns[64];                // theta^(-2f / rot) / 2 pi
};

// Up to this many tokens the 4 waves of a workgroup share one.
constexpr int64_t kAppendShared = 256;

template <int D, typename E>
__global__ __launch_bounds__(256) void gated_delta_paged_append_kernel(AppendParams p) {
  constexpr int LPR = D / 16, RPW = kWave / LPR, U = 2;  // lanes a row, rows a pass, passes in flight
  using X8 = typename Pack<E>::x8;
  __shared__ __align__(16) float tab[4][2][D / 2];
  const int lane = threadIdx.x % kWave, w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int li = lane % LPR, sub = lane / LPR, half = p.rot >> 1, np = half >> 3;
  const bool in_rot = li < np;
  const int d0 = in_rot ? 8 * li : p.rot + 16 * (li - np), d1 = in_rot ? d0 + half : d0 + 8;  // the lane's two pieces
  const int rows = p.HQ + 2 * p.HKV, r_first = (w % p.wpt) * RPW + sub, r_step = p.wpt * RPW;
  const int64_t stride = (int64_t)gridDim.x * 4 / p.wpt;
  for (int64_t bt = ((int64_t)blockIdx.x * 4 + w) / p.wpt; bt < p.tokens; bt += stride) {
    const int64_t bi = bt / p.T, ti = bt - bi * p.T;
    auto kind = [&](int r) { return r < p.HQ ? 0 : r < p.HQ + p.HKV ? 1 : 2; };
    auto head = [&](int r, int m) { return r - (m == 0 ? 0 : m == 1 ? p.HQ : p.HQ + p.HKV); };
    X8 xv[U][2];
    auto load = [&](int r0) {  // U passes' rows; past the last the last again
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = imin(r0 + u * r_step, rows - 1), m = kind(r);
        const int64_t sb = m == 0 ? p.sb[0] : m == 1 ? p.sb[1] : p.sb[2], st = m == 0 ? p.st[0] : m == 1 ? p.st[1] : p.st[2];
        const E* base = static_cast<const E*>(m == 0 ? p.x[0] : m == 1 ? p.x[1] : p.x[2]);
        const E* src = base + bi * sb + ti * st + head(r, m) * (m == 0 ? p.sh[0] : m == 1 ? p.sh[1] : p.sh[2]);
        xv[u][0] = *reinterpret_cast<const X8*>(src + d0);
        xv[u][1] = *reinterpret_cast<const X8*>(src + d1);
      }
    };
    load(r_first);
    // the token's sequence, its place there and its row of the cache
    int64_t num = bi, first = 0, count = p.T;
    bool member = true;
    if (p.cu) {
      int64_t below = 0;
      for (int64_t base = 0; base <= p.N; base += kWave) {
        const int64_t j = base + lane;
        const uint64_t m = __ballot(j <= p.N && load_index(p.cu, p.cu_i32, j) <= bt);
        below += __popcll(m);
        if (m != ~0ull) break;
      }
      num = uniform64(below) - 1;
      member = num >= 0 && num < p.N;
      if (member) {
        first = uniform64(load_index(p.cu, p.cu_i32, num));
        count = uniform64(load_index(p.cu, p.cu_i32, num + 1)) - first;
        member = bt - first < count;
      }
    }
    const int64_t length = member ? uniform64(load_index(p.lengths, p.len_i32, num)) : 0;
    const int64_t place = length - count + (p.cu ? bt - first : ti);
    int64_t page = -1;
    if (member && place >= 0 && place < (int64_t)p.width << p.shift && length <= (int64_t)p.width << p.shift) {
      page = __builtin_amdgcn_readfirstlane(p.table[num * p.table_stride + (place >> p.shift)]);
      if (page >= p.pages) page = -1;
    }
    const int64_t in = place & ((1 << p.shift) - 1);
    const int64_t pos = p.pos ? load_index(p.pos, p.pos_i32, bi * p.pb + ti * p.pt) : place;
    for (int f = lane; f < half; f += kWave) {
      const double turn = (double)pos * p.turns[f];
      float sv, cv;
      sincospif(2.f * (float)(turn - rint(turn)), &sv, &cv);
      tab[w][0][f] = cv;
      tab[w][1][f] = sv;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // the table is the wave's own
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    float c[8], s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      c[e] = in_rot ? tab[w][0][d0 + e] : 1.f;  // of others unused
      s[e] = in_rot ? tab[w][1][d0 + e] : 0.f;
    }
    for (int r0 = r_first; r0 < rows; r0 += U * r_step) {  // uniform inside a row's lanes
      if (r0 != r_first) load(r0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * r_step;
        if (r >= rows) break;
        const int m = kind(r), h = head(r, m);
        X8 o0 = xv[u][0], o1 = xv[u][1];
        if (m < 2) {
          const float* wt = m ? p.w[1] : p.w[0];
          float x[16], ss = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            x[e] = (float)xv[u][e >> 3][e & 7];
            ss += x[e] * x[e];
          }
          if (wt) {
            ss = dpp_add<0x4e, 0xf>(dpp_add<0xb1, 0xf>(ss));  // over quads, then over the halves of a row of 16 lanes
            if (LPR == 8) ss = dpp_add<0x141, 0xf>(ss);
            const float rr = 1.f / sqrtf(ss / (float)D + p.eps);
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = x[e] * rr * wt[(e < 8 ? d0 : d1) + (e & 7)];
          }
          // what does not turn stays by itself: times 1 and 0 an infinity would reach the entry beside it
          if (in_rot) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float a = x[e], b = x[8 + e];
              o0[e] = (E)(a * c[e] - b * s[e]);
              o1[e] = (E)(b * c[e] + a * s[e]);
            }
          } else if (wt) {
#pragma unroll
            for (int e = 0; e < 8; ++e) o0[e] = (E)x[e], o1[e] = (E)x[8 + e];
          }
        }
        E* dst;
        if (m == 0) {
          dst = static_cast<E*>(p.q_out) + (bt * p.HQ + h) * D;
          if (!member) o0 = X8{}, o1 = X8{};
        } else {
          if (page < 0) continue;
          const int i = m - 1;
          dst = static_cast<E*>(i ? p.cache[1] : p.cache[0]) + page * (i ? p.cp[1] : p.cp[0]) + h * (i ? p.ch[1] : p.ch[0]) +
                in * (i ? p.ct[1] : p.ct[0]);
        }
        *reinterpret_cast<X8*>(dst + d0) = o0;
        *reinterpret_cast<X8*>(dst + d1) = o1;
      }
    }
    __builtin_amdgcn_wave_barrier();  // the table is read before the next token's is written
  }
}

// ------------------------------------------------------------------------------------------------ attention, many rows
// Tiles of 128 rows (token, q head of the group) of a kv head; where they are few their keys are cut into `splits` runs.
// Measured, 16 heads on 4 of 128: 512 new tokens of 4 sequences over up to 8,192 160 us, 562 TFLOP/s, bound as the forward over whole
// sequences, and 15 us for the join of two runs (without runs 241 us); trees of 61 tokens of 8 sequences over up to 4,096 31 us
// and 9, bound by start and end of runs of 5 to 8 blocks.
template <int D, typename E>
__global__ __launch_bounds__(256, 2) void gated_delta_paged_attn_kernel(FlashParams p) {
  __shared__ __align__(16) E Ks0[kBK * D];
  __shared__ __align__(16) E Ks1[kBK * D];
  __shared__ __align__(16) E Vs0[kBK * D];
  __shared__ __align__(16) E Vs1[kBK * D];
  flash_forward<D, E, true>(p, Ks0, Ks1, Vs0, Vs1);
}

// ------------------------------------------------------------------------------------------------ attention, few new tokens
// A kv head's new rows (token, q head of the group) in tiles of 32; the keys that they see in blocks of 32, cut into `splits`
// runs, a workgroup each. Every wave takes blocks of its own, loaded straight into its own LDS one ahead: no barrier until the
// four waves' sums meet, 128 KB a CU under way. Bound by the cache's bytes: 64 sequences of up to 8,192 tokens, 4 kv heads of 128,
// 147-153 us, 4.6-4.8 TB/s (a large copy: 5.1); with a window of 1,024, 8 kv heads of 64, 31 us, 4.3 TB/s. One token of one
// sequence over 32,768 takes 16.4 us, 4.1 TB/s, and 4.7 for the join: the start of a run (length, table, first loads, one after
// the other) is as long as its work.
constexpr int kFewRows = 32, kFewKeys = 32;

template <int D, typename E>
__global__ __launch_bounds__(256, 1) void gated_delta_paged_attn_few_kernel(FlashParams p) {
  using X8 = typename Pack<E>::x8;
  constexpr int DS = D / 16, DT = D / 32, CPR = D / 8, RPL = 512 / D, LPB = kFewKeys / RPL, TILE = kFewKeys * D, CH = D / 4;
  __shared__ __align__(16) E K0[4 * TILE];
  __shared__ __align__(16) E K1[4 * TILE];
  __shared__ __align__(16) E V0[4 * TILE];
  __shared__ __align__(16) E V1[4 * TILE];
  __shared__ float ml[4][2][kFewRows];
  __shared__ uint32_t redo_rows;  // rows whose sums are not finite
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), hh = lane >> 5, li = lane & 31;
  const int rep = p.HQ / p.HKV;
  PagedPlan f;
  const int64_t jobs = p.tiles * p.HKV, job = blockIdx.x % jobs;
  const int split = (int)(blockIdx.x / jobs);
  if (!paged_plan<kFewRows, kFewKeys>(p, job / p.HKV, (int)(job % p.HKV), f) || split >= f.used) return;
  const int n0 = split * f.per, n1 = imin(n0 + f.per, f.bl.count);
  const int* const table = f.sq.num >= 0 ? p.table + f.sq.num * p.table_stride : nullptr;
  const int row = f.row0 + imin(li, f.rows - 1);  // the lane's query: token row / rep, head row % rep of the group
  const RowView view = row_view(p, f, row);
  auto q_at = [&](int r) {
    return static_cast<const E*>(p.q) + f.sq.row * p.qsb + (f.sq.start + r / rep) * p.qst + (f.hkv * rep + r % rep) * p.qsh;
  };
  X8 qf[DS];
  {
    const E* q = q_at(row);
#pragma unroll
    for (int s = 0; s < DS; ++s) qf[s] = *reinterpret_cast<const X8*>(q + 16 * s + 8 * hh);
  }
  const char* const kbase = reinterpret_cast<const char*>(static_cast<const E*>(p.k) + f.hkv * p.ksh);
  const char* const vbase = reinterpret_cast<const char*>(static_cast<const E*>(p.v) + f.hkv * p.vsh);
  const int kst = (int)p.kst * 2, vst = (int)p.vst * 2, in_page = (1 << p.shift) - 1;
  int pid[2];
  auto look_up = [&](int n) {
    const int jb = f.bl.at(n);
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int key = jb * kFewKeys + 16 * g;
      const int id = key < f.klen ? page_at(table, key >> p.shift) : -1;
      pid[g] = id >= 0 && id < p.pages ? id : -1;
    }
  };
  auto fetch = [&](int n, E* kd, E* vd) {
    const int jb = f.bl.at(n);
    __amdgpu_buffer_rsrc_t rk[2], rv[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int key = jb * kFewKeys + 16 * g, left = imin(16, f.klen - key), in = key & in_page;
      const bool any = pid[g] >= 0 && left > 0;
      const int64_t page = any ? pid[g] : 0;
      rk[g] = make_rsrc(kbase + page * p.ksb * 2 + (int64_t)in * kst, any ? (uint32_t)((left - 1) * kst + 2 * D) : 0u);
      rv[g] = make_rsrc(vbase + page * p.vsb * 2 + (int64_t)in * vst, any ? (uint32_t)((left - 1) * vst + 2 * D) : 0u);
    }
#pragma unroll
    for (int u = 0; u < LPB; ++u) {
      const int r = RPL * u + lane / CPR, ch = (lane % CPR) ^ swz<D>(r);
      load_lds16(rk[RPL * u / 16], kd + u * 512, (uint32_t)((r & 15) * kst + ch * 16));
      load_lds16(rv[RPL * u / 16], vd + u * 512, (uint32_t)((r & 15) * vst + ch * 16));
    }
  };
  auto ok_bits = [&]() { return (pid[0] >= 0 ? 1 : 0) | (pid[1] >= 0 ? 2 : 0); };
  TileReads<D> rd;
  rd.init(lane);
  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
  float m = -INFINITY, l = 0.f;
  const float c = p.scale_log2, slack = fminf(8.f / c, 3e38f);
  int ok = 3, ok_next = 3;
  auto step = [&](int n, const E* kc, E* vc, E* kn, E* vn) {
    const int k0 = f.bl.at(n) * kFewKeys, k1 = k0 + kFewKeys - 1;
    if (n + 4 < n1) {
      ok_next = ok_bits();
      fetch(n + 4, kn, vn);
      if (n + 8 < n1) look_up(n + 8);
      if (LPB == 8) __builtin_amdgcn_s_waitcnt(0x4F70);  // vmcnt(16): all but the loads just issued have landed
      else __builtin_amdgcn_s_waitcnt(0x0F78);           // vmcnt(8)
    } else {
      wait_loads();
    }
    asm volatile("" ::: "memory");
    const bool partial = k1 >= f.klen || ok != 3;
    if (partial) {  // rows behind the end or on no page: zeros among the values
#pragma unroll
      for (int u = 0; u < LPB; ++u) {
        const int r = RPL * u + lane / CPR;
        if (k0 + r >= f.klen || !(ok >> (r >> 4) & 1)) *reinterpret_cast<X8*>(vc + u * 512 + lane * 8) = X8{};
      }
    }
    f32x16 s[1] = {f32x16{}};
#pragma unroll
    for (int st = 0; st < DS; ++st) s[0] = mma32(row_frag(kc, rd, st), qf[st], s[0]);
    if (partial || (p.tree && k1 >= f.base) || !all_see(f.first, f.last, k0, k1, p.window, p.sinks)) {
      uint32_t seen = (uint32_t)(view.block(k0, p.window, p.sinks) & bits_below(f.klen - k0));
      seen &= (ok & 1 ? 0xffffu : 0u) | (ok & 2 ? 0xffff0000u : 0u);
      seen >>= 4 * hh;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[0][e] = seen >> (8 * (e >> 2) + (e & 3)) & 1 ? s[0][e] : -INFINITY;
    }
    softmax_step<1, D, E>(s, acc, m, l, c, slack, vc, rd);
    ok = ok_next;
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): this block's reads are done before its buffer is loaded again
    asm volatile("" ::: "memory");
  };
  E *const k0p = K0 + w * TILE, *const k1p = K1 + w * TILE, *const v0p = V0 + w * TILE, *const v1p = V1 + w * TILE;
  if (n0 + w < n1) {
    look_up(n0 + w);
    ok = ok_bits();
    fetch(n0 + w, k0p, v0p);
    if (n0 + w + 4 < n1) look_up(n0 + w + 4);
    for (int n = n0 + w; n < n1; n += 8) {
      step(n, k0p, v0p, k1p, v1p);
      if (n + 4 < n1) step(n + 4, k1p, v1p, k0p, v0p);
    }
  }

  // The four waves' sums at one maximum. A row's 16-byte piece i lies at i ^ (row & 31) of its D floats.
  l += __shfl_xor(l, 32, kWave);
  if (hh == 0) {
    ml[w][0][li] = m;
    ml[w][1][li] = l;
  }
  if (t == 0) redo_rows = 0;
  __syncthreads();  // every wave is done with its tiles, which take the sums
  const float top = fmaxf(fmaxf(ml[0][0][li], ml[1][0][li]), fmaxf(ml[2][0][li], ml[3][0][li]));
  const float mine = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - top) * c);
  float* const red = reinterpret_cast<float*>(w < 2 ? K0 : K1) + (w & 1) * kFewRows * D;
  auto put = [&](float by) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int piece = (8 * d + 2 * j + hh) ^ (li & (CH - 1));
        *reinterpret_cast<f32x4*>(red + li * D + 4 * piece) =
            f32x4{acc[d][4 * j] * by, acc[d][4 * j + 1] * by, acc[d][4 * j + 2] * by, acc[d][4 * j + 3] * by};
      }
  };
  auto take = [&](int r, int piece) {
    f32x4 x{};
#pragma unroll
    for (int v = 0; v < 4; ++v)
      x += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(v < 2 ? K0 : K1) + (v & 1) * kFewRows * D + r * D +
                                           4 * (piece ^ (r & (CH - 1))));
    return x;
  };
  put(mine);
  __syncthreads();
  const int64_t place = f.job * p.splits + split;
  float* const po = p.part + place * kFewRows * D;
  float* const pml = p.part + p.tiles * p.HKV * p.splits * kFewRows * D + place * 2 * kFewRows;
  auto out_row = [&](int r) {
    return static_cast<E*>(p.o) + (((f.sq.row * p.seqs.T + f.sq.start + r / rep) * p.HQ) + f.hkv * rep + r % rep) * D;
  };
  auto sum_of = [&](int r) {  // of the row's weights, at the four waves' maximum
    const float tm = fmaxf(fmaxf(ml[0][0][r], ml[1][0][r]), fmaxf(ml[2][0][r], ml[3][0][r]));
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float mv = ml[v][0][r];
      sum += mv == -INFINITY ? ml[v][1][r] : ml[v][1][r] * __builtin_amdgcn_exp2f((mv - tm) * c);  // of the former 0, or NaN
    }
    return sum;
  };
  auto write = [&](int r, int piece, f32x4 x) {
    if (f.used == 1) {
      typename Pack<E>::x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (E)x[e];
      *reinterpret_cast<typename Pack<E>::x4*>(out_row(f.row0 + r) + 4 * piece) = y;
    } else {
      *reinterpret_cast<f32x4*>(po + r * D + 4 * piece) = x;
    }
  };
  for (int i = t; i < f.rows * CH; i += 256) {
    const int r = i / CH, piece = i % CH;
    float sum = sum_of(r);
    const f32x4 x = take(r, piece);
    if (f.used == 1 && sum == 0.f && sees_any<kFewKeys>(p, f, row_view(p, f, f.row0 + r))) sum = NAN;
    if (sum == sum && !(finite_f(x[0]) && finite_f(x[1]) && finite_f(x[2]) && finite_f(x[3]))) atomicOr(&redo_rows, 1u << r);
    write(r, piece, x * (sum == 0.f ? 0.f : 1.f / sum));
    if (f.used > 1 && piece == 0) {
      pml[r] = fmaxf(fmaxf(ml[0][0][r], ml[1][0][r]), fmaxf(ml[2][0][r], ml[3][0][r]));
      pml[kFewRows + r] = sum;
    }
  }
  wait_loads();  // what was written above is there before rows are written again
  __syncthreads();
  const uint32_t redo = __builtin_amdgcn_readfirstlane(redo_rows);
  if (!redo) return;
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
  const float all = sum_of(li), by = all == 0.f ? 0.f : exp2f(raise<E>) / all;
  for (int n = n0 + w; n < n1; n += 4) {
    const int k0 = f.bl.at(n) * kFewKeys;
    auto row_of = [&](const char* base, int64_t page_bytes, int64_t row_bytes, int j) {
      if (k0 + j >= f.klen) return static_cast<const E*>(nullptr);
      const int id = table[(k0 + j) >> p.shift];
      return id < 0 || id >= p.pages ? static_cast<const E*>(nullptr)
                                     : reinterpret_cast<const E*>(base + id * page_bytes + ((k0 + j) & in_page) * row_bytes);
    };
    look_up(n);
    const uint64_t there = (pid[0] >= 0 ? 0xffffu : 0u) | (pid[1] >= 0 ? 0xffff0000u : 0u);
    again_block<1, D, E>(acc, qf, view.block(k0, p.window, p.sinks) & bits_below(f.klen - k0) & there,
                         [&](int j) { return row_of(kbase, p.ksb * 2, kst, j); }, [&](int j) { return row_of(vbase, p.vsb * 2, vst, j); },
                         V0 + w * TILE, c, top == -INFINITY ? 0.f : Pack<E>::lift - top * c, by, rd);
  }
  put(exp2f(-raise<E>));
  __syncthreads();
  for (int i = t; i < f.rows * CH; i += 256)
    if (redo >> i / CH & 1) write(i / CH, i % CH, take(i / CH, i % CH));
}

// A run's result (maximum, sum, O divided by the sum) joins what others left: O as an average by the sums at the larger maximum,
// so that no more than fp32 holds is ever added up.
__device__ __forceinline__ void join_run(float& top, float& sum, f32x4& x, float m, float l, f32x4 y, float c) {
  const float now = fmaxf(top, m), a = sum * (now == top ? 1.f : __builtin_amdgcn_exp2f((top - now) * c));
  const float b = l * (m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - now) * c));
  sum = a + b;
  const float by = sum == 0.f ? 0.f : __builtin_amdgcn_rcpf(sum);  // off by 2^-23; divisions cost one token over 32,768 keys 0.3 us
  x = x * (a * by) + y * (b * by);
  top = now;
}

// The runs' results of each row joined: D / 4 threads a row, each in `groups` groups that take every groups-th run, so that many
// runs' loads are under way at once. In a fixed order.
template <int D, typename E, int ROWS, int BK>
__global__ __launch_bounds__(256) void gated_delta_paged_attn_merge_kernel(FlashParams p, int groups, int passes) {
  constexpr int CH = D / 4;
  __shared__ __align__(16) float xs[256 * 4];
  __shared__ float ms[256], ls[256];
  PagedPlan f;
  const int64_t job = blockIdx.x / passes;
  if (!paged_plan<ROWS, BK>(p, job / p.HKV, (int)(job % p.HKV), f) || f.used == 1) return;
  const int t = threadIdx.x, piece = t % CH, g = t / CH % groups, rep = p.HQ / p.HKV;
  const int r = (int)(blockIdx.x % passes) * (256 / CH / groups) + t / CH / groups;
  const float* const po = p.part + f.job * p.splits * ROWS * D;
  const float* const pml = p.part + p.tiles * p.HKV * p.splits * ROWS * D + f.job * p.splits * 2 * ROWS;
  float top = -INFINITY, sum = 0.f;
  f32x4 x{};
  if (r < f.rows) {
#pragma unroll 4
    for (int s = g; s < f.used; s += groups) {
      const float m = pml[s * 2 * ROWS + r], l = pml[(s * 2 + 1) * ROWS + r];
      const f32x4 y = *reinterpret_cast<const f32x4*>(po + (int64_t)(s * ROWS + r) * D + 4 * piece);
      join_run(top, sum, x, m, l, y, p.scale_log2);
    }
  }
  ms[t] = top;
  ls[t] = sum;
  *reinterpret_cast<f32x4*>(xs + 4 * t) = x;
  __syncthreads();
  if (g || r >= f.rows) return;
  for (int i = 1; i < groups; ++i) {
    const int o = t + i * CH;
    join_run(top, sum, x, ms[o], ls[o], *reinterpret_cast<const f32x4*>(xs + 4 * o), p.scale_log2);
  }
  const int row = f.row0 + r;
  const bool lost = sum == 0.f && sees_any<BK>(p, f, row_view(p, f, row));
  typename Pack<E>::x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (E)(lost ? NAN : x[e]);
  *reinterpret_cast<typename Pack<E>::x4*>(static_cast<E*>(p.o) + (((f.sq.row * p.seqs.T + f.sq.start + row / rep) * p.HQ) +
                                                                   f.hkv * rep + row % rep) * D + 4 * piece) = y;
}

// ------------------------------------------------------------------------------------------------ host
static int log2_of(int64_t x) {
  int s = 0;
  while (((int64_t)1 << s) < x) ++s;
  return s;
}

static int paged_check(const char* name, int64_t B, int64_t T, int64_t HQ, int64_t HKV, int64_t D, int64_t N, const void* cu,
                       int64_t pages, int64_t page_size, int64_t width, int dtype) {
  if (B <= 0 || T < 0 || HQ < 0 || HKV <= 0 || N <= 0 || (cu ? B != 1 : N != B) || pages <= 0 || width <= 0 || page_size <= 0) {
    gdn_internal_set_error("%s: bad sizes B=%lld T=%lld HQ=%lld HKV=%lld N=%lld pages=%lld page_size=%lld table width=%lld "
                           "(cu_seqlens requires B == 1)", name, (long long)B, (long long)T, (long long)HQ, (long long)HKV,
                           (long long)N, (long long)pages, (long long)page_size, (long long)width);
    return GDN_ERR_INVALID;
  }
  if (D != 64 && D != 128) {
    gdn_internal_set_error("%s: head dim %lld unsupported (64 or 128)", name, (long long)D);
    return GDN_ERR_UNSUPPORTED;
  }
  if (dtype != GDN_DTYPE_BF16 && dtype != GDN_DTYPE_F16) {
    gdn_internal_set_error("%s: dtype %d unsupported (bf16 or fp16)", name, dtype);
    return GDN_ERR_UNSUPPORTED;
  }
  if (page_size < 16 || page_size > 65536 || (page_size & (page_size - 1))) {
    gdn_internal_set_error("%s: page size %lld unsupported (a power of two from 16 to 65536)", name, (long long)page_size);
    return GDN_ERR_UNSUPPORTED;
  }
  if (T >= kFar / 2 || width >= kFar || width * page_size >= kFar / 2 || N >= kFar || pages > 0x7fffffff || HQ > 65536 ||
      HKV > 65536 || B * T > (1LL << 40)) {
    gdn_internal_set_error("%s: too many tokens, pages or heads (B=%lld T=%lld N=%lld pages=%lld table width=%lld HQ=%lld HKV=%lld)",
                           name, (long long)B, (long long)T, (long long)N, (long long)pages, (long long)width, (long long)HQ,
                           (long long)HKV);
    return GDN_ERR_UNSUPPORTED;
  }
  return GDN_OK;
}

// every stride of rows a multiple of 8 elements and none negative, every pointer on 16 bytes
static bool rows_ok(const int64_t* st, int n, uintptr_t all) {
  for (int i = 0; i < n; ++i)
    if (st[i] < 0 || st[i] % 8) return false;
  return !(all & 15);
}

// How a call is cut: tiles of `rows` rows, blocks of `keys` keys, `splits` runs of them a tile. bf16, 16 / 4 heads of 128, us:
//   rows a sequence (new tokens times heads of a group): tiles of 32 with a run of keys a wave, or of 128 that share what they
//   load. Up to 64 rows the former; up to 256 while the tiles make no more than 4,400 blocks of keys in all:
//     tokens, cached   1 sequence      2               4
//       61,  1,000     14.7, 18.9      16.1, 20.2      18.9, 22.0
//       61,  4,000     20.5, 23.9      25.7, 27.0      36.5, 31.2
//       64, 16,000     37.6, 34.9      58.9, 42.1       102, 60.9
//     Two sequences of 61 tokens over 4,000 keys (8,100 blocks) are 5% slower in tiles of 128, which they take; four (16,200) faster.
//     With bounds the mean number of new tokens counts: 512 of one sequence beside single ones of 63 others over 4,000 keys take
//     157 us in tiles of 32; each part alone 50 and 103.
//   runs: as many as make about kFewGroups or kManyGroups workgroups (256 and 512: one token over 32,768 keys 20.8 and 26.2,
//   1,024 workgroups 36.9; 8 trees of 61 tokens 48.3 and 41.0, 59.5), of 4 blocks at least (one token over 1,024 keys with 4, 8
//   and 16: 10.6, 11.6, 14.1). Up to 256 keys one run without a merge (8.1, with two runs 9.8). The lengths are on the device and
//   have no part in this: one sequence of 32,768 in a batch of 64 with 256 tokens else is read by 4 workgroups, 415 us (by itself 26).
struct PagedCut {
  int rows, keys, splits;
  int64_t tiles;
};
constexpr int64_t kFewMost = 64, kFewMostShort = 256, kFewBlocks = 4400, kFewGroups = 256, kManyGroups = 512;
static PagedCut paged_cut(int64_t B, int64_t T, int64_t HQ, int64_t HKV, int64_t N, bool varlen, int64_t page_size, int64_t width,
                          int64_t window, int64_t sinks) {
  const int64_t rep = HQ / HKV, tokens = varlen ? (T + N - 1) / N : T;
  auto tiles_of = [&](int rows) { return varlen ? packed_tiles(T, N, (int)rep, rows) : B * ((T * rep + rows - 1) / rows); };
  auto blocks_seen = [&](int rows, int keys) {  // by a tile, at most
    int64_t most = width * page_size;
    if (window > 0 && window < most) {
      const int64_t some = window + rows / rep + 1 + (sinks < most ? sinks : most);
      if (some < most) most = some;
    }
    return (most + keys - 1) / keys + 1;
  };
  const bool few = tokens * rep <= kFewMost ||
                   (tokens * rep <= kFewMostShort && tiles_of(kFewRows) * HKV * blocks_seen(kFewRows, kFewKeys) <= kFewBlocks);
  PagedCut c{few ? kFewRows : kBQ, few ? kFewKeys : kBK, 1, 0};
  c.tiles = tiles_of(c.rows);
  const int64_t busy = (varlen ? (T * rep + c.rows - 1) / c.rows + N : c.tiles) * HKV;  // about as many do anything
  const int64_t blocks = blocks_seen(c.rows, c.keys), most = blocks * c.keys <= 256 + c.keys ? 1 : (blocks + 3) / 4;
  const int64_t splits = ((few ? kFewGroups : kManyGroups) + busy - 1) / busy;
  c.splits = (int)(splits > most ? most : splits);
  return c;
}

}  // namespace gdn

using namespace gdn;

extern "C" int gdn_paged_append(const void* q, int64_t q_batch_stride, int64_t q_token_stride, int64_t q_head_stride,
                                const void* k, int64_t k_batch_stride, int64_t k_token_stride, int64_t k_head_stride,
                                const void* v, int64_t v_batch_stride, int64_t v_token_stride, int64_t v_head_stride,
                                const float* q_weight, const float* k_weight, void* q_out, void* k_cache, int64_t kc_page_stride,
                                int64_t kc_head_stride, int64_t kc_token_stride, void* v_cache, int64_t vc_page_stride,
                                int64_t vc_head_stride, int64_t vc_token_stride, const int32_t* page_table,
                                int64_t table_stride, const void* lengths, int lengths_i32, const void* positions,
                                int64_t pos_batch_stride, int64_t pos_token_stride, int pos_i32, const void* cu_seqlens,
                                int64_t B, int64_t T, int64_t HQ, int64_t HKV, int64_t D, int64_t N, int64_t pages,
                                int64_t page_size, int64_t width, int dtype, int rot_dim, double theta, float eps,
                                unsigned flags, void* stream) {
  const char* name = "gdn_paged_append";
  if (int rc = paged_check(name, B, T, q ? HQ : 0, HKV, D, N, cu_seqlens, pages, page_size, width, dtype)) return rc;
  if (rot_dim < 0 || rot_dim > D || rot_dim % 16) {
    gdn_internal_set_error("%s: rot_dim=%d unsupported (a multiple of 16 up to D)", name, rot_dim);
    return GDN_ERR_UNSUPPORTED;
  }
  if (!(theta > 0.) || !(theta < 1e300) || !(eps >= 0.f) || (q && HQ <= 0)) {
    gdn_internal_set_error("%s: bad arguments HQ=%lld theta=%g eps=%g", name, (long long)HQ, theta, (double)eps);
    return GDN_ERR_INVALID;
  }
  if (T == 0) return GDN_OK;
  const int64_t st[15] = {k_batch_stride, k_token_stride, k_head_stride, v_batch_stride, v_token_stride, v_head_stride,
                          kc_page_stride, kc_head_stride, kc_token_stride, vc_page_stride, vc_head_stride, vc_token_stride,
                          q ? q_batch_stride : 0, q ? q_token_stride : 0, q ? q_head_stride : 0};
  if (!k || !v || !k_cache || !v_cache || !page_table || !lengths || (q && !q_out) ||
      !rows_ok(st, 15, reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                           reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
                           (q ? reinterpret_cast<uintptr_t>(q_out) : 0))) {
    gdn_internal_set_error("%s: null tensor pointer, or rows not 16-byte aligned", name);
    return GDN_ERR_INVALID;
  }
  AppendParams p{{q, k, v}, {q_batch_stride, k_batch_stride, v_batch_stride}, {q_token_stride, k_token_stride, v_token_stride},
                 {q_head_stride, k_head_stride, v_head_stride}, {q_weight, k_weight}, q_out, {k_cache, v_cache},
                 {kc_page_stride, vc_page_stride}, {kc_head_stride, vc_head_stride}, {kc_token_stride, vc_token_stride},
                 page_table, table_stride, lengths, positions, pos_batch_stride, pos_token_stride, cu_seqlens,
                 lengths_i32, pos_i32, (flags & GDN_FLAG_CU_INT32) ? 1 : 0, (int)width, log2_of(page_size), (int)pages,
                 T, N, B * T, q ? (int)HQ : 0, (int)HKV, rot_dim, B * T <= kAppendShared ? 4 : 1, eps};
  for (int f = 0; f < rot_dim / 2; ++f) p.turns[f] = pow(theta, -2. * f / rot_dim) / 6.283185307179586;
  const int64_t want = p.wpt == 4 ? p.tokens : (p.tokens + 3) / 4;
  const dim3 grid((unsigned)(want < kMaxGroups256 ? want : kMaxGroups256)), block(256);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == GDN_DTYPE_BF16) {
    if (D == 128) hipLaunchKernelGGL((gated_delta_paged_append_kernel<128, bf16>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((gated_delta_paged_append_kernel<64, bf16>), grid, block, 0, s, p);
  } else {
    if (D == 128) hipLaunchKernelGGL((gated_delta_paged_append_kernel<128, f16>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((gated_delta_paged_append_kernel<64, f16>), grid, block, 0, s, p);
  }
  return gdn_internal_check_launch("gated_delta_paged_append_kernel");
}

extern "C" size_t gdn_paged_attn_workspace_size(int64_t B, int64_t T, int64_t HQ, int64_t HKV, int64_t D, int64_t N,
                                                int64_t page_size, int64_t width, int64_t window, int64_t sinks, int varlen) {
  if (B <= 0 || T <= 0 || HQ <= 0 || HKV <= 0 || HQ % HKV || D <= 0 || N <= 0 || page_size <= 0 || width <= 0) return 0;
  const PagedCut c = paged_cut(B, T, HQ, HKV, N, varlen != 0, page_size, width, window, sinks);
  return c.splits == 1 ? 0 : (size_t)c.tiles * HKV * c.splits * c.rows * (D + 2) * 4;
}

extern "C" int gdn_paged_attn_fwd(const void* q, int64_t q_batch_stride, int64_t q_token_stride, int64_t q_head_stride,
                                  const void* k_cache, int64_t kc_page_stride, int64_t kc_head_stride, int64_t kc_token_stride,
                                  const void* v_cache, int64_t vc_page_stride, int64_t vc_head_stride, int64_t vc_token_stride,
                                  const int32_t* page_table, int64_t table_stride, const void* lengths, int lengths_i32,
                                  const int64_t* tree, int64_t tree_batch_stride, int64_t tree_token_stride, void* o,
                                  const void* cu_seqlens, int64_t B, int64_t T, int64_t HQ, int64_t HKV, int64_t D, int64_t N,
                                  int64_t pages, int64_t page_size, int64_t width, int dtype, int64_t window, int64_t sinks,
                                  float scale, unsigned flags, void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "gdn_paged_attn_fwd";
  if (int rc = paged_check(name, B, T, HQ, HKV, D, N, cu_seqlens, pages, page_size, width, dtype)) return rc;
  if (HQ <= 0 || HQ % HKV || window < 0 || sinks < 0) {
    gdn_internal_set_error("%s: bad arguments HQ=%lld HKV=%lld window=%lld sinks=%lld (HQ a multiple of HKV)", name,
                           (long long)HQ, (long long)HKV, (long long)window, (long long)sinks);
    return GDN_ERR_INVALID;
  }
  if (T * (HQ / HKV) >= kFar) {  // row numbers inside a sequence are 32 bits, tiles from here on are none
    gdn_internal_set_error("%s: too many rows (T=%lld times HQ / HKV=%lld)", name, (long long)T, (long long)(HQ / HKV));
    return GDN_ERR_UNSUPPORTED;
  }
  if (!(scale > 0.f) || scale > 2.0e38f) {
    gdn_internal_set_error("%s: scale %g unsupported (a positive finite softmax scale)", name, (double)scale);
    return GDN_ERR_INVALID;
  }
  if (T == 0) return GDN_OK;
  const int64_t st[9] = {q_batch_stride, q_token_stride, q_head_stride, kc_page_stride, kc_head_stride, kc_token_stride,
                         vc_page_stride, vc_head_stride, vc_token_stride};
  if (!q || !k_cache || !v_cache || !page_table || !lengths || !o ||
      !rows_ok(st, 9, reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) |
                          reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(o)) ||
      kc_token_stride * 2 > kMaxRowBytes || vc_token_stride * 2 > kMaxRowBytes) {
    gdn_internal_set_error("%s: null tensor pointer, rows not 16-byte aligned, or cache rows more than %lld bytes apart", name,
                           (long long)kMaxRowBytes);
    return GDN_ERR_INVALID;
  }
  FlashParams p{};
  p.q = q, p.k = k_cache, p.v = v_cache, p.o = o;
  p.qsb = q_batch_stride, p.qst = q_token_stride, p.qsh = q_head_stride;
  p.ksb = kc_page_stride, p.ksh = kc_head_stride, p.kst = kc_token_stride;
  p.vsb = vc_page_stride, p.vsh = vc_head_stride, p.vst = vc_token_stride;
  p.seqs = Packed{cu_seqlens, (flags & GDN_FLAG_CU_INT32) ? 1 : 0, N, T};
  p.B = B;
  p.HQ = (int)HQ, p.HKV = (int)HKV, p.parts = job_parts(HKV);
  p.window = window <= 0 || window > kFar ? kFar : (int)window;
  p.sinks = window <= 0 ? 0 : sinks > kFar ? kFar : (int)sinks;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.table = page_table, p.table_stride = table_stride, p.lengths = lengths, p.len_i32 = lengths_i32;
  p.width = (int)width, p.shift = log2_of(page_size), p.pages = (int)pages;
  p.tree = tree, p.tb = tree_batch_stride, p.tt = tree_token_stride;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 block(256);
  auto by_type = [&](auto go) {
    if (dtype == GDN_DTYPE_BF16) D == 128 ? go(bf16{}, std::integral_constant<int, 128>{}) : go(bf16{}, std::integral_constant<int, 64>{});
    else D == 128 ? go(f16{}, std::integral_constant<int, 128>{}) : go(f16{}, std::integral_constant<int, 64>{});
  };
  const PagedCut cut = paged_cut(B, T, HQ, HKV, N, cu_seqlens != nullptr, page_size, width, window, sinks);
  p.tiles = cut.tiles, p.splits = cut.splits, p.part = static_cast<float*>(workspace);
  const size_t need = gdn_paged_attn_workspace_size(B, T, HQ, HKV, D, N, page_size, width, window, sinks, cu_seqlens != nullptr);
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))) {
    gdn_internal_set_error("%s: workspace of %zu bytes needed, 16-byte aligned", name, need);
    return GDN_ERR_INVALID;
  }
  const bool few = cut.rows == kFewRows;
  const int64_t jobs = cut.tiles * HKV, groups = (few ? jobs : job_groups(HKV, 1, cut.tiles)) * cut.splits;
  // the merge: a row's threads in up to 8 groups, two runs for each at least, while that makes no more than 2,048 workgroups
  const int64_t tile_rows = cu_seqlens || T * (HQ / HKV) > cut.rows ? cut.rows : T * (HQ / HKV);
  int merge_groups = 1;
  while (merge_groups < 8 && merge_groups * 4 <= cut.splits && jobs * tile_rows * (D / 4) * merge_groups * 2 <= 2048 * 256) merge_groups *= 2;
  const int merge_rows = (int)(256 / (D / 4) / merge_groups);
  const int merge_passes = (int)((tile_rows + merge_rows - 1) / merge_rows);
  if (groups > kMaxGroups256 || (cut.splits > 1 && jobs * merge_passes > kMaxGroups256)) {
    gdn_internal_set_error("%s: grid too large", name);
    return GDN_ERR_UNSUPPORTED;
  }
  by_type([&](auto e, auto d) {
    constexpr int kD = decltype(d)::value;
    using E = decltype(e);
    if (few) hipLaunchKernelGGL((gated_delta_paged_attn_few_kernel<kD, E>), dim3((unsigned)groups), block, 0, s, p);
    else hipLaunchKernelGGL((gated_delta_paged_attn_kernel<kD, E>), dim3((unsigned)groups), block, 0, s, p);
  });
  if (int rc = gdn_internal_check_launch("gated_delta_paged_attn_kernel")) return rc;
  if (cut.splits == 1) return GDN_OK;
  by_type([&](auto e, auto d) {
    constexpr int kD = decltype(d)::value;
    using E = decltype(e);
    const dim3 grid((unsigned)(jobs * merge_passes));
    if (few) hipLaunchKernelGGL((gated_delta_paged_attn_merge_kernel<kD, E, kFewRows, kFewKeys>), grid, block, 0, s, p, merge_groups, merge_passes);
    else hipLaunchKernelGGL((gated_delta_paged_attn_merge_kernel<kD, E, kBQ, kBK>), grid, block, 0, s, p, merge_groups, merge_passes);
  });
  return gdn_internal_check_launch("gated_delta_paged_attn_merge_kernel");
}
