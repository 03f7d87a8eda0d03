// Attention with a sliding window and a few first tokens that stay visible (sinks), over whole sequences, and its backward.
//
//   p_ij = softmax_j(scale q_i . k_j) over the keys that i sees;  o_i = sum_j p_ij v_j
//   delta_i = do_i . o_i;  ds_ij = p_ij (do_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j;  dk_j = scale sum_i ds_ij q_i;  dv_j = sum_i p_ij do_i
//
// Bound by the matrix and the vector units in turn: of the cycles of a prompt's forward each is busy in 36%, LDS in 18%; two waves a
// SIMD overlap them only in part, and 64 queries a wave, which would halve the LDS reads, do not fit the registers. The backward
// computes S and dP again from the row's logarithm: one kernel holds 32 queries a wave and walks their keys (dq, and delta on the
// way), the other holds 32 keys and walks their queries (dk, dv, summed over the q heads of the kv head in fp32). No atomics.
//
// Measured on 2 x 4,096 tokens, 16 heads on 4 of 128, window 1,024, 4 sinks, each kernel by itself in a trace, operations of
// visible pairs only (a large bf16 product reaches 1,228 TFLOP/s): forward 100 us, 601 TFLOP/s; dq 135 us, 672; dk and dv 216 us,
// 560, and 7 for the launch behind it; sinks 7 us; the step as a whole 425-431. A prompt of 8,192 tokens 100 us by itself, 87-88
// among others of its kind. 5,003 tokens in 7 documents, 8 heads on 2 of 64, window 200: 20, 25, 31 and 5 us, join 5, sinks 4.

#include "gdn_flash.h"

namespace gdn {

template <int D, typename E>
__global__ __launch_bounds__(256, 2) void gated_delta_window_attn_fwd_kernel(FlashParams p) {
  __shared__ __align__(16) E Ks0[kBK * D];
  __shared__ __align__(16) E Ks1[kBK * D];
  __shared__ __align__(16) E Vs0[kBK * D];
  __shared__ __align__(16) E Vs1[kBK * D];
  flash_forward<D, E, false>(p, Ks0, Ks1, Vs0, Vs1);
}

struct WindowBwdParams {
  const bf16 *q, *k, *v, *o, *d_o;  // o, d_o [B, T, HQ, D]
  int64_t qsb, qst, qsh, ksb, kst, ksh, vsb, vst, vsh;
  const bf16* o_rest;               // [B, T, HQ, D]
  const float* lse;                 // [HQ, B T]
  float* delta;                     // [HQ, B T]
  bf16 *dq, *dk, *dv;               // contiguous
  Packed seqs;
  int64_t B, q_tiles, k_tiles;
  int HQ, HKV, parts, window, sinks;
  float scale, scale_log2;
  // far queries of the sinks: slots for pieces of them and, behind those, for the near ones, per kv head and tile of 128 sinks:
  // [far_jobs + near slots][HKV][2][sink rows][D]
  float* part;
  FarList far;
  int64_t far_jobs;
  int sink_rows;
  // few key tiles: the near queries of one are dealt out to `shares` workgroups, whose sums meet in another kernel:
  // [shares][B T][HKV][2][D]
  float* near;
  int shares;
};

// Loads of 64 rows of `stride` bytes from `base` (the block's first row) into a tile, `rows` of them there.
template <int D>
struct BlockLoad {
  int w, lane;
  static constexpr int CPR = D / 8, RPL = 512 / D, LPT = kBK / (4 * RPL);
  __device__ __forceinline__ void load(const char* base, int stride, int rows, bf16* to) const {
    const auto r = make_rsrc(base, rows <= 0 ? 0u : (uint32_t)((rows - 1) * stride + 2 * D));
    const int drow = w * RPL + lane / CPR;
    const uint32_t off = (uint32_t)(drow * stride + ((lane % CPR) ^ swz<D>(drow)) * 16);
#pragma unroll
    for (int u = 0; u < LPT; ++u) load_lds16(r, to + (w + 4 * u) * 512, off + u * 4 * RPL * stride);
  }
  // the rows of the wave's own loads from `rows` on: zeros
  __device__ __forceinline__ void clean(int rows, bf16* to) const {
#pragma unroll
    for (int u = 0; u < LPT; ++u)
      if ((w + 4 * u) * RPL + lane / CPR >= rows) *reinterpret_cast<bf16x8*>(to + (w + 4 * u) * 512 + lane * 8) = bf16x8{};
  }
};

template <int D>
__device__ __forceinline__ float dot8(bf16x8 a, bf16x8 b) {
  float x = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) x += (float)a[e] * (float)b[e];
  return x;
}

// dq and delta: 128 queries of one head a workgroup, as the forward's. delta takes o with what its rounding left (kept by a forward
// that a backward follows): where few keys are seen dp - delta is small against o, and o's half step would come out larger in
// dq and dk than the roundings of ds and of the results together.
template <int D>
__global__ __launch_bounds__(256, 2) void gated_delta_window_attn_dq_kernel(WindowBwdParams p) {
  constexpr int DS = D / 16, DT = D / 32;
  __shared__ __align__(16) bf16 Ks0[kBK * D];
  __shared__ __align__(16) bf16 Ks1[kBK * D];
  __shared__ __align__(16) bf16 Vs0[kBK * D];
  __shared__ __align__(16) bf16 Vs1[kBK * D];
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), hh = lane >> 5, li = lane & 31;
  const int rep = p.HQ / p.HKV;
  Job job;
  if (!job_of(blockIdx.x, p.HKV, rep, p.parts, p.q_tiles, job)) return;
  Seq sq;
  if (p.seqs.cu) {
    sq = packed_tile(p.seqs, job.tile, 1, kBQ);
  } else {
    const int64_t per = (p.seqs.T + kBQ - 1) / kBQ;
    sq = Seq{job.tile % p.B, 0, (int)p.seqs.T, 0, (int)(per - 1 - job.tile / p.B)};
  }
  const int q0 = sq.tile * kBQ, hq = job.hkv * rep + job.hm;
  if (q0 >= sq.len) return;
  const int q1 = imin(q0 + kBQ, sq.len) - 1, qi = q0 + 32 * w + li, wq0 = q0 + 32 * w, wq1 = imin(wq0 + 31, q1);
  const bool wave_live = wq0 <= wq1, row_ok = wave_live && qi < sq.len;
  const RowView view{qi, kFar, 0};
  Blocks bl = blocks_of<kBK>(q0, q1, p.window, p.sinks);
  if (sq.num < 0) bl.count = 0;
  const int64_t tok = sq.row * p.seqs.T + sq.start, all = p.B * p.seqs.T;
  const int qc = imin(qi, sq.len - 1);
  const bf16* qrow = p.q + sq.row * p.qsb + (sq.start + qc) * p.qst + hq * p.qsh;
  const int64_t orow = ((tok + qc) * p.HQ + hq) * D;
  bf16x8 qf[DS], df[DS];
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < DS; ++s) {
    qf[s] = *reinterpret_cast<const bf16x8*>(qrow + 16 * s + 8 * hh);
    df[s] = *reinterpret_cast<const bf16x8*>(p.d_o + orow + 16 * s + 8 * hh);
    delta += dot8<D>(df[s], *reinterpret_cast<const bf16x8*>(p.o + orow + 16 * s + 8 * hh));
    delta += dot8<D>(df[s], *reinterpret_cast<const bf16x8*>(p.o_rest + orow + 16 * s + 8 * hh));
  }
  delta += __shfl_xor(delta, 32, kWave);
  const float lse = p.lse[hq * all + tok + qc];
  if (row_ok && hh == 0) p.delta[hq * all + tok + qi] = finite_f(lse) ? delta : NAN;  // of those no ds is finite

  const char* const kbase = reinterpret_cast<const char*>(p.k + sq.row * p.ksb + sq.start * p.kst + job.hkv * p.ksh);
  const char* const vbase = reinterpret_cast<const char*>(p.v + sq.row * p.vsb + sq.start * p.vst + job.hkv * p.vsh);
  const int kst = (int)p.kst * 2, vst = (int)p.vst * 2;
  const BlockLoad<D> io{w, lane};
  auto fetch = [&](int jb, bf16* kd, bf16* vd) {
    io.load(kbase + (int64_t)jb * kBK * kst, kst, imin(kBK, sq.len - jb * kBK), kd);
    io.load(vbase + (int64_t)jb * kBK * vst, vst, imin(kBK, sq.len - jb * kBK), vd);
  };
  TileReads<D> rd;
  rd.init(lane);
  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
  const float c = p.scale_log2;
  auto block = [&](bool masked, const bf16* kb, const bf16* vb, int k0) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      f32x16 s{}, dp{};
#pragma unroll
      for (int st = 0; st < DS; ++st) s = mma32(row_frag(kb + 32 * kt * D, rd, st), qf[st], s);
#pragma unroll
      for (int st = 0; st < DS; ++st) dp = mma32(row_frag(vb + 32 * kt * D, rd, st), df[st], dp);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], c, -lse)) * (dp[e] - delta);
      if (masked) {
        const uint32_t seen = (uint32_t)(view.block(k0 + 32 * kt, p.window, p.sinks) >> 4 * hh);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = seen >> (8 * (e >> 2) + (e & 3)) & 1 ? s[e] : 0.f;
      }
      bf16x8 pb[2];
      pack16<bf16>(s, pb);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] = mma32(tr_frag(kb + (2 * kt + h) * 16 * D, rd, d), pb[h], acc[d]);
    }
  };
  auto arrive = [&](int jb, bf16* kd) {  // the wave's loads of block jb have landed; keys behind the end: zeros
    wait_loads();
    if ((jb + 1) * kBK > sq.len) io.clean(sq.len - jb * kBK, kd);
  };
  auto step = [&](int n, const bf16* kc, const bf16* vc, bf16* kn, bf16* vn) {
    const int jb = bl.at(n), next = bl.at(n + 1);
    if (n + 1 < bl.count) fetch(next, kn, vn);
    const int k0 = jb * kBK, k1 = k0 + kBK - 1;
    if (wave_live && !none_sees(wq0, wq1, k0, k1, p.window, p.sinks))
      block(!all_see(wq0, wq1, k0, k1, p.window, p.sinks), kc, vc, k0);
    if (n + 1 < bl.count) arrive(next, kn);
    __syncthreads();
  };
  if (bl.count > 0) {
    fetch(bl.at(0), Ks0, Vs0);
    arrive(bl.at(0), Ks0);
    __syncthreads();
    for (int n = 0; n < bl.count; n += 2) {
      step(n, Ks0, Vs0, Ks1, Vs1);
      if (n + 1 < bl.count) step(n + 1, Ks1, Vs1, Ks0, Vs0);
    }
  }
  bool fine = finite_all(acc);
  fine = lse != lse || !finite_f(delta) || (__shfl_xor((int)fine, 32, kWave) && fine);  // of those no ds that is seen is finite
  auto write = [&]() {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<bf16x4*>(p.dq + orow + 32 * d + 8 * j + 4 * hh) =
            to_bf16x4(acc[d][4 * j] * p.scale, acc[d][4 * j + 1] * p.scale, acc[d][4 * j + 2] * p.scale, acc[d][4 * j + 3] * p.scale);
  };
  if (row_ok) write();
  if (!__any(row_ok && !fine)) return;
  // Rows whose sums are not finite, over the wave's blocks once more: infinities and NaN among the keys are left out of the products,
  // and the rows that see them become NaN there (the score is -inf, and 0 times them is none).
  wait_loads();  // what was written above is there before rows are written again
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
  bf16* const tile = w == 0 ? Ks0 : w == 1 ? Ks1 : w == 2 ? Vs0 : Vs1;  // all waves are behind their last block
  constexpr int CPR = D / 8, RPL = 512 / D;
  for (int n = 0; n < bl.count; ++n) {
    const int k0 = bl.at(n) * kBK;
    if (none_sees(wq0, wq1, k0, k0 + kBK - 1, p.window, p.sinks)) continue;
#pragma unroll 4
    for (int u = 0; u < kBK / RPL; ++u) {
      const int r = u * RPL + lane / CPR, ch = lane % CPR;
      *reinterpret_cast<bf16x8*>(tile + r * D + ((ch ^ swz<D>(r)) << 3)) =
          k0 + r < sq.len ? *reinterpret_cast<const bf16x8*>(kbase + (int64_t)(k0 + r) * kst + 16 * ch) : bf16x8{};
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma nounroll
    for (int kt = 0; kt < 2; ++kt) {
      f32x16 s{}, dp{}, one;
      const bf16* const v = reinterpret_cast<const bf16*>(vbase + (int64_t)imin(k0 + 32 * kt + li, sq.len - 1) * vst);
#pragma unroll
      for (int st = 0; st < DS; ++st) s = mma32(row_frag(tile + 32 * kt * D, rd, st), qf[st], s);
#pragma unroll
      for (int st = 0; st < DS; ++st) dp = mma32(ld8(v + 16 * st + 8 * hh), df[st], dp);
      const uint32_t seen = (uint32_t)(view.block(k0 + 32 * kt, p.window, p.sinks) >> 4 * hh);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const bool see = seen >> (8 * (e >> 2) + (e & 3)) & 1;
        s[e] = see ? __builtin_amdgcn_exp2f(fmaf(s[e], c, -lse)) * (dp[e] - delta) : 0.f;
        one[e] = see ? 1.f : 0.f;
      }
      bf16x8 pb[2], ones[2];
      pack16<bf16>(s, pb);
      pack16<bf16>(one, ones);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          bf16x8 x = tr_frag(tile + (2 * kt + h) * 16 * D, rd, d), up, down;
          split_infinite<bf16>(x, up, down);
          acc[d] = mma32(x, pb[h], acc[d]);
          add_infinite<bf16>(acc[d], up + down, up + down, ones[h]);
        }
    }
    __builtin_amdgcn_wave_barrier();  // the tile is read before the next block's is written
  }
  if (row_ok && !fine) write();
}

// dk and dv: 128 keys of one kv head a workgroup, 32 a wave in registers; blocks of 64 queries with their do pass through LDS,
// head after head. Two teams of four waves take every other block and add their sums at the end: two waves a SIMD also where a
// layer has no more key tiles than there are CUs (368 -> 207 us at the training size above). Where it has fewer, several
// workgroups share a tile's blocks. Sinks are seen by far queries too: the first k_tiles * shares jobs are every tile's near
// queries, the others a piece of the far queries for one tile of sinks. A tile's sums over those meet in
// gated_delta_window_attn_sinks_kernel.
//
// BAD: a launch behind the one that computes everything, which takes a tile again if masked blocks of it hold queries whose
// logarithm or delta is not finite, and ends at once if none does. There a masked weight, 0, met an infinity or NaN of do or q, and
// keys that do not see it became NaN too. (As a second path of one kernel it cost the ordinary one registers, and the training
// step 420 -> 433 to 449 us; summing such keys again row by row took 95 ms for 6,000 tokens of 16:4 heads under a NaN loss.)
template <int D, bool BAD>
__global__ __launch_bounds__(512, 2) void gated_delta_window_attn_dkv_kernel(WindowBwdParams p) {
  // of D = 128 half of each wave's V fragments lie in LDS (VL k-steps): with all of them in registers the loop reloads spilled
  // ones, and waits for the tiles under way with them
  constexpr int DS = D / 16, DT = D / 32, VL = D == 128 ? DS / 2 : 0, VR = DS - VL;
  __shared__ __align__(16) bf16 Qs0[2 * kBK * D];
  __shared__ __align__(16) bf16 Qs1[2 * kBK * D];
  __shared__ __align__(16) bf16 Ds0[2 * kBK * D];
  __shared__ __align__(16) bf16 Ds1[2 * kBK * D];
  __shared__ __align__(16) float Ls0[2][2 * kBK];  // lse, delta
  __shared__ __align__(16) float Ls1[2][2 * kBK];
  __shared__ __align__(16) bf16 Vs[VL ? 4 * VL * kWave * 8 : 8];
  __shared__ int bads[8];
  const int t = threadIdx.x, lane = t & 63, w8 = __builtin_amdgcn_readfirstlane(t >> 6), hh = lane >> 5, li = lane & 31;
  const int w = w8 & 3, team = w8 >> 2;
  const int rep = p.HQ / p.HKV;
  Job job;
  if (!job_of(blockIdx.x, p.HKV, 1, p.parts, p.k_tiles * p.shares + p.far_jobs, job)) return;
  const bool far_job = job.tile >= p.k_tiles * p.shares;
  Seq sq;
  int tile, from, to, share = 0;
  int64_t slot;  // where sums over part of a sink's queries go
  if (!far_job) {
    const int64_t kt = job.tile / p.shares;
    share = (int)(job.tile - kt * p.shares);
    if (p.seqs.cu) sq = packed_tile(p.seqs, kt, 1, kBQ);
    else sq = Seq{kt % p.B, 0, (int)p.seqs.T, (int)(kt % p.B), (int)(kt / p.B)};  // those that most see first
    tile = sq.tile;
    if (tile * kBQ >= sq.len) return;
    from = tile * kBQ;
    to = sq.num < 0 ? from : near_end(tile, p.window, sq.len);
    slot = to < sq.len && sq.num >= 0 && p.shares == 1 ? p.far_jobs + near_slot(p.far, sq, tile) : -1;
  } else {
    slot = job.tile - p.k_tiles * p.shares;
    const FarWork f = far_work(p.seqs, p.far, p.B, slot);
    sq = f.sq;
    tile = f.sink_tile;
    if (tile < 0 || tile * kBQ >= sq.len) return;
    from = imax(near_end(tile, p.window, sq.len), p.far.first_query() + sq.tile * p.far.far);
    to = imin(sq.len, p.far.first_query() + (sq.tile + 1) * p.far.far);
    if (from >= to) return;
  }
  const int wk0 = tile * kBQ + 32 * w, key = wk0 + li, kc = imin(key, sq.len - 1);
  const bool wave_live = wk0 < sq.len && !(far_job && wk0 >= p.sinks);
  const bool row_ok = key < sq.len && !(far_job && key >= p.sinks);
  const int64_t tok = sq.row * p.seqs.T + sq.start, all = p.B * p.seqs.T;
  const bf16* const krow = p.k + sq.row * p.ksb + (sq.start + kc) * p.kst + job.hkv * p.ksh;
  const bf16* const vrow = p.v + sq.row * p.vsb + (sq.start + kc) * p.vst + job.hkv * p.vsh;
  if constexpr (BAD) {
    // masked blocks are those with a near tile's first and last queries, and of far pieces all; as whole blocks, which reach past them
    const int lo = from / kBK * kBK, hi = imin((to + kBK - 1) / kBK * kBK, sq.len), most = from < to ? hi - lo : 0;
    const int some = imin(most, far_job ? most : 256), each = far_job ? some : 2 * some;
    bool bad = false;
    for (int x = t; x < rep * each; x += 512) {
      const int h = x / each, r = x - h * each, i = r < some ? lo + r : hi - 2 * some + r;
      bad |= !finite_f(p.delta[(job.hkv * rep + h) * all + tok + i]);
    }
    const bool any = __any(bad);
    if (lane == 0) bads[w8] = any;
    __syncthreads();
    int count = 0;
    for (int x = 0; x < 8; ++x) count += bads[x];
    if (!count) return;
  }
  bf16x8 kf[DS], vf[VR];
#pragma unroll
  for (int s = 0; s < DS; ++s) kf[s] = *reinterpret_cast<const bf16x8*>(krow + 16 * s + 8 * hh);
#pragma unroll
  for (int s = 0; s < VR; ++s) vf[s] = *reinterpret_cast<const bf16x8*>(vrow + 16 * s + 8 * hh);
  bf16* const vl = Vs + (w * VL * kWave + lane) * 8;
  if (!team) {  // read behind the first barrier
#pragma unroll
    for (int s = 0; s < VL; ++s) *reinterpret_cast<bf16x8*>(vl + s * kWave * 8) = *reinterpret_cast<const bf16x8*>(vrow + 16 * (VR + s) + 8 * hh);
  }
  const char* const qbase = reinterpret_cast<const char*>(p.q + sq.row * p.qsb + sq.start * p.qst + (int64_t)job.hkv * rep * p.qsh);
  const char* const dbase = reinterpret_cast<const char*>(p.d_o + (tok * p.HQ + job.hkv * rep) * D);
  const int qst = (int)p.qst * 2, dst = p.HQ * D * 2;
  const BlockLoad<D> io{w, lane};
  auto fetch = [&](int h, int blk, bf16* qd, bf16* dd, float* ld) {
    const int rows = imin(kBK, sq.len - blk * kBK);
    io.load(qbase + h * p.qsh * 2 + (int64_t)blk * kBK * qst, qst, rows, qd);
    io.load(dbase + (int64_t)h * D * 2 + (int64_t)blk * kBK * dst, dst, rows, dd);
    if (w < 2) {
      const float* src = (w ? p.delta : p.lse) + (job.hkv * rep + h) * all + tok + blk * kBK;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(make_rsrc(src, (uint32_t)(rows * 4)),
                                               (__attribute__((address_space(3))) void*)(ld + w * kBK), 4, lane * 4, 0, 0, 0);
    }
  };
  TileReads<D> reads;
  reads.init(lane);
  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) dk[d] = f32x16{}, dv[d] = f32x16{};
  const float c = p.scale_log2;
  auto block = [&](bool masked, const bf16* qb, const bf16* db, const float* lb, int q0) {
    const bf16* const vh = vl + opaque_int(0);
    // the block's queries that see the lane's key (made here: registers are short)
    uint64_t seen = ~0ull;
    if (masked) {
      const int kk = wk0 + (opaque_int(lane) & 31), hi = kk < p.sinks ? to : imin(to, kk + p.window);
      seen = (bits_below(hi - q0) & ~bits_below(imax(kk, from) - q0)) >> 4 * hh;
    }
#pragma unroll
    for (int qt = 0; qt < 2; ++qt) {
      f32x16 s{}, dp{};
      TileReads<D> rd = reads.here();
#pragma unroll
      for (int st = 0; st < DS; ++st) s = mma32(row_frag(qb + 32 * qt * D, rd, st), kf[st], s);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 ls = ld4f(lb + 32 * qt + 8 * j + 4 * hh);
        s[4 * j] = __builtin_amdgcn_exp2f(fmaf(s[4 * j], c, -ls.x));
        s[4 * j + 1] = __builtin_amdgcn_exp2f(fmaf(s[4 * j + 1], c, -ls.y));
        s[4 * j + 2] = __builtin_amdgcn_exp2f(fmaf(s[4 * j + 2], c, -ls.z));
        s[4 * j + 3] = __builtin_amdgcn_exp2f(fmaf(s[4 * j + 3], c, -ls.w));
      }
      if (masked) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = (uint32_t)(seen >> 32 * qt) >> (8 * (e >> 2) + (e & 3)) & 1 ? s[e] : 0.f;
      }
      bf16x8 pb[2];
      pack16<bf16>(s, pb);
      rd = reads.here();
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int d = 0; d < DT; ++d) dv[d] = mma32(tr_frag(db + (2 * qt + h) * 16 * D, rd, d), pb[h], dv[d]);
      rd = reads.here();
#pragma unroll
      for (int st = 0; st < DS; ++st)
        dp = mma32(row_frag(db + 32 * qt * D, rd, st), st < VR ? vf[st < VR ? st : 0] : ld8(vh + (st - VR) * kWave * 8), dp);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 de = ld4f(lb + kBK + 32 * qt + 8 * j + 4 * hh);
        s[4 * j] *= dp[4 * j] - de.x;
        s[4 * j + 1] *= dp[4 * j + 1] - de.y;
        s[4 * j + 2] *= dp[4 * j + 2] - de.z;
        s[4 * j + 3] *= dp[4 * j + 3] - de.w;
      }
      if (masked) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = (uint32_t)(seen >> 32 * qt) >> (8 * (e >> 2) + (e & 3)) & 1 ? s[e] : 0.f;
      }
      pack16<bf16>(s, pb);
      rd = reads.here();
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int d = 0; d < DT; ++d) dk[d] = mma32(tr_frag(qb + (2 * qt + h) * 16 * D, rd, d), pb[h], dk[d]);
    }
  };
  // The same with queries whose logarithm (`lbad`: all their weights are NaN) or delta (`dbad`: none of their ds is finite) is not
  // finite: their entries that are not are left out of the products, and the keys that see them become NaN, or of do's infinities
  // those, by sign.
  auto block_bad = [&](const bf16* qb, const bf16* db, const float* lb, int q0) {
    const uint64_t there = bits_below(to - q0), lbad = __ballot(!finite_f(lb[lane])) & there;
    const uint64_t dbad = __ballot(!finite_f(lb[kBK + lane])) & there;
    const int kk = wk0 + li, hi = kk < p.sinks ? to : imin(to, kk + p.window);
    const uint64_t seen = bits_below(hi - q0) & ~bits_below(imax(kk, from) - q0);
    const uint64_t seen_v = (seen & ~lbad) >> 4 * hh, seen_k = (seen & ~(lbad | dbad)) >> 4 * hh;
    const float to_k = seen & (lbad | dbad) ? NAN : 0.f, to_v = seen & lbad ? NAN : 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) dk[d] += to_k, dv[d] += to_v;
#pragma nounroll
    for (int qt = 0; qt < 2; ++qt) {
      TileReads<D> rd = reads.here();
      f32x16 s{}, dp{}, one;
#pragma unroll
      for (int st = 0; st < DS; ++st) s = mma32(row_frag(qb + 32 * qt * D, rd, st), kf[st], s);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const bool see = (uint32_t)(seen_v >> 32 * qt) >> (8 * (e >> 2) + (e & 3)) & 1;
        s[e] = see ? __builtin_amdgcn_exp2f(fmaf(s[e], c, -lb[32 * qt + 8 * (e >> 2) + 4 * hh + (e & 3)])) : 0.f;
        one[e] = see ? 1.f : 0.f;
      }
      bf16x8 pb[2], ones[2];
      pack16<bf16>(s, pb);
      pack16<bf16>(one, ones);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          bf16x8 x = tr_frag(db + (2 * qt + h) * 16 * D, rd, d), up, down;
          split_infinite<bf16>(x, up, down);
          dv[d] = mma32(x, pb[h], dv[d]);
          add_infinite<bf16>(dv[d], up, down, ones[h]);
        }
#pragma unroll
      for (int st = 0; st < DS; ++st)
        dp = mma32(row_frag(db + 32 * qt * D, rd, st), st < VR ? vf[st < VR ? st : 0] : ld8(vl + (st - VR) * kWave * 8), dp);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const bool see = (uint32_t)(seen_k >> 32 * qt) >> (8 * (e >> 2) + (e & 3)) & 1;
        s[e] = see ? s[e] * (dp[e] - lb[kBK + 32 * qt + 8 * (e >> 2) + 4 * hh + (e & 3)]) : 0.f;
      }
      pack16<bf16>(s, pb);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          bf16x8 x = tr_frag(qb + (2 * qt + h) * 16 * D, rd, d), up, down;
          split_infinite<bf16>(x, up, down);
          dk[d] = mma32(x, pb[h], dk[d]);
        }
    }
  };
  auto arrive = [&](int blk, bf16* qd, bf16* dd) {
    wait_loads();
    if ((blk + 1) * kBK > sq.len) {
      io.clean(sq.len - blk * kBK, qd);
      io.clean(sq.len - blk * kBK, dd);
    }
  };
  const int qb0 = from / kBK, nqb = from < to ? (to - 1) / kBK + 1 - qb0 : 0;
  const int step_by = far_job ? 2 : 2 * p.shares;  // blocks between two of a team's
  int g = 0, qb = 2 * share + team;  // the team's block: head of the group, block from qb0
  auto place = [&] {
    while (qb >= nqb && g < rep) qb -= nqb, ++g;
  };
  auto step = [&](const bf16* qc, const bf16* dc, const float* lc, bf16* qn, bf16* dn, float* ln) {
    const int g0 = g, q0 = (qb0 + qb) * kBK, q1 = q0 + kBK - 1;
    qb += step_by;
    place();
    if (g < rep) fetch(g, qb0 + qb, qn, dn, ln);
    if (g0 < rep && wave_live && !none_sees(q0, q1, wk0, wk0 + 31, p.window, p.sinks))
      block(q0 < from || q1 >= to || !all_see(q0, q1, wk0, wk0 + 31, p.window, p.sinks), qc, dc, lc, q0);
    if (g < rep) arrive(qb0 + qb, qn, dn);
    __syncthreads();
  };
  bf16 *const q0p = Qs0 + team * kBK * D, *const q1p = Qs1 + team * kBK * D, *const d0p = Ds0 + team * kBK * D, *const d1p = Ds1 + team * kBK * D;
  if (nqb) {
    place();
    if (g < rep) {
      fetch(g, qb0 + qb, q0p, d0p, Ls0[team]);
      arrive(qb0 + qb, q0p, d0p);
    }
    __syncthreads();
    const int turns = (rep * nqb + step_by - 1) / step_by;  // the same for both teams
    if constexpr (!BAD) {
      for (int n = 0; n < turns; n += 2) {
        step(q0p, d0p, Ls0[team], q1p, d1p, Ls1[team]);
        if (n + 1 < turns) step(q1p, d1p, Ls1[team], q0p, d0p, Ls0[team]);
      }
    } else {
      for (int n = 0; n < turns; ++n) {
        const int q0 = (qb0 + qb) * kBK, q1 = q0 + kBK - 1;
        if (g < rep && wave_live && !none_sees(q0, q1, wk0, wk0 + 31, p.window, p.sinks)) block_bad(q0p, d0p, Ls0[team], q0);
        qb += step_by;
        place();
        __syncthreads();
        if (g < rep) {
          fetch(g, qb0 + qb, q0p, d0p, Ls0[team]);
          arrive(qb0 + qb, q0p, d0p);
        }
        __syncthreads();
      }
    }
    // the second team's sums, a wave's 32 KB (16 KB) in a tile array
    f32x4* const sums = reinterpret_cast<f32x4*>(w == 0 ? Qs0 : w == 1 ? Qs1 : w == 2 ? Ds0 : Ds1) + lane;
    if (team) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sums[(4 * d + j) * kWave] = f32x4{dk[d][4 * j], dk[d][4 * j + 1], dk[d][4 * j + 2], dk[d][4 * j + 3]};
          sums[(4 * (DT + d) + j) * kWave] = f32x4{dv[d][4 * j], dv[d][4 * j + 1], dv[d][4 * j + 2], dv[d][4 * j + 3]};
        }
    }
    __syncthreads();
    if (!team) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x4 a = sums[(4 * d + j) * kWave], b = sums[(4 * (DT + d) + j) * kWave];
#pragma unroll
          for (int e = 0; e < 4; ++e) dk[d][4 * j + e] += a[e], dv[d][4 * j + e] += b[e];
        }
    }
  }
  if (team) return;
  const int64_t out = ((tok + kc) * p.HKV + job.hkv) * D;
  // sums that meet others': where those of key j go (dk; dv `dv_at` behind them), null: the result
  const bool alone = far_job || p.shares == 1;
  const int dv_at = alone ? p.sink_rows * D : D;
  auto part_at = [&](int j) -> float* {
    if (!alone) return p.near + ((share * all + tok + j) * p.HKV + job.hkv) * 2 * D;
    return slot >= 0 && j < p.sinks
               ? p.part + (slot * p.HKV + job.hkv) * 2 * p.sink_rows * D + (j - tile * kBQ) * D
               : nullptr;
  };
  float* const part = part_at(kc);
  if (row_ok) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = 32 * d + 8 * j + 4 * hh;
        const f32x4 a = {dk[d][4 * j], dk[d][4 * j + 1], dk[d][4 * j + 2], dk[d][4 * j + 3]};
        const f32x4 b = {dv[d][4 * j], dv[d][4 * j + 1], dv[d][4 * j + 2], dv[d][4 * j + 3]};
        if (part) {
          *reinterpret_cast<f32x4*>(part + at) = a;
          *reinterpret_cast<f32x4*>(part + dv_at + at) = b;
        } else {
          *reinterpret_cast<bf16x4*>(p.dk + out + at) = to_bf16x4(a[0] * p.scale, a[1] * p.scale, a[2] * p.scale, a[3] * p.scale);
          *reinterpret_cast<bf16x4*>(p.dv + out + at) = to_bf16x4(b[0], b[1], b[2], b[3]);
        }
      }
  }
}

// dk and dv of sinks that far queries see: the near queries' sums and each piece's, in order. A workgroup a near slot and kv head.
__global__ __launch_bounds__(256) void gated_delta_window_attn_sinks_kernel(WindowBwdParams p, int D) {
  const int hkv = blockIdx.x % p.HKV;
  const FarWork f = near_work(p.seqs, p.far, blockIdx.x / p.HKV);
  const Seq sq = f.sq;
  const int tile = f.sink_tile, len = sq.len;
  if (tile < 0) return;
  const int near = near_end(tile, p.window, len), rows = imin(imin(p.sinks, len) - tile * kBQ, kBQ);
  if (near >= len || rows <= 0) return;  // written where it was computed
  const int64_t first = far_slot(p.seqs, p.far, sq, tile), step = far_step(p.seqs, p.far, sq, p.B);
  const int q0 = p.far.first_query(), n0 = (near - q0) / p.far.far, n1 = (len - 1 - q0) / p.far.far;
  const int quads = D / 4;
  const int64_t one = (int64_t)2 * p.sink_rows * D, per = p.HKV * one;
  for (int i = threadIdx.x; i < 2 * rows * quads; i += 256) {
    const int which = i / (rows * quads), r = i / quads % rows, d = i % quads * 4;
    const int64_t at = hkv * one + (which * p.sink_rows + r) * D + d;
    const int64_t token = sq.row * p.seqs.T + sq.start + tile * kBQ + r;
    f32x4 x{};
    if (p.shares == 1) x = *reinterpret_cast<const f32x4*>(p.part + (p.far_jobs + near_slot(p.far, sq, tile)) * per + at);
    else
      for (int n = 0; n < p.shares; ++n)
        x += *reinterpret_cast<const f32x4*>(p.near + (((n * p.B * p.seqs.T + token) * p.HKV + hkv) * 2 + which) * D + d);
    for (int n = n0; n <= n1; ++n) x += *reinterpret_cast<const f32x4*>(p.part + (first + n * step) * per + at);
    if (!which) x *= p.scale;
    bf16* to = (which ? p.dv : p.dk) + (token * p.HKV + hkv) * D + d;
    *reinterpret_cast<bf16x4*>(to) = to_bf16x4(x[0], x[1], x[2], x[3]);
  }
}

// dk and dv of shared key tiles: the workgroups' sums, in order. Four columns a thread. Rows of sinks that far queries see are
// written again by the kernel above.
__global__ __launch_bounds__(256) void gated_delta_window_attn_join_kernel(WindowBwdParams p, int D) {
  const int64_t rows = p.B * p.seqs.T * p.HKV, quads = rows * 2 * D / 4;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < quads; i += (int64_t)gridDim.x * 256) {
    f32x4 x{};
    for (int n = 0; n < p.shares; ++n) x += *reinterpret_cast<const f32x4*>(p.near + (n * quads + i) * 4);
    const int64_t row = i / (D / 2);
    const int at = (int)(i - row * (D / 2)) * 4;
    if (at < D) x *= p.scale;
    *reinterpret_cast<bf16x4*>((at < D ? p.dk : p.dv) + row * D + at % D) = to_bf16x4(x[0], x[1], x[2], x[3]);
  }
}

// ------------------------------------------------------------------------------------------------ host
static int window_check(const char* name, int64_t B, int64_t T, int64_t HQ, int64_t HKV, int64_t D, int64_t N, const void* cu,
                        const int64_t* st, int64_t window, int64_t sinks, float scale) {
  if (B <= 0 || T < 0 || HQ <= 0 || HKV <= 0 || HQ % HKV || N <= 0 || (cu ? B != 1 : N != B) || window < 0 || sinks < 0) {
    gdn_internal_set_error("%s: bad sizes B=%lld T=%lld HQ=%lld HKV=%lld N=%lld window=%lld sinks=%lld (HQ a multiple of HKV; "
                           "cu_seqlens requires B == 1)", name, (long long)B, (long long)T, (long long)HQ, (long long)HKV,
                           (long long)N, (long long)window, (long long)sinks);
    return GDN_ERR_INVALID;
  }
  if (D != 64 && D != 128) {
    gdn_internal_set_error("%s: head dim %lld unsupported (64 or 128)", name, (long long)D);
    return GDN_ERR_UNSUPPORTED;
  }
  if (!(scale > 0.f) || scale > 2.0e38f) {
    gdn_internal_set_error("%s: scale %g unsupported (a positive finite softmax scale)", name, (double)scale);
    return GDN_ERR_INVALID;
  }
  if (T >= kFar / 2 || N >= kFar || HQ > 65536 || B * T > (1LL << 40)) {
    gdn_internal_set_error("%s: too many tokens or heads (B=%lld T=%lld N=%lld HQ=%lld)", name, (long long)B, (long long)T,
                           (long long)N, (long long)HQ);
    return GDN_ERR_UNSUPPORTED;
  }
  for (int i = 0; i < 9; ++i)
    if (st[i] < 0 || st[i] % 8 || (i % 3 == 1 && st[i] * 2 > kMaxRowBytes)) {
      gdn_internal_set_error("%s: strides must be multiples of 8 elements, between tokens at most %lld bytes", name,
                             (long long)kMaxRowBytes);
      return GDN_ERR_INVALID;
    }
  if (HQ * D * 2 > kMaxRowBytes) {
    gdn_internal_set_error("%s: HQ * D = %lld too large", name, (long long)(HQ * D));
    return GDN_ERR_UNSUPPORTED;
  }
  return GDN_OK;
}

static int far_window(int64_t window) { return window <= 0 || window > kFar ? kFar : (int)window; }
// without a window sinks say nothing; sinks as far as the first window reaches neither change who sees what, nor are they cut
static int far_sinks(int64_t window, int64_t sinks) { return window <= 0 ? 0 : sinks > kFar ? kFar : (int)sinks; }

// Far queries a job, with one tile of sinks: short jobs, which fill up the CUs behind the near ones.
constexpr int kFarPiece = 256;
constexpr int64_t kCus = 256;

struct FarPlan {
  FarList list;
  int sink_rows;
  int64_t jobs, near;  // slots of far pieces and of near queries, both times tiles of sinks
};
// Slots by number where all sequences together have no more tiles of sinks than there is room for by start (batch rows always);
// else by start: 65,536 tokens in 2,000 documents, 8 kv heads of 128, window 256, 4 sinks take 138 MB, by number 1.1 GB.
static FarPlan far_plan(int64_t B, int64_t T, int64_t N, bool varlen, int window, int sinks) {
  FarPlan f{FarList{kFarPiece, 0, 0, 0}, 0, 0, 0};
  if (!sinks || (int64_t)window + kBQ > T) return f;  // every query is a near one
  FarList& l = f.list;
  const int64_t some = sinks < T ? sinks : T;
  l.tiles = (int)((some + kBQ - 1) / kBQ);
  l.far = kFarPiece * l.tiles;  // with more tiles longer pieces: the partial sums stay as large
  l.reach = window + kBQ;
  const int by_start = far_by_start(l.reach, l.tiles);
  if (varlen && N * l.tiles > T / by_start) {
    l.by_start = by_start;
    f.jobs = f.near = T / by_start;
  } else {
    f.jobs = (varlen ? packed_tiles(T, N, 1, l.far) : B * ((T + l.far - 1) / l.far)) * l.tiles;
    f.near = N * l.tiles;
  }
  f.sink_rows = l.tiles > 1 ? kBQ : (int)((some + 31) / 32 * 32);
  return f;
}

// Workgroups that share a key tile's queries: as many as there are idle CUs for, with 8 blocks of queries each at least; and
// where the first tiles have twice the average to do (no window), two waves of workgroups, with 24 blocks each at least.
// Measured, training step of 16 query heads and D = 128 in us, one workgroup a tile -> this rule: 1,024 tokens of 1 kv head
// 611 -> 123; 4,096 of 4 without a window 762 -> 418, window 512 182 -> 152; 8,192 of 4 1,792 -> 1,283. The other side: three
// waves and 8 blocks cost 4,096 tokens of 16 kv heads 414 -> 447, sharing where far pieces of sinks fill the card
// (4,096 tokens, 4 kv heads, window 300) 158 -> 182. Each share costs 8 D bytes a key and kv head, written and read.
static int dkv_shares(int64_t T, int64_t HQ, int64_t HKV, int64_t k_tiles, int64_t far_tiles, int window) {
  const int64_t jobs = k_tiles * HKV, blocks = HQ / HKV * ((T < window + kBQ ? T : window + kBQ) / kBK + 1);
  const int64_t idle = (kCus - far_tiles * HKV) / jobs;
  int64_t n = idle < blocks / 8 ? idle : blocks / 8;
  if (window > T / 2) {
    const int64_t even = (2 * kCus + jobs - 1) / jobs, m = even < blocks / 24 ? even : blocks / 24;
    n = n > m ? n : m;
  }
  return (int)(n < 1 ? 1 : n > 16 ? 16 : n);
}

struct BwdSizes {
  FarPlan far;
  int64_t tiles;
  int shares;
  size_t delta, part, near;  // bytes
};
static BwdSizes bwd_sizes(int64_t B, int64_t T, int64_t HQ, int64_t HKV, int64_t D, int64_t N, bool varlen, int window, int sinks) {
  BwdSizes b{far_plan(B, T, N, varlen, window, sinks), varlen ? packed_tiles(T, N, 1, kBQ) : B * ((T + kBQ - 1) / kBQ), 1, 0, 0, 0};
  b.shares = dkv_shares(T, HQ, HKV, b.tiles, b.far.jobs, window);
  b.delta = ((size_t)(B * T * HQ) * 4 + 255) / 256 * 256;
  b.part = (size_t)(b.far.jobs + b.far.near) * HKV * 2 * b.far.sink_rows * D * 4;
  b.near = b.shares > 1 ? (size_t)b.shares * B * T * HKV * 2 * D * 4 : 0;
  return b;
}

}  // namespace gdn

using namespace gdn;

extern "C" int gdn_window_attn_fwd(const void* q, int64_t q_batch_stride, int64_t q_token_stride, int64_t q_head_stride,
                                   const void* k, int64_t k_batch_stride, int64_t k_token_stride, int64_t k_head_stride,
                                   const void* v, int64_t v_batch_stride, int64_t v_token_stride, int64_t v_head_stride,
                                   void* o, float* kept, const void* cu_seqlens, int64_t B, int64_t T, int64_t HQ, int64_t HKV,
                                   int64_t D, int64_t N, int dtype, int64_t window, int64_t sinks, float scale, unsigned flags,
                                   void* stream) {
  const int64_t st[9] = {q_batch_stride, q_token_stride, q_head_stride, k_batch_stride, k_token_stride, k_head_stride,
                         v_batch_stride, v_token_stride, v_head_stride};
  if (int rc = window_check("gdn_window_attn_fwd", B, T, HQ, HKV, D, N, cu_seqlens, st, window, sinks, scale)) return rc;
  if (dtype != GDN_DTYPE_BF16 && dtype != GDN_DTYPE_F16) {
    gdn_internal_set_error("gdn_window_attn_fwd: dtype %d unsupported (bf16 or fp16)", dtype);
    return GDN_ERR_UNSUPPORTED;
  }
  if (T == 0) return GDN_OK;
  if (!q || !k || !v || !o || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                                reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(kept)) & 15)) {
    gdn_internal_set_error("gdn_window_attn_fwd: null or misaligned (16 bytes) tensor pointer");
    return GDN_ERR_INVALID;
  }
  FlashParams p{};
  p.q = q, p.k = k, p.v = v, p.o = o;
  p.o_rest = kept, p.lse = kept ? kept + B * T * HQ * D / 2 : nullptr;
  p.qsb = st[0], p.qst = st[1], p.qsh = st[2], p.ksb = st[3], p.kst = st[4], p.ksh = st[5], p.vsb = st[6], p.vst = st[7], p.vsh = st[8];
  p.seqs = Packed{cu_seqlens, (flags & GDN_FLAG_CU_INT32) ? 1 : 0, N, T};
  p.B = B;
  p.tiles = cu_seqlens ? packed_tiles(T, N, 1, kBQ) : B * ((T + kBQ - 1) / kBQ);
  p.HQ = (int)HQ, p.HKV = (int)HKV, p.parts = job_parts(HKV);
  p.window = far_window(window), p.sinks = far_sinks(window, sinks);
  p.scale_log2 = scale * 1.4426950408889634f;
  const int64_t groups = job_groups(HKV, HQ / HKV, p.tiles);
  if (groups > kMaxGroups256) {
    gdn_internal_set_error("gdn_window_attn_fwd: grid too large");
    return GDN_ERR_UNSUPPORTED;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)groups), block(256);
  if (dtype == GDN_DTYPE_BF16) {
    if (D == 128) hipLaunchKernelGGL((gated_delta_window_attn_fwd_kernel<128, bf16>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((gated_delta_window_attn_fwd_kernel<64, bf16>), grid, block, 0, s, p);
  } else {
    if (D == 128) hipLaunchKernelGGL((gated_delta_window_attn_fwd_kernel<128, f16>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((gated_delta_window_attn_fwd_kernel<64, f16>), grid, block, 0, s, p);
  }
  return gdn_internal_check_launch("gated_delta_window_attn_fwd_kernel");
}

extern "C" size_t gdn_window_attn_bwd_workspace_size(int64_t B, int64_t T, int64_t HQ, int64_t HKV, int64_t D, int64_t N,
                                                     int64_t window, int64_t sinks, int varlen) {
  if (B <= 0 || T <= 0 || HQ <= 0 || HKV <= 0 || HQ % HKV || D <= 0 || N <= 0 || window < 0 || sinks < 0) return 0;
  const BwdSizes b = bwd_sizes(B, T, HQ, HKV, D, N, varlen != 0, far_window(window), far_sinks(window, sinks));
  return b.delta + b.part + b.near;
}

extern "C" int gdn_window_attn_bwd(const void* q, int64_t q_batch_stride, int64_t q_token_stride, int64_t q_head_stride,
                                   const void* k, int64_t k_batch_stride, int64_t k_token_stride, int64_t k_head_stride,
                                   const void* v, int64_t v_batch_stride, int64_t v_token_stride, int64_t v_head_stride,
                                   const void* o, const float* kept, const void* d_o, const void* cu_seqlens, int64_t B, int64_t T,
                                   int64_t HQ, int64_t HKV, int64_t D, int64_t N, int64_t window, int64_t sinks, float scale,
                                   unsigned flags, void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  const int64_t st[9] = {q_batch_stride, q_token_stride, q_head_stride, k_batch_stride, k_token_stride, k_head_stride,
                         v_batch_stride, v_token_stride, v_head_stride};
  if (int rc = window_check("gdn_window_attn_bwd", B, T, HQ, HKV, D, N, cu_seqlens, st, window, sinks, scale)) return rc;
  if (T == 0) return GDN_OK;
  uintptr_t every = 0;
  bool null = false;
  const void* const all[] = {q, k, v, o, kept, d_o, dq, dk, dv, workspace};
  for (const void* x : all) every |= reinterpret_cast<uintptr_t>(x), null |= !x;
  if (null || (every & 15)) {
    gdn_internal_set_error("gdn_window_attn_bwd: null or misaligned (16 bytes) tensor pointer");
    return GDN_ERR_INVALID;
  }
  const size_t need = gdn_window_attn_bwd_workspace_size(B, T, HQ, HKV, D, N, window, sinks, cu_seqlens != nullptr);
  if (workspace_bytes < need) {
    gdn_internal_set_error("gdn_window_attn_bwd: workspace of %zu bytes needed", need);
    return GDN_ERR_INVALID;
  }
  WindowBwdParams p{};
  p.q = static_cast<const bf16*>(q), p.k = static_cast<const bf16*>(k), p.v = static_cast<const bf16*>(v);
  p.o = static_cast<const bf16*>(o), p.d_o = static_cast<const bf16*>(d_o);
  p.o_rest = reinterpret_cast<const bf16*>(kept), p.lse = kept + B * T * HQ * D / 2;
  p.qsb = st[0], p.qst = st[1], p.qsh = st[2], p.ksb = st[3], p.kst = st[4], p.ksh = st[5], p.vsb = st[6], p.vst = st[7], p.vsh = st[8];
  p.dq = static_cast<bf16*>(dq), p.dk = static_cast<bf16*>(dk), p.dv = static_cast<bf16*>(dv);
  p.delta = static_cast<float*>(workspace);
  p.seqs = Packed{cu_seqlens, (flags & GDN_FLAG_CU_INT32) ? 1 : 0, N, T};
  p.B = B;
  p.HQ = (int)HQ, p.HKV = (int)HKV, p.parts = job_parts(HKV);
  p.window = far_window(window), p.sinks = far_sinks(window, sinks);
  p.scale = scale, p.scale_log2 = scale * 1.4426950408889634f;
  const BwdSizes sizes = bwd_sizes(B, T, HQ, HKV, D, N, cu_seqlens != nullptr, p.window, p.sinks);
  const FarPlan& f = sizes.far;
  p.q_tiles = p.k_tiles = sizes.tiles;
  p.shares = sizes.shares;
  p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + sizes.delta);
  p.near = reinterpret_cast<float*>(static_cast<char*>(workspace) + sizes.delta + sizes.part);
  p.far = f.list, p.far_jobs = f.jobs, p.sink_rows = f.sink_rows;
  const int64_t q_groups = job_groups(HKV, HQ / HKV, p.q_tiles);
  const int64_t k_groups = job_groups(HKV, 1, p.k_tiles * p.shares + p.far_jobs), s_groups = f.near * HKV;
  if (q_groups > kMaxGroups256 || k_groups > kMaxGroups256 / 2 || s_groups > kMaxGroups256) {  // k_groups: of 512 threads
    gdn_internal_set_error("gdn_window_attn_bwd: grid too large");
    return GDN_ERR_UNSUPPORTED;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 block(256);
  if (D == 128) hipLaunchKernelGGL(gated_delta_window_attn_dq_kernel<128>, dim3((unsigned)q_groups), block, 0, s, p);
  else hipLaunchKernelGGL(gated_delta_window_attn_dq_kernel<64>, dim3((unsigned)q_groups), block, 0, s, p);
  if (int rc = gdn_internal_check_launch("gated_delta_window_attn_dq_kernel")) return rc;
  if (D == 128) hipLaunchKernelGGL((gated_delta_window_attn_dkv_kernel<128, false>), dim3((unsigned)k_groups), dim3(512), 0, s, p);
  else hipLaunchKernelGGL((gated_delta_window_attn_dkv_kernel<64, false>), dim3((unsigned)k_groups), dim3(512), 0, s, p);
  if (int rc = gdn_internal_check_launch("gated_delta_window_attn_dkv_kernel")) return rc;
  if (D == 128) hipLaunchKernelGGL((gated_delta_window_attn_dkv_kernel<128, true>), dim3((unsigned)k_groups), dim3(512), 0, s, p);
  else hipLaunchKernelGGL((gated_delta_window_attn_dkv_kernel<64, true>), dim3((unsigned)k_groups), dim3(512), 0, s, p);
  if (int rc = gdn_internal_check_launch("gated_delta_window_attn_dkv_kernel")) return rc;
  if (p.shares > 1) {
    const int64_t quads = B * T * HKV * 2 * D / 4, groups = (quads + 255) / 256;
    hipLaunchKernelGGL(gated_delta_window_attn_join_kernel, dim3((unsigned)(groups < 4096 ? groups : 4096)), block, 0, s, p, (int)D);
    if (int rc = gdn_internal_check_launch("gated_delta_window_attn_join_kernel")) return rc;
  }
  if (f.near) {
    hipLaunchKernelGGL(gated_delta_window_attn_sinks_kernel, dim3((unsigned)s_groups), block, 0, s, p, (int)D);
    return gdn_internal_check_launch("gated_delta_window_attn_sinks_kernel");
  }
  return GDN_OK;
}
