// Linear attention with a decay for each head, token by token: S = exp(g) S + k v^T, o = scale S^T q, in fp32.
//
// A workgroup of 4 waves holds 64 columns of one (sequence, value head) state in registers: thread t the columns
// 4 (t % 16) .. + 3 of the rows t / 16 + 16 i. The state is read once and written once, which is what bounds the step of
// one token; the tokens' rows pass through LDS 16 at a time. A token's output is a sum over all rows: 4 row groups by
// lane swaps, the 4 waves through LDS after the 16 tokens, so that 16 tokens take two barriers. A token for 64 sequences of 16
// heads of 128: 24 us for 135 MB, 5.6 TB/s; for one sequence 4.5 us. Long calls go token by token, 0.6 us each: 4,096 tokens
// of 16 heads of 128 in fp32 take 2.5 ms for one sequence and 2.9 for four.

#include <type_traits>

#include "gdn_common.h"

namespace gdn {

struct LinRecParams {
  const void *q, *k, *v, *g;
  const float* h0;
  void* o;
  float* ht;
  const void* cu;
  int cu_i32, dg, zero_rest;  // zero_rest: write zeros to the rows of o outside all sequences
  int64_t gb, gt, gh;
  int64_t T, N, H, HV, slices;  // slices: V / 64
  float scale;
};

constexpr int kLinRecTok = 16;  // tokens in LDS

template <typename E, int KD>
__global__ __launch_bounds__(256) void gated_deltaless_recurrent_kernel(LinRecParams p) {
  constexpr int RPT = KD / 16;
  __shared__ __align__(16) float qs[kLinRecTok][KD], ks[kLinRecTok][KD], vs[kLinRecTok][64], as[kLinRecTok];
  __shared__ __align__(16) float red[kLinRecTok][4][64];
  const int t = threadIdx.x, cg = t % 16, rg = t / 16, lane = t % kWave, w = t / kWave;
  const int64_t sl = blockIdx.x % p.slices, hv = blockIdx.x / p.slices % p.HV, n = blockIdx.x / p.slices / p.HV;
  const int64_t VD = p.slices * 64, h = hv / (p.HV / p.H);
  E* o = static_cast<E*>(p.o);
  int64_t tok0 = n * p.T, len = p.T;
  if (p.cu) {
    // captured calls do not check the bounds: nothing outside the tensors is touched whatever they hold
    const int64_t a = load_index(p.cu, p.cu_i32, n), e = load_index(p.cu, p.cu_i32, n + 1);
    tok0 = a < 0 ? 0 : a > p.T ? p.T : a;
    const int64_t end = e < 0 ? 0 : e > p.T ? p.T : e;
    len = end - tok0;
    if (p.zero_rest) {  // the rows before the first sequence and behind the last
      if (n == 0)
        for (int64_t c = t; c < tok0 * 64; c += 256) o[(c / 64 * p.HV + hv) * VD + sl * 64 + c % 64] = (E)0.f;
      if (n == p.N - 1)
        for (int64_t c = end * 64 + t; c < p.T * 64; c += 256) o[(c / 64 * p.HV + hv) * VD + sl * 64 + c % 64] = (E)0.f;
    }
  }
  const int64_t st0 = (n * p.HV + hv) * KD * VD + sl * 64 + 4 * cg;
  float4 s[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i)
    s[i] = p.h0 ? *reinterpret_cast<const float4*>(p.h0 + st0 + (rg + 16 * i) * VD) : float4{0.f, 0.f, 0.f, 0.f};
  const E *q = static_cast<const E*>(p.q), *k = static_cast<const E*>(p.k), *v = static_cast<const E*>(p.v);
  const int64_t g0 = p.cu ? tok0 * p.gt : n * p.gb;
  for (int64_t t0 = 0; t0 < len; t0 += kLinRecTok) {
    const int nt = len - t0 < kLinRecTok ? (int)(len - t0) : kLinRecTok;
    for (int c = t; c < nt * KD; c += 256) {
      const int64_t at = ((tok0 + t0 + c / KD) * p.H + h) * KD + c % KD;
      qs[c / KD][c % KD] = (float)q[at] * p.scale;
      ks[c / KD][c % KD] = (float)k[at];
    }
    for (int c = t; c < nt * 64; c += 256)
      vs[c / 64][c % 64] = (float)v[((tok0 + t0 + c / 64) * p.HV + hv) * VD + sl * 64 + c % 64];
    if (t < nt) as[t] = p.g ? expf(load_as_f32(p.g, p.dg, g0 + (t0 + t) * p.gt + hv * p.gh)) : 1.f;
    __syncthreads();
    for (int j = 0; j < nt; ++j) {
      const float a = as[j];
      const float4 vv = *reinterpret_cast<const float4*>(&vs[j][4 * cg]);
      float x = 0.f, y = 0.f, z = 0.f, u = 0.f;
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const float kr = ks[j][rg + 16 * i], qr = qs[j][rg + 16 * i];
        s[i].x = a * s[i].x + kr * vv.x;
        s[i].y = a * s[i].y + kr * vv.y;
        s[i].z = a * s[i].z + kr * vv.z;
        s[i].w = a * s[i].w + kr * vv.w;
        x += qr * s[i].x;
        y += qr * s[i].y;
        z += qr * s[i].z;
        u += qr * s[i].w;
      }
      x = xor32_sum(xor16_sum(x));
      y = xor32_sum(xor16_sum(y));
      z = xor32_sum(xor16_sum(z));
      u = xor32_sum(xor16_sum(u));
      if (lane < 16) *reinterpret_cast<float4*>(&red[j][w][4 * cg]) = float4{x, y, z, u};
    }
    __syncthreads();
    for (int c = t; c < nt * 64; c += 256) {
      const int j = c / 64, col = c % 64;
      o[((tok0 + t0 + j) * p.HV + hv) * VD + sl * 64 + col] =
          (E)((red[j][0][col] + red[j][1][col]) + (red[j][2][col] + red[j][3][col]));
    }
  }
  if (p.ht) {
#pragma unroll
    for (int i = 0; i < RPT; ++i) *reinterpret_cast<float4*>(p.ht + st0 + (rg + 16 * i) * VD) = s[i];
  }
}

}  // namespace gdn

using namespace gdn;

extern "C" int gdn_decay_attn_recurrent_fwd(const void* q, const void* k, const void* v, const void* g,
                                            const float* initial_state, void* o, float* final_state,
                                            const void* cu_seqlens, int64_t B, int64_t T, int64_t H, int64_t HV, int64_t K,
                                            int64_t V, int64_t N, int qkv_dtype, int g_dtype, int64_t g_batch_stride,
                                            int64_t g_token_stride, int64_t g_head_stride, float scale, unsigned flags,
                                            void* stream) {
  const char* name = "gdn_decay_attn_recurrent_fwd";
  if (B <= 0 || T < 0 || H <= 0 || HV <= 0 || HV % H || N <= 0 || (cu_seqlens ? B != 1 : N != B)) {
    gdn_internal_set_error("%s: bad sizes B=%lld T=%lld H=%lld HV=%lld N=%lld (cu_seqlens requires B == 1, N == B without "
                           "it)", name, (long long)B, (long long)T, (long long)H, (long long)HV, (long long)N);
    return GDN_ERR_INVALID;
  }
  if (T > 0 && (!q || !k || !v || !o)) {
    gdn_internal_set_error("%s: null tensor pointer", name);
    return GDN_ERR_INVALID;
  }
  if ((K != 64 && K != 128) || (V != 64 && V != 128)) {
    gdn_internal_set_error("%s: head dims K=%lld V=%lld unsupported (each must be 64 or 128)", name, (long long)K,
                           (long long)V);
    return GDN_ERR_UNSUPPORTED;
  }
  if (qkv_dtype < GDN_DTYPE_F32 || qkv_dtype > GDN_DTYPE_F16 || g_dtype < GDN_DTYPE_F32 || g_dtype > GDN_DTYPE_F16) {
    gdn_internal_set_error("%s: unknown dtype %d / %d", name, qkv_dtype, g_dtype);
    return GDN_ERR_INVALID;
  }
  if ((reinterpret_cast<uintptr_t>(initial_state) | reinterpret_cast<uintptr_t>(final_state)) & 15) {
    gdn_internal_set_error("%s: states must be 16-byte aligned", name);
    return GDN_ERR_INVALID;
  }
  const int64_t blocks = N * HV * (V / 64);
  if (blocks > kMaxGroups256) {
    gdn_internal_set_error("%s: too many sequences and heads for one launch", name);
    return GDN_ERR_UNSUPPORTED;
  }
  LinRecParams p{q, k, v, g, initial_state, o, final_state, cu_seqlens, (flags & GDN_FLAG_CU_INT32) ? 1 : 0, g_dtype,
                 (flags & GDN_FLAG_ZERO_REST) ? 1 : 0, g_batch_stride, g_token_stride, g_head_stride, T, N, H, HV, V / 64, scale};
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto e) {
    using E = decltype(e);
    if (K == 128) hipLaunchKernelGGL((gated_deltaless_recurrent_kernel<E, 128>), dim3((unsigned)blocks), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((gated_deltaless_recurrent_kernel<E, 64>), dim3((unsigned)blocks), dim3(256), 0, s, p);
  };
  if (qkv_dtype == GDN_DTYPE_BF16) go(bf16{});
  else if (qkv_dtype == GDN_DTYPE_F16) go(f16{});
  else go(float{});
  return gdn_internal_check_launch("gated_deltaless_recurrent_kernel");
}
