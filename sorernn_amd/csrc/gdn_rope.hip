// RMSNorm of every query and key head with the rotary position embedding in the same pass, and its backward.
//
//   y = x rsqrt(mean(x^2) + eps) w;  out = y with its first rot entries rotated: (lo c - hi s, hi c + lo s),
//   lo = y[0 : rot / 2], hi = y[rot / 2 : rot], c, s = cos, sin(position theta^(-2f / rot)), f = 0 .. rot / 2 - 1
//
// fp32 throughout, one rounding at the end. Bound by the bytes of the rows: 16,384 tokens of 16 + 16 heads of 128 in bf16 take
// 62 us forward and 92 backward as slices of a projection in memory, 4.3 and 4.4 TB/s. A wave takes a token (with few tokens a
// workgroup's 4 waves share one) and its heads D / 8 lanes each; a lane holds two pieces of 4 elements that turn with one
// another, so that nothing is exchanged between lanes but the sum of squares. Angles are taken in turns in 64 bits,
// position * (theta^(-2f / rot) / 2 pi) less its whole part: at position 1,000,000 a 32-bit angle is off by 0.06 rad.
// A token's rot / 2 pairs of cos and sin are computed once for all its heads and pass through LDS.

#include <math.h>

#include <type_traits>

#include "gdn_common.h"

namespace gdn {

// Workgroups of the backward, at most: each leaves one row of weight gradient sums, which a second kernel adds. bf16, with
// 256, 512 and 1,024 of them, both kernels: 16 + 16 heads of 128, 4,096 tokens 31, 28 and 28 us, 16,384 tokens 108, 89 and
// 86; 1 + 1 heads of 64, 4,096 tokens 13, 11 and 14, 16,384 tokens 32, 22 and 23.
constexpr int64_t kRopeBwdBlocks = 512;
// Up to this many tokens the 4 waves of a workgroup share one: a workgroup a CU. Shared and a wave each, bf16, us:
//   heads x D       256 tokens: forward   backward      512 tokens: forward   backward
//   16 + 16 x 128             4.6, 6.3    9.3, 11.0               6.8, 6.6   11.7, 11.6
//   16 + 2 x 128              4.5, 5.5    8.8, 9.8                6.3, 5.6   11.2, 10.2
//   8 + 8 x 256               4.8, 6.4    9.3, 10.9               7.1, 6.7   12.4, 11.7
//   1 + 1 x 128               4.1, 4.1    8.3, 7.6                5.7, 4.1   10.5, 7.9
// With few heads three of the waves have no rows, which costs the backward 0.7 us from 128 tokens on.
constexpr int64_t kRopeShared = 256;

struct QkRopeParams {
  const void* x[2];              // q, k [B, T, heads, D] by strides (elements), last axis contiguous
  int64_t sb[2], st[2], sh[2];
  const void* dy[2];             // backward: [B, T, heads, D] contiguous
  const float* w[2];             // [D] or null
  void* y[2];                    // forward: out, backward: dx; contiguous
  float* partial;                // backward: [blocks][2][D]
  const void* pos;               // [B, T] by strides, or null: the token index, from each document's start with cu
  int64_t pb, pt;
  const void* cu;
  int pos_i32, cu_i32;
  int64_t T, N, tokens;
  int heads[2], rot, wpt;        // wpt: waves that share a token
  float eps;
  double turns[128];             // theta^(-2f / rot) / 2 pi
};

__device__ __forceinline__ int64_t rope_position(const QkRopeParams& p, int64_t bt, int64_t bi, int64_t ti) {
  if (p.pos) return load_index(p.pos, p.pos_i32, bi * p.pb + ti * p.pt);
  if (!p.cu) return ti;
  int64_t lo = 0, hi = p.N;  // cu[lo] <= bt < cu[hi]
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (load_index(p.cu, p.cu_i32, mid) <= bt) lo = mid;
    else hi = mid;
  }
  return bt - load_index(p.cu, p.cu_i32, lo);
}

template <int D, typename E, bool BWD>
__global__ __launch_bounds__(256) void gated_delta_qk_norm_rope_kernel(QkRopeParams p) {
  constexpr int LPR = D / 8, RPW = kWave / LPR, U = sizeof(E) == 2 ? 4 : 2;  // lanes a row, rows a pass, passes in flight
  using V4 __attribute__((aligned(4 * sizeof(E)))) = E __attribute__((ext_vector_type(4)));
  __shared__ __align__(16) float tab[4][2][D / 2];
  __shared__ float sums[BWD ? 4 * RPW * 2 * D : 1];
  const int lane = threadIdx.x % kWave, w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int li = lane % LPR, sub = lane / LPR, half = p.rot >> 1, np = half >> 2;
  const bool in_rot = li < np;
  const int d0 = in_rot ? 4 * li : p.rot + 8 * (li - np), d1 = in_rot ? d0 + half : d0 + 4;  // the lane's two pieces
  const int hs = p.heads[0] + p.heads[1], r_first = (w % p.wpt) * RPW + sub, r_step = p.wpt * RPW;
  float wt[2][8], dw[2][8];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      wt[m][e] = p.w[m] ? p.w[m][(e < 4 ? d0 : d1) + (e & 3)] : 1.f;
      dw[m][e] = 0.f;
    }
  const int64_t stride = (int64_t)gridDim.x * 4 / p.wpt;
  for (int64_t bt = ((int64_t)blockIdx.x * 4 + w) / p.wpt; bt < p.tokens; bt += stride) {
    const int64_t bi = bt / p.T, ti = bt - bi * p.T;
    const E* x0[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) x0[m] = static_cast<const E*>(p.x[m]) + bi * p.sb[m] + ti * p.st[m];
    const E *dy0 = static_cast<const E*>(p.dy[0]) + bt * p.heads[0] * D, *dy1 = static_cast<const E*>(p.dy[1]) + bt * p.heads[1] * D;
    E *y0 = static_cast<E*>(p.y[0]) + bt * p.heads[0] * D, *y1 = static_cast<E*>(p.y[1]) + bt * p.heads[1] * D;
    V4 xv[U][2], dv[U][2];
    auto load = [&](int r0) {  // U passes' rows; past the last head the last again
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * r_step < hs ? r0 + u * r_step : hs - 1;
        const bool m = r >= p.heads[0];
        const int hh = r - (m ? p.heads[0] : 0);
        const E* src = (m ? x0[1] : x0[0]) + hh * (m ? p.sh[1] : p.sh[0]);
        xv[u][0] = *reinterpret_cast<const V4*>(src + d0);
        xv[u][1] = *reinterpret_cast<const V4*>(src + d1);
        if (BWD) {
          const E* up = (m ? dy1 : dy0) + hh * D;
          dv[u][0] = *reinterpret_cast<const V4*>(up + d0);
          dv[u][1] = *reinterpret_cast<const V4*>(up + d1);
        }
      }
    };
    int r0 = r_first;
    load(r0);
    const int64_t pos = rope_position(p, bt, bi, ti);
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
    float c[4], s[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c[e] = in_rot ? tab[w][0][d0 + e] : 1.f;
      s[e] = in_rot ? tab[w][1][d0 + e] : 0.f;
    }
    for (; r0 < hs; r0 += U * r_step) {  // uniform inside a row's lanes
      if (r0 != r_first) load(r0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * r_step;
        if (r >= hs) break;
        const bool m = r >= p.heads[0];
        float x[8], ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = (float)xv[u][e >> 2][e & 3];
          ss += x[e] * x[e];
        }
        const float rr = 1.f / sqrtf(group_sum<LPR>(ss) / (float)D + p.eps);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = BWD ? (float)dv[u][e >> 2][e & 3] : x[e] * rr * (m ? wt[1][e] : wt[0][e]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = y[e], b = y[4 + e], sn = BWD ? -s[e] : s[e];  // the backward turns by the negative angle
          y[e] = a * c[e] - b * sn;
          y[4 + e] = b * c[e] + a * sn;
        }
        if (BWD) {
          float dot = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float add = y[e] * (x[e] * rr);
            dw[0][e] += m ? 0.f : add;
            dw[1][e] += m ? add : 0.f;
            y[e] *= m ? wt[1][e] : wt[0][e];
            dot += y[e] * x[e];
          }
          const float k = rr * (rr * (group_sum<LPR>(dot) / (float)D));  // of the order of y: r^3 alone may be subnormal
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = rr * y[e] - x[e] * rr * k;
        }
        V4 o0, o1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o0[e] = (E)y[e];
          o1[e] = (E)y[4 + e];
        }
        E* dst = (m ? y1 : y0) + (int64_t)(r - (m ? p.heads[0] : 0)) * D;
        *reinterpret_cast<V4*>(dst + d0) = o0;
        *reinterpret_cast<V4*>(dst + d1) = o1;
      }
    }
    __builtin_amdgcn_wave_barrier();  // the table is read before the next token's is written
  }
  if (BWD && p.partial) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[((w * RPW + sub) * 2 + m) * D + (e < 4 ? d0 : d1) + (e & 3)] = dw[m][e];
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * D; c += 256) {
      float x = 0.f;
      for (int r = 0; r < 4 * RPW; ++r) x += sums[r * 2 * D + c];
      p.partial[(int64_t)blockIdx.x * 2 * D + c] = x;
    }
  }
}

// The weights' gradients from the workgroups' sums: 16 columns a workgroup, 64 threads a column, in a fixed order.
__global__ __launch_bounds__(1024) void gated_delta_qk_norm_rope_param_grad_kernel(const float* partial, int rows, int D,
                                                                                  float* dqw, float* dkw) {
  __shared__ float part[64][17];
  const int col = threadIdx.x % 16, at = blockIdx.x * 16 + col;
  float x = 0.f;
#pragma unroll 8
  for (int r = threadIdx.x / 16; r < rows; r += 64) x += partial[(int64_t)r * 2 * D + at];
  part[threadIdx.x / 16][col] = x;
  __syncthreads();
  if (threadIdx.x >= 16) return;
  x = 0.f;
  for (int r = 0; r < 64; ++r) x += part[r][col];
  float* out = at < D ? dqw : dkw;
  if (out) out[at % D] = x;
}

static int rope_check(const char* name, QkRopeParams& p, int64_t B, int64_t T, int64_t HQ, int64_t HK, int64_t D, int64_t N,
                      int dtype, int rot_dim, double theta, float eps) {
  if (B <= 0 || T < 0 || HQ <= 0 || HK <= 0 || HQ + HK > 65536 || N <= 0 || (p.cu && (B != 1 || p.pos)) ||
      !(theta > 0.) || !(theta < 1e300) || !(eps >= 0.f)) {
    gdn_internal_set_error("%s: bad arguments B=%lld T=%lld HQ=%lld HK=%lld N=%lld theta=%g eps=%g (cu_seqlens requires "
                           "B == 1 and no positions)", name, (long long)B, (long long)T, (long long)HQ, (long long)HK,
                           (long long)N, theta, (double)eps);
    return GDN_ERR_INVALID;
  }
  if ((D != 64 && D != 128 && D != 256) || rot_dim < 0 || rot_dim > D || rot_dim % 16) {
    gdn_internal_set_error("%s: D=%lld rot_dim=%d unsupported (D = 64, 128 or 256, rot_dim a multiple of 16 up to D)", name,
                           (long long)D, rot_dim);
    return GDN_ERR_UNSUPPORTED;
  }
  if (dtype < GDN_DTYPE_F32 || dtype > GDN_DTYPE_F16) {
    gdn_internal_set_error("%s: unknown dtype %d", name, dtype);
    return GDN_ERR_INVALID;
  }
  if (B * T > (1LL << 40)) {
    gdn_internal_set_error("%s: too many tokens (%lld)", name, (long long)(B * T));
    return GDN_ERR_UNSUPPORTED;
  }
  const int64_t unit = dtype == GDN_DTYPE_F32 ? 4 : 8;  // elements in 16 bytes
  uintptr_t all = 0;
  for (int m = 0; m < 2; ++m) {
    all |= reinterpret_cast<uintptr_t>(p.x[m]) | reinterpret_cast<uintptr_t>(p.dy[m]) | reinterpret_cast<uintptr_t>(p.y[m]);
    if (p.sb[m] % unit || p.st[m] % unit || p.sh[m] % unit) all |= 1;
  }
  if (all & 15) {
    gdn_internal_set_error("%s: rows must be 16-byte aligned", name);
    return GDN_ERR_INVALID;
  }
  p.T = T;
  p.N = N;
  p.tokens = B * T;
  p.heads[0] = (int)HQ;
  p.heads[1] = (int)HK;
  p.rot = rot_dim;
  p.eps = eps;
  p.wpt = p.tokens <= kRopeShared ? 4 : 1;
  for (int f = 0; f < rot_dim / 2; ++f) p.turns[f] = pow(theta, -2. * f / rot_dim) / 6.283185307179586;
  return GDN_OK;
}

template <bool BWD>
static void launch_rope(const QkRopeParams& p, int64_t D, int dtype, int64_t blocks, hipStream_t s) {
  auto go = [&](auto e, auto d) {
    hipLaunchKernelGGL((gated_delta_qk_norm_rope_kernel<decltype(d)::value, decltype(e), BWD>), dim3((unsigned)blocks),
                       dim3(256), 0, s, p);
  };
  auto by_dim = [&](auto e) {
    if (D == 64) go(e, std::integral_constant<int, 64>{});
    else if (D == 128) go(e, std::integral_constant<int, 128>{});
    else go(e, std::integral_constant<int, 256>{});
  };
  if (dtype == GDN_DTYPE_BF16) by_dim(bf16{});
  else if (dtype == GDN_DTYPE_F16) by_dim(f16{});
  else by_dim(float{});
}

static int64_t rope_blocks(int64_t tokens) { return tokens <= kRopeShared ? tokens : (tokens + 3) / 4; }
static int64_t rope_bwd_blocks(int64_t tokens) { return rope_blocks(tokens) < kRopeBwdBlocks ? rope_blocks(tokens) : kRopeBwdBlocks; }

}  // namespace gdn

using namespace gdn;

extern "C" int gdn_qk_norm_rope_fwd(const void* q, int64_t q_batch_stride, int64_t q_token_stride, int64_t q_head_stride,
                                    const void* k, int64_t k_batch_stride, int64_t k_token_stride, int64_t k_head_stride,
                                    const float* q_weight, const float* k_weight, const void* positions,
                                    int64_t pos_batch_stride, int64_t pos_token_stride, int pos_i32, void* q_out, void* k_out,
                                    const void* cu_seqlens, int64_t B, int64_t T, int64_t HQ, int64_t HK, int64_t D,
                                    int64_t N, int dtype, int rot_dim, double theta, float eps, unsigned flags,
                                    void* stream) {
  if (T > 0 && (!q || !k || !q_out || !k_out)) {
    gdn_internal_set_error("gdn_qk_norm_rope_fwd: null tensor pointer");
    return GDN_ERR_INVALID;
  }
  QkRopeParams p{{q, k}, {q_batch_stride, k_batch_stride}, {q_token_stride, k_token_stride}, {q_head_stride, k_head_stride},
                 {nullptr, nullptr}, {q_weight, k_weight}, {q_out, k_out}, nullptr, positions, pos_batch_stride,
                 pos_token_stride, cu_seqlens, pos_i32, (flags & GDN_FLAG_CU_INT32) ? 1 : 0};
  if (int rc = rope_check("gdn_qk_norm_rope_fwd", p, B, T, HQ, HK, D, N, dtype, rot_dim, theta, eps)) return rc;
  if (T == 0) return GDN_OK;
  const int64_t blocks = rope_blocks(p.tokens);
  launch_rope<false>(p, D, dtype, blocks < kMaxGroups256 ? blocks : kMaxGroups256, static_cast<hipStream_t>(stream));
  return gdn_internal_check_launch("gated_delta_qk_norm_rope_kernel");
}

extern "C" size_t gdn_qk_norm_rope_bwd_workspace_size(int64_t B, int64_t T, int64_t D) {
  if (B <= 0 || T < 0 || D <= 0) return 0;
  return (size_t)(rope_bwd_blocks(B * T) * 2 * D * 4);
}

extern "C" int gdn_qk_norm_rope_bwd(const void* q, int64_t q_batch_stride, int64_t q_token_stride, int64_t q_head_stride,
                                    const void* k, int64_t k_batch_stride, int64_t k_token_stride, int64_t k_head_stride,
                                    const float* q_weight, const float* k_weight, const void* positions,
                                    int64_t pos_batch_stride, int64_t pos_token_stride, int pos_i32, const void* dq_out,
                                    const void* dk_out, void* dq, void* dk, float* dq_weight, float* dk_weight,
                                    const void* cu_seqlens, int64_t B, int64_t T, int64_t HQ, int64_t HK, int64_t D,
                                    int64_t N, int dtype, int rot_dim, double theta, float eps, unsigned flags,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  if (T > 0 && (!q || !k || !dq_out || !dk_out || !dq || !dk)) {
    gdn_internal_set_error("gdn_qk_norm_rope_bwd: null tensor pointer");
    return GDN_ERR_INVALID;
  }
  const bool params = dq_weight || dk_weight;
  QkRopeParams p{{q, k}, {q_batch_stride, k_batch_stride}, {q_token_stride, k_token_stride}, {q_head_stride, k_head_stride},
                 {dq_out, dk_out}, {q_weight, k_weight}, {dq, dk}, params ? static_cast<float*>(workspace) : nullptr,
                 positions, pos_batch_stride, pos_token_stride, cu_seqlens, pos_i32, (flags & GDN_FLAG_CU_INT32) ? 1 : 0};
  if (int rc = rope_check("gdn_qk_norm_rope_bwd", p, B, T, HQ, HK, D, N, dtype, rot_dim, theta, eps)) return rc;
  const size_t need = gdn_qk_norm_rope_bwd_workspace_size(B, T, D);
  if (params && need && (!workspace || workspace_bytes < need)) {
    gdn_internal_set_error("gdn_qk_norm_rope_bwd: workspace of %zu bytes needed", need);
    return GDN_ERR_INVALID;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t blocks = rope_bwd_blocks(p.tokens);
  if (T > 0) {
    launch_rope<true>(p, D, dtype, blocks, s);
    if (int rc = gdn_internal_check_launch("gated_delta_qk_norm_rope_kernel(bwd)")) return rc;
  }
  if (params) {  // without tokens: zeros
    hipLaunchKernelGGL(gated_delta_qk_norm_rope_param_grad_kernel, dim3((unsigned)(2 * D / 16)), dim3(1024), 0, s, p.partial,
                       (int)blocks, (int)D, dq_weight, dk_weight);
    return gdn_internal_check_launch("gated_delta_qk_norm_rope_param_grad_kernel");
  }
  return GDN_OK;
}
