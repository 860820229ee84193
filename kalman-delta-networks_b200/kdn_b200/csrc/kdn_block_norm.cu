// The norms around a block: u = act(g) scale norm(y) post_weight,
// z = alpha x + u, h = norm(z) weight, with norm(t) = t / sqrt(mean(t^2) + eps)
// per row of D values, and its gradients.  With s = act(g), yh = y ry,
// zh = z rz (ry, rz the reciprocal roots, saved by the forward):
//   Z  = dz + rz (w dh - zh mean(w dh zh))         total cotangent of z
//   dx = alpha Z,  du = Z,  dw = sum over rows of dh zh
//   dscale = sum Z s yh post,  dpost = sum Z s scale yh
//   dg = Z scale yh post act'(g)
//   dy = ry (t - yh mean(t yh)),  t = Z s scale post   (t itself without the norm)
// z is formed again from x, y and g in the backward rather than read back
// from its rounded copy, so the gradients are those of the unrounded sum.
//
// Bound by the bytes of its tensors.  A group of threads owns a row (8
// consecutive values per thread and slot), several rows are walked per group
// so that each thread keeps its columns' weights and weight-gradient sums in
// registers; the groups' sums are added in a fixed order by a second kernel.
#include "kdn_common.cuh"

namespace kdn {
namespace {

constexpr int kBnVec = 8;      // values per thread and slot
constexpr int kBnMaxD = 16384;
constexpr int kBnMaxRowGroups = 148 * 8;  // row groups of a launch at most

struct BnGeom {
  int slots;    // slots per thread (1 or 2)
  int tpr;      // threads per row
  int rpb;      // rows per CTA
  unsigned grid;
};

inline BnGeom bn_geom(int64_t rows, int64_t D) {
  BnGeom g;
  const int nv = (int)((D + kBnVec - 1) / kBnVec);
  g.slots = nv > 1024 ? 2 : 1;
  g.tpr = ((nv + g.slots - 1) / g.slots + 31) / 32 * 32;
  g.rpb = g.tpr >= 256 ? 1 : 256 / g.tpr;
  const int64_t want = (rows + g.rpb - 1) / g.rpb, most = kBnMaxRowGroups / g.rpb;
  g.grid = (unsigned)(want < most ? (want > 0 ? want : 1) : most);
  return g;
}

struct BnParams {
  KdnBlockNormArgs a;
  float* partial;  // [row groups][3][D]
  int tpr;
};

__device__ __forceinline__ float sigmoid_f(float x) { return 1.f / (1.f + expf(-x)); }

// n (<= 8) consecutive values; vec: 16-byte aligned and n == 8
template <class T>
__device__ __forceinline__ void ldn(float (&d)[8], const T* p, int n, bool vec) {
  if (vec) {
    ld8(d, p);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = i < n ? to_f(p[i]) : 0.f;
  }
}
template <class T>
__device__ __forceinline__ void stn(T* p, const float (&s)[8], int n, bool vec) {
  if (vec) {
    st8(p, s);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = from_f<T>(s[i]);
  }
}
__device__ __forceinline__ void ldw(float (&d)[8], const void* p, int col, int n, bool bf) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    d[i] = !p ? 1.f : i >= n ? 0.f : bf ? to_f(static_cast<const bf16*>(p)[col + i]) : static_cast<const float*>(p)[col + i];
}

__device__ __forceinline__ bool aligned16(const void* p, int64_t stride, size_t elem) {
  return ((reinterpret_cast<uintptr_t>(p) | ((size_t)stride * elem)) & 15) == 0;
}

// Sums of N values over the threads of a row group (tpr threads, its own
// named barrier); `red` alternates between two buffers from call to call, so
// one barrier per call is enough.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* red /* [2][32][N] of this group */, int& phase,
                                          int tpr, int group) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if (tpr == 32) return;
  const int t = threadIdx.x - group * tpr, warp = t >> 5;
  float* r = red + phase * 32 * N;
  phase ^= 1;
  if ((t & 31) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) r[warp * N + i] = v[i];
  bar_sync(1 + group, tpr);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float s = 0.f;
    for (int w = 0; w < tpr / 32; ++w) s += r[w * N + i];
    v[i] = s;
  }
}

template <class TX, class TY, int SLOTS>
__global__ void __launch_bounds__(1024) block_norm_fwd_kernel(const __grid_constant__ BnParams prm) {
  const KdnBlockNormArgs& a = prm.a;
  __shared__ float red_all[8][2 * 32];
  const int tpr = prm.tpr, group = threadIdx.x / tpr, t = threadIdx.x - group * tpr, rpb = blockDim.x / tpr;
  const int D = (int)a.D;
  const bool wb = a.weights_bf16 != 0;
  const bool vx = aligned16(a.x, a.x_stride, sizeof(TX)), vy = a.y && aligned16(a.y, a.y_stride, sizeof(TY)),
             vg = a.gate && aligned16(a.gate, a.gate_stride, sizeof(TY)), vz = a.z && aligned16(a.z, D, sizeof(TX)),
             vh = aligned16(a.h, D, sizeof(TY));
  int phase = 0;
  float pw[SLOTS][8], w[SLOTS][8];  // scale * post_weight, weight
  int col[SLOTS], n[SLOTS];
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    col[s] = (t + s * tpr) * kBnVec;
    n[s] = min(max(D - col[s], 0), kBnVec);
    float sc[8];
    ldw(sc, a.scale, col[s], n[s], wb);
    ldw(pw[s], a.post_weight, col[s], n[s], wb);
    ldw(w[s], a.weight, col[s], n[s], wb);
#pragma unroll
    for (int i = 0; i < 8; ++i) pw[s][i] *= sc[i];
  }
  for (int64_t row = (int64_t)blockIdx.x * rpb + group; row < a.rows; row += (int64_t)gridDim.x * rpb) {
    float x[SLOTS][8], y[SLOTS][8], g[SLOTS][8];
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const bool full = n[s] == kBnVec;
      ldn(x[s], static_cast<const TX*>(a.x) + row * a.x_stride + col[s], n[s], vx && full);
      if (a.y) ldn(y[s], static_cast<const TY*>(a.y) + row * a.y_stride + col[s], n[s], vy && full);
      if (a.gate) ldn(g[s], static_cast<const TY*>(a.gate) + row * a.gate_stride + col[s], n[s], vg && full);
    }
    float sum[1] = {0.f};
    float ry = 1.f;
    if (a.post_weight) {
#pragma unroll
      for (int s = 0; s < SLOTS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[0] = fmaf(y[s][i], y[s][i], sum[0]);
      group_sum<1>(sum, red_all[group], phase, tpr, group);
      ry = rsqrtf(sum[0] / (float)D + a.eps);
    }
    sum[0] = 0.f;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (a.y) {
          float u = y[s][i] * ry * pw[s][i];
          if (a.gate) {
            const float sg = sigmoid_f(g[s][i]);
            u *= a.swish ? g[s][i] * sg : sg;
          }
          x[s][i] = fmaf(a.alpha, x[s][i], u);
        }
        sum[0] = fmaf(x[s][i], x[s][i], sum[0]);
      }
    group_sum<1>(sum, red_all[group], phase, tpr, group);
    const float rz = rsqrtf(sum[0] / (float)D + a.eps);
    if (a.rstd && t == 0) {
      a.rstd[row] = ry;
      a.rstd[a.rows + row] = rz;
    }
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const bool full = n[s] == kBnVec;
      if (a.y) stn(static_cast<TX*>(a.z) + row * D + col[s], x[s], n[s], vz && full);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[s][i] *= rz * w[s][i];
      stn(static_cast<TY*>(a.h) + row * D + col[s], x[s], n[s], vh && full);
    }
  }
}

template <class TX, class TY, int SLOTS>
__global__ void __launch_bounds__(1024) block_norm_bwd_kernel(const __grid_constant__ BnParams prm) {
  const KdnBlockNormArgs& a = prm.a;
  __shared__ float red_all[8][2 * 32];
  const int tpr = prm.tpr, group = threadIdx.x / tpr, t = threadIdx.x - group * tpr, rpb = blockDim.x / tpr;
  const int D = (int)a.D;
  const float inv_D = 1.f / (float)D;
  const bool wb = a.weights_bf16 != 0;
  const bool vx = aligned16(a.x, a.x_stride, sizeof(TX)), vy = a.y && aligned16(a.y, a.y_stride, sizeof(TY)),
             vg = a.gate && aligned16(a.gate, a.gate_stride, sizeof(TY)), vdz = a.dz && aligned16(a.dz, D, sizeof(TX)),
             vdh = a.dh && aligned16(a.dh, D, sizeof(TY)), vdx = aligned16(a.dx, D, sizeof(TX)),
             vdy = aligned16(a.dy, D, sizeof(TY)), vdg = aligned16(a.dgate, D, sizeof(TY));
  int phase = 0;
  float dw[SLOTS][8], dp[SLOTS][8], ds[SLOTS][8];
  int col[SLOTS], n[SLOTS];
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    col[s] = (t + s * tpr) * kBnVec;
    n[s] = min(max(D - col[s], 0), kBnVec);
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[s][i] = dp[s][i] = ds[s][i] = 0.f;
  }
  for (int64_t row = (int64_t)blockIdx.x * rpb + group; row < a.rows; row += (int64_t)gridDim.x * rpb) {
    const float ry = a.rstd[row], rz = a.rstd[a.rows + row];
    float z[SLOTS][8], dz[SLOTS][8], dh[SLOTS][8];
    float sum[1] = {0.f};
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const bool full = n[s] == kBnVec;
      float sc[8], pw[8], w[8], y[8], g[8];
      ldn(z[s], static_cast<const TX*>(a.x) + row * a.x_stride + col[s], n[s], vx && full);
      if (a.dz)
        ldn(dz[s], static_cast<const TX*>(a.dz) + row * D + col[s], n[s], vdz && full);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) dz[s][i] = 0.f;
      if (a.dh)
        ldn(dh[s], static_cast<const TY*>(a.dh) + row * D + col[s], n[s], vdh && full);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) dh[s][i] = 0.f;
      if (a.y) {
        ldn(y, static_cast<const TY*>(a.y) + row * a.y_stride + col[s], n[s], vy && full);
        if (a.gate) ldn(g, static_cast<const TY*>(a.gate) + row * a.gate_stride + col[s], n[s], vg && full);
        ldw(sc, a.scale, col[s], n[s], wb);
        ldw(pw, a.post_weight, col[s], n[s], wb);
      }
      ldw(w, a.weight, col[s], n[s], wb);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (a.y) {
          float u = y[i] * ry * pw[i] * sc[i];
          if (a.gate) {
            const float sg = sigmoid_f(g[i]);
            u *= a.swish ? g[i] * sg : sg;
          }
          z[s][i] = fmaf(a.alpha, z[s][i], u);
        }
        z[s][i] *= rz;
        dw[s][i] = fmaf(dh[s][i], z[s][i], dw[s][i]);
        dh[s][i] *= w[i];
        sum[0] = fmaf(dh[s][i], z[s][i], sum[0]);
      }
    }
    group_sum<1>(sum, red_all[group], phase, tpr, group);
    const float c1 = sum[0] * inv_D;
    sum[0] = 0.f;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const bool full = n[s] == kBnVec;
#pragma unroll
      for (int i = 0; i < 8; ++i) dz[s][i] = fmaf(rz, dh[s][i] - z[s][i] * c1, dz[s][i]);
      if (a.dx) {
        float dx[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) dx[i] = a.alpha * dz[s][i];
        stn(static_cast<TX*>(a.dx) + row * D + col[s], dx, n[s], vdx && full);
      }
      if (!a.y) continue;
      float sc[8], pw[8], y[8], g[8], dg[8];
      ldn(y, static_cast<const TY*>(a.y) + row * a.y_stride + col[s], n[s], vy && full);
      if (a.gate) ldn(g, static_cast<const TY*>(a.gate) + row * a.gate_stride + col[s], n[s], vg && full);
      ldw(sc, a.scale, col[s], n[s], wb);
      ldw(pw, a.post_weight, col[s], n[s], wb);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float yh = y[i] * ry;
        float act = 1.f, slope = 0.f;
        if (a.gate) {
          const float sg = sigmoid_f(g[i]);
          act = a.swish ? g[i] * sg : sg;
          slope = a.swish ? sg * (1.f + g[i] * (1.f - sg)) : sg * (1.f - sg);
        }
        const float Z = dz[s][i];
        dg[i] = Z * sc[i] * yh * pw[i] * slope;
        ds[s][i] = fmaf(Z * act, yh * pw[i], ds[s][i]);
        dp[s][i] = fmaf(Z * act, sc[i] * yh, dp[s][i]);
        const float tt = Z * act * sc[i] * pw[i];
        dz[s][i] = tt;  // the cotangent of yh from here on
        z[s][i] = yh;
        sum[0] = fmaf(tt, yh, sum[0]);
      }
      if (a.dgate) stn(static_cast<TY*>(a.dgate) + row * D + col[s], dg, n[s], vdg && full);
    }
    if (!a.y) continue;
    float c2 = 0.f;
    if (a.post_weight) {
      group_sum<1>(sum, red_all[group], phase, tpr, group);
      c2 = sum[0] * inv_D;
    }
    if (a.dy)
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {
        float dy[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) dy[i] = ry * (dz[s][i] - z[s][i] * c2);
        stn(static_cast<TY*>(a.dy) + row * D + col[s], dy, n[s], vdy && n[s] == kBnVec);
      }
  }
  if (prm.partial) {
    float* p = prm.partial + (size_t)(blockIdx.x * rpb + group) * 3 * D;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n[s]) {
          p[col[s] + i] = dw[s][i];
          p[D + col[s] + i] = dp[s][i];
          p[2 * D + col[s] + i] = ds[s][i];
        }
  }
}

// Weight gradients: column sums of the groups' partial rows in a fixed order
// (32 columns x 8 chains per CTA).
__global__ void block_norm_weights_kernel(const __grid_constant__ BnParams prm, int groups) {
  const KdnBlockNormArgs& a = prm.a;
  __shared__ float red[8][33];
  void* out = blockIdx.y == 0 ? a.dweight : blockIdx.y == 1 ? a.dpost : a.dscale;
  if (!out) return;
  const int D = (int)a.D, lane = threadIdx.x & 31, chain = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (col < D)
    for (int p = chain; p < groups; p += 8) s += prm.partial[((size_t)p * 3 + blockIdx.y) * D + col];
  red[chain][lane] = s;
  __syncthreads();
  if (chain == 0 && col < D) {
#pragma unroll
    for (int c = 1; c < 8; ++c) s += red[c][lane];
    if (a.weights_bf16)
      static_cast<bf16*>(out)[col] = from_f<bf16>(s);
    else
      static_cast<float*>(out)[col] = s;
  }
}

template <class TX, class TY>
void bn_launch(const BnParams& p, const BnGeom& g, bool bwd, cudaStream_t st) {
  const unsigned threads = (unsigned)(g.tpr * g.rpb);
  if (bwd) {
    if (g.slots == 1) block_norm_bwd_kernel<TX, TY, 1><<<g.grid, threads, 0, st>>>(p);
    else block_norm_bwd_kernel<TX, TY, 2><<<g.grid, threads, 0, st>>>(p);
  } else {
    if (g.slots == 1) block_norm_fwd_kernel<TX, TY, 1><<<g.grid, threads, 0, st>>>(p);
    else block_norm_fwd_kernel<TX, TY, 2><<<g.grid, threads, 0, st>>>(p);
  }
}

void bn_dispatch(const BnParams& p, const BnGeom& g, bool bwd, cudaStream_t st) {
  if (p.a.act_bf16 && p.a.stream_bf16) bn_launch<bf16, bf16>(p, g, bwd, st);
  else if (p.a.act_bf16) bn_launch<float, bf16>(p, g, bwd, st);
  else bn_launch<float, float>(p, g, bwd, st);
}

int bn_check(const char* what, const KdnBlockNormArgs* p) {
  if (!p) return set_error(KDN_ERR_INVALID, "%s: null args", what);
  const KdnBlockNormArgs& a = *p;
  if (a.rows < 0 || a.D < 1 || a.D > kBnMaxD)
    return set_error(KDN_ERR_INVALID, "%s: rows >= 0 and D in [1, %d] required", what, kBnMaxD);
  if (a.stream_bf16 && !a.act_bf16)
    return set_error(KDN_ERR_INVALID, "%s: fp32 activations need an fp32 residual stream", what);
  if (a.rows == 0) return KDN_OK;
  if (!a.x || !a.weight) return set_error(KDN_ERR_INVALID, "%s: null pointer", what);
  if (!a.y && (a.gate || a.post_weight || a.scale || a.alpha != 1.f))
    return set_error(KDN_ERR_INVALID, "%s: gate, post_weight, scale and alpha need a block output y", what);
  if (a.rows > 1 && (a.x_stride < a.D || (a.y && a.y_stride < a.D) || (a.gate && a.gate_stride < a.D)))
    return set_error(KDN_ERR_INVALID, "%s: row strides smaller than the rows", what);
  return KDN_OK;
}

}  // namespace
}  // namespace kdn

using namespace kdn;

extern "C" {

size_t kdn_block_norm_workspace_bytes(int64_t rows, int64_t D) {
  if (rows <= 0 || D < 1 || D > kBnMaxD) return 0;
  const BnGeom g = bn_geom(rows, D);
  return align_up(sizeof(float) * 3 * (size_t)D * g.grid * g.rpb, 256);
}

int kdn_block_norm_fwd(const KdnBlockNormArgs* args, kdn_stream_t stream) {
  if (int rc = bn_check("kdn_block_norm_fwd", args)) return rc;
  const KdnBlockNormArgs& a = *args;
  if (a.rows == 0) return KDN_OK;
  if (!a.h || (a.y && !a.z)) return set_error(KDN_ERR_INVALID, "kdn_block_norm_fwd: null output");
  const BnGeom g = bn_geom(a.rows, a.D);
  bn_dispatch(BnParams{a, nullptr, g.tpr}, g, false, (cudaStream_t)stream);
  return check_launch("block_norm_fwd_kernel");
}

int kdn_block_norm_bwd(const KdnBlockNormArgs* args, kdn_stream_t stream) {
  if (int rc = bn_check("kdn_block_norm_bwd", args)) return rc;
  const KdnBlockNormArgs& a = *args;
  const bool weights = a.dweight || a.dpost || a.dscale;
  cudaStream_t st = (cudaStream_t)stream;
  if (a.rows == 0) {
    const size_t bytes = (size_t)a.D * (a.weights_bf16 ? 2 : 4);
    for (void* p : {a.dweight, a.dpost, a.dscale})
      if (p && cudaMemsetAsync(p, 0, bytes, st) != cudaSuccess) return check_launch("kdn_block_norm_bwd: memset");
    return KDN_OK;
  }
  if (!a.rstd) return set_error(KDN_ERR_INVALID, "kdn_block_norm_bwd: the forward's rstd is required");
  if ((a.dpost && !a.post_weight) || (a.dscale && !a.scale) || (a.dgate && !a.gate) || (a.dy && !a.y))
    return set_error(KDN_ERR_INVALID, "kdn_block_norm_bwd: a gradient of an absent input");
  if (weights && (!a.workspace || a.workspace_bytes < kdn_block_norm_workspace_bytes(a.rows, a.D)))
    return set_error(KDN_ERR_WORKSPACE, "kdn_block_norm_bwd: workspace too small");
  const BnGeom g = bn_geom(a.rows, a.D);
  const BnParams p{a, weights ? static_cast<float*>(a.workspace) : nullptr, g.tpr};
  bn_dispatch(p, g, true, st);
  if (int rc = check_launch("block_norm_bwd_kernel")) return rc;
  if (!weights) return KDN_OK;
  block_norm_weights_kernel<<<dim3((unsigned)((a.D + 31) / 32), 3), 256, 0, st>>>(p, (int)(g.grid * g.rpb));
  return check_launch("block_norm_weights_kernel");
}

}  // extern "C"
