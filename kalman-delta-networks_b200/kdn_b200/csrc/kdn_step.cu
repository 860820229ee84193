// One new token per sequence through a whole KDN mixer between its
// projections: the single-token form of the short convolution, the q / k
// normalisation, the gate frontend, the covariance gain, the memory scan and
// the gated output norm (both variants), on a pool of per-sequence states
// updated in place.  Per sequence and head, with the raw projections x:
//   c = silu(sum_j w[c, j] x[t - 3 + j, c])  for q, k, v
//   q, k <- normalised;  ln alpha = -exp(A_log) softplus(f + dt_bias)
//   iso:  z = mean(alpha^2) p + omega, beta = z / (r + z),
//         p <- r z / (r + s z), kappa = beta k
//   diag: z = alpha^2 p + omega, kappa = z k / (r + sum z k^2),
//         p <- z / (1 + D k^2 / r z); alpha floored at 1e-6 in the memory
//   S^ = Diag(alpha) S,  u = S^T k,  w = S^T q  (one pass over the state)
//   delta = v - u,  S <- S^ + kappa delta^T,  o = D^-1/2 (w + (q.kappa) delta)
//   y = o / sqrt(mean(o^2) + eps) * weight * act(gate)
// All of it in fp32 (the conv outputs, q, k and o, which the training path
// rounds to bf16 between its kernels, stay in registers here).
//
// Bound by the state's bytes: 8 D^2 per sequence and head, read once and
// written once.  One CTA holds one head's state in registers (D = 128: 8
// float4 per thread): the state's loads are issued first and the token's
// small vectors (3D conv channels, D gates: one thread each) are prepared
// while they are in flight.
#include "kdn_common.cuh"

namespace kdn {
namespace {

struct StepParams {
  KdnStepArgs a;
};

__device__ __forceinline__ float softplus_f(float x) { return x > 20.f ? x : log1pf(expf(x)); }
__device__ __forceinline__ float sigmoid_f(float x) { return 1.f / (1.f + expf(-x)); }

template <class T>
__device__ __forceinline__ float ld1(const void* p, size_t i) {
  return to_f(static_cast<const T*>(p)[i]);
}

// D channels per head, 4 D threads: groups of D threads prepare q, k, v and
// the gates; for the state, D / 4 threads cover a row (float4 each) and 16
// row groups hold D / 16 consecutive rows each.
template <int D, bool DIAG, class T>
__global__ void __launch_bounds__(4 * D, 1024 / (4 * D)) step_kernel(const __grid_constant__ StepParams prm) {
  const KdnStepArgs& a = prm.a;
  constexpr int ROWS = D / 16, WG = D / 32, PARTS = D / 8;  // rows per thread, warps per group, warps in all
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t b = blockIdx.x / a.H;
  const int h = (int)(blockIdx.x - b * a.H);
  const int group = tid / D, d = tid - group * D;
  const size_t C = (size_t)a.H * D;  // channels of one section of qkv
  const size_t ch = (size_t)h * D + d;

  const int64_t slot = !a.slots ? b
                       : a.slots_i64 ? static_cast<const int64_t*>(a.slots)[b]
                                     : (int64_t) static_cast<const int32_t*>(a.slots)[b];
  T* y = static_cast<T*>(a.y) + (size_t)b * C + ch;
  if (slot < 0 || slot >= a.num_slots) {  // an idle row: no state, a zero output
    if (group == 0) *y = from_f<T>(0.f);
    return;
  }

  // the state, requested before anything else
  const int c4 = tid % (D / 4), rg = tid / (D / 4);
  float4* S = reinterpret_cast<float4*>(a.memory + ((size_t)slot * a.H + h) * (D * D)) + c4;
  float4 st[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) st[i] = S[(size_t)(rg * ROWS + i) * (D / 4)];

  __shared__ __align__(16) float part[2][PARTS][D];  // read and written as float4, like sdelta
  __shared__ __align__(16) float sdelta[D];
  __shared__ float sq[D], sk[D], sv[D], sal[D], skap[D], sact[D], sw[D];
  __shared__ float red[3][WG], sscal[4], sred[WG];

  // ---- the token's vectors ----
  float mine = 0.f, prior = 0.f, alpha = 0.f, r = 0.f;
  if (group < 3) {
    const size_t gc = (size_t)group * C + ch;
    T* win = static_cast<T*>(a.window) + (size_t)slot * 9 * C + gc;
    const T x3 = static_cast<const T*>(a.qkv)[(size_t)b * a.qkv_stride + gc];
    const T x1 = win[3 * C], x2 = win[6 * C];
    const float4 w = reinterpret_cast<const float4*>(a.conv_weight)[gc];
    float c = w.x * to_f(win[0]);
    c = fmaf(w.y, to_f(x1), c);
    c = fmaf(w.z, to_f(x2), c);
    c = fmaf(w.w, to_f(x3), c);
    win[0] = x1;
    win[3 * C] = x2;
    win[6 * C] = x3;
    mine = c * sigmoid_f(c);
  }
  // the decay: a group of its own (iso); the k threads (diag), which need it
  // beside k for sum z k^2
  if (group == (DIAG ? 1 : 3)) {
    const float f = ld1<T>(a.decay_raw, (size_t)b * a.decay_stride + ch) + a.dt_bias[ch];
    const float la = -expf(a.A_log[h]) * softplus_f(f);
    alpha = expf(la);
  }
  if (DIAG) {
    if (group == 1) {
      float* pc = a.covariance + (size_t)slot * C + ch;
      const float omega = a.omega_min + softplus_f(ld1<T>(a.omega_raw, (size_t)b * a.omega_stride + ch));
      r = a.r_min + softplus_f(ld1<T>(a.r_raw, (size_t)b * a.r_stride + h));
      prior = fmaf(alpha * alpha, *pc, omega);
      sal[d] = fmaxf(alpha, 1e-6f);
    }
    if (group == 3) {
      const float g = ld1<T>(a.gate, (size_t)b * a.gate_stride + ch), s = sigmoid_f(g);
      sact[d] = (a.swish ? g * s : s) * (a.norm_weight ? a.norm_weight[d] : 1.f);
    }
  } else {
    if (group == 3) sal[d] = alpha;
    if (group == 2) {
      const float g = ld1<T>(a.gate, (size_t)b * a.gate_stride + ch), s = sigmoid_f(g);
      sact[d] = (a.swish ? g * s : s) * (a.norm_weight ? a.norm_weight[d] : 1.f);
    }
    if (tid == 3 * D) {
      sscal[0] = a.omega_min + softplus_f(ld1<T>(a.omega_raw, (size_t)b * a.omega_stride + h) + a.omega_bias[h]);
      sscal[1] = a.r_min + softplus_f(ld1<T>(a.r_raw, (size_t)b * a.r_stride + h) + a.r_bias[h]);
      sscal[2] = a.covariance[(size_t)slot * a.H + h];
    }
  }
  if (group == 0) sq[d] = mine;
  if (group == 1) sk[d] = mine;
  if (group == 2) sv[d] = mine;
  {
    // row sums: q^2, k^2 and alpha^2 (iso) or z k^2 (diag, by the k threads)
    float s = group == 3 ? alpha * alpha : mine * mine;
    s = warp_sum(s);
    if (lane == 0 && (group < 2 || (!DIAG && group == 3))) red[group == 3 ? 2 : group][warp % WG] = s;
    if (DIAG && group == 1) {
      const float zk = warp_sum(prior * mine * mine);
      if (lane == 0) red[2][warp % WG] = zk;
    }
  }
  __syncthreads();

  float ssq = 0.f, ssk = 0.f, third = 0.f;
#pragma unroll
  for (int i = 0; i < WG; ++i) {
    ssq += red[0][i];
    ssk += red[1][i];
    third += red[2][i];
  }
  float rq, rk;
  if (DIAG) {  // the diagonal boundary's norm: x / max(|x|, 1e-12)
    rq = 1.f / fmaxf(sqrtf(ssq), 1e-12f);
    rk = 1.f / fmaxf(sqrtf(ssk), 1e-12f);
    if (group == 1) {
      const float kn = mine * rk;
      skap[d] = prior * kn / (r + third * rk * rk);
      a.covariance[(size_t)slot * C + ch] = prior / (1.f + (float)D * kn * kn / r * prior);
    }
  } else {  // x / sqrt(|x|^2 + 1e-6)
    rq = rsqrtf(ssq + 1e-6f);
    rk = rsqrtf(ssk + 1e-6f);
    const float om = sscal[0], rr = sscal[1];
    const float z = fmaf(third * (1.f / (float)D), sscal[2], om);
    if (group == 1) skap[d] = z / (rr + z) * (mine * rk);
    if (tid == 0) a.covariance[(size_t)slot * a.H + h] = rr * z / fmaf(a.posterior_scale, z, rr);
  }

  // ---- one pass over the state: S^ = alpha S, u = S^T k, w = S^T q ----
  float4 u = make_float4(0.f, 0.f, 0.f, 0.f), w = u;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = rg * ROWS + i;
    const float al = sal[row], kk = sk[row], qq = sq[row];
    st[i].x *= al; st[i].y *= al; st[i].z *= al; st[i].w *= al;
    u.x = fmaf(kk, st[i].x, u.x); u.y = fmaf(kk, st[i].y, u.y);
    u.z = fmaf(kk, st[i].z, u.z); u.w = fmaf(kk, st[i].w, u.w);
    w.x = fmaf(qq, st[i].x, w.x); w.y = fmaf(qq, st[i].y, w.y);
    w.z = fmaf(qq, st[i].z, w.z); w.w = fmaf(qq, st[i].w, w.w);
  }
  if (D == 64) {  // a warp holds two row groups
    u.x += __shfl_xor_sync(0xffffffffu, u.x, 16); u.y += __shfl_xor_sync(0xffffffffu, u.y, 16);
    u.z += __shfl_xor_sync(0xffffffffu, u.z, 16); u.w += __shfl_xor_sync(0xffffffffu, u.w, 16);
    w.x += __shfl_xor_sync(0xffffffffu, w.x, 16); w.y += __shfl_xor_sync(0xffffffffu, w.y, 16);
    w.z += __shfl_xor_sync(0xffffffffu, w.z, 16); w.w += __shfl_xor_sync(0xffffffffu, w.w, 16);
  }
  if (lane < D / 4) {
    reinterpret_cast<float4*>(part[0][warp])[c4] = u;
    reinterpret_cast<float4*>(part[1][warp])[c4] = w;
  }
  __syncthreads();
  if (group < 2) {  // D threads finish u and delta, D threads w
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) s += part[group][i][d];
    if (group == 1)
      sw[d] = s * rq;
    else
      sdelta[d] = sv[d] - s * rk;
  }
  // q . kappa, by one warp that has no column to sum
  if (warp == 2 * WG) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < WG; ++i) s = fmaf(sq[lane + 32 * i], skap[lane + 32 * i], s);
    s = warp_sum(s);
    if (lane == 0) sscal[3] = s * rq;
  }
  __syncthreads();
  const float4 dl = reinterpret_cast<const float4*>(sdelta)[c4];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const float ka = skap[rg * ROWS + i];
    st[i].x = fmaf(ka, dl.x, st[i].x); st[i].y = fmaf(ka, dl.y, st[i].y);
    st[i].z = fmaf(ka, dl.z, st[i].z); st[i].w = fmaf(ka, dl.w, st[i].w);
    S[(size_t)(rg * ROWS + i) * (D / 4)] = st[i];
  }
  if (group == 0) {
    const float o = a.scale * fmaf(sscal[3], sdelta[d], sw[d]);
    const float s = warp_sum(o * o);
    if (lane == 0) sred[warp] = s;
    bar_sync(1, D);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < WG; ++i) ss += sred[i];
    *y = from_f<T>(o * rsqrtf(ss * (1.f / (float)D) + a.eps) * sact[d]);
  }
}

template <int D, class T>
void launch_step(const StepParams& p, unsigned grid, cudaStream_t st) {
  if (p.a.variant == KDN_DIAG)
    step_kernel<D, true, T><<<grid, 4 * D, 0, st>>>(p);
  else
    step_kernel<D, false, T><<<grid, 4 * D, 0, st>>>(p);
}

}  // namespace
}  // namespace kdn

using namespace kdn;

extern "C" int kdn_step(const KdnStepArgs* args, kdn_stream_t stream) {
  if (!args) return set_error(KDN_ERR_INVALID, "kdn_step: null args");
  const KdnStepArgs& a = *args;
  if (a.variant != KDN_ISO && a.variant != KDN_DIAG)
    return set_error(KDN_ERR_INVALID, "kdn_step: variant must be KDN_ISO or KDN_DIAG");
  if (a.B < 0 || a.H < 1 || a.num_slots < 0 || (a.D != 64 && a.D != 128))
    return set_error(KDN_ERR_INVALID, "kdn_step: B >= 0, H >= 1, num_slots >= 0 and D in {64, 128} required");
  if (a.H > (1 << 20) || a.B > (int64_t)INT32_MAX / a.H)
    return set_error(KDN_ERR_INVALID, "kdn_step: size too large");
  const int64_t HD = a.H * a.D;
  const bool diag = a.variant == KDN_DIAG;
  auto bad = [](int64_t stride, int64_t width) { return stride < width && stride != 0; };  // 0: one row for all
  if (a.B > 1 && (bad(a.qkv_stride, 3 * HD) || bad(a.decay_stride, HD) || bad(a.gate_stride, HD) ||
                  bad(a.omega_stride, diag ? HD : a.H) || bad(a.r_stride, a.H)))
    return set_error(KDN_ERR_INVALID, "kdn_step: row strides smaller than the rows");
  if (a.B == 0) return KDN_OK;
  if (!a.qkv || !a.decay_raw || !a.omega_raw || !a.r_raw || !a.gate || !a.conv_weight || !a.A_log || !a.dt_bias ||
      !a.y || (!diag && (!a.omega_bias || !a.r_bias)))
    return set_error(KDN_ERR_INVALID, "kdn_step: null pointer");
  if (a.num_slots > 0 && (!a.memory || !a.covariance || !a.window))
    return set_error(KDN_ERR_INVALID, "kdn_step: null state pointer");
  if (!a.slots && a.num_slots < a.B)
    return set_error(KDN_ERR_INVALID, "kdn_step: without slots the pool must hold a state per row");
  if ((reinterpret_cast<uintptr_t>(a.memory) | reinterpret_cast<uintptr_t>(a.conv_weight)) & 15)
    return set_error(KDN_ERR_INVALID, "kdn_step: memory and conv_weight must be 16-byte aligned");
  StepParams p{a};
  const unsigned grid = (unsigned)(a.B * a.H);
  cudaStream_t st = (cudaStream_t)stream;
  if (a.D == 128) {
    if (a.act_bf16) launch_step<128, bf16>(p, grid, st);
    else launch_step<128, float>(p, grid, st);
  } else {
    if (a.act_bf16) launch_step<64, bf16>(p, grid, st);
    else launch_step<64, float>(p, grid, st);
  }
  return check_launch("step_kernel");
}
