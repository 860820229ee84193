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
// written once.  One CTA takes one head's state.  Its copy into shared memory
// is requested first (cp.async; every thread reads only what it copied), and
// the token's small vectors (3 D conv channels, D gates: one thread each) are
// prepared meanwhile.  Three CTAs share an SM (D = 128: 75 KB and 512 threads
// each), so that one loads while the others compute and store: 106 us for 256
// sequences of 18 x 128 (5.95 TB/s, 0.91 of the copy rate; 111 us diagonal),
// 146 us with the state in registers and two CTAs.  Few sequences are bound by
// one CTA's latency: 6.4 us for one.
#include "kdn_launch.cuh"

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
template <int D>
struct StepShared {
  float4 state[D * D / 4];        // [row in its group][thread]
  float part[2][D / 16][D];       // sums of S^T k, S^T q; their totals end in row 0
  float q[D], k[D], alpha[D], kappa[D];
  float red[3][D / 32], out[D / 32], scalar[4];
};

template <int D, bool DIAG, class T>
__global__ void __launch_bounds__(4 * D, D == 128 ? 3 : 6) step_kernel(const __grid_constant__ StepParams prm) {
  const KdnStepArgs& a = prm.a;
  constexpr int ROWS = D / 16, WG = D / 32, HALF = D / 16;  // rows per thread, warps per group, half of the warps
  extern __shared__ __align__(16) unsigned char raw[];
  StepShared<D>& sh = *reinterpret_cast<StepShared<D>*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t b = blockIdx.x / (unsigned)a.H;
  const int h = (int)(blockIdx.x % (unsigned)a.H);
  const int group = tid / D, d = tid - group * D;
  const size_t C = (size_t)a.H * D;  // channels of one section of qkv
  const size_t ch = (size_t)h * D + d;

  const int64_t slot = !a.slots ? b
                       : a.slots_i64 ? static_cast<const int64_t*>(a.slots)[b]
                                     : (int64_t) static_cast<const int32_t*>(a.slots)[b];
  T* y = static_cast<T*>(a.y) + (size_t)b * C + ch;
  if (slot < 0 || slot >= a.num_slots) {  // an idle row: no state, a zero output
    if (group == 2) *y = from_f<T>(0.f);
    return;
  }

  // the state, requested before anything else
  const int c4 = tid % (D / 4), rg = tid / (D / 4);
  float4* S = reinterpret_cast<float4*>(a.memory + ((size_t)slot * a.H + h) * (D * D)) + rg * ROWS * (D / 4) + c4;
  float4* held = sh.state + tid;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) cp_async16(held + i * 4 * D, S + i * (D / 4));
  cp_async_commit();

  // ---- the token's vectors ----
  float mine = 0.f, prior = 0.f, alpha = 0.f, r = 0.f, act = 0.f;
  float gate = 0.f, weight = 1.f;
  if (group == 2) {  // the v threads finish the output: its gate and norm weight stay with them
    gate = ld1<T>(a.gate, (size_t)b * a.gate_stride + ch);
    if (a.norm_weight) weight = a.norm_weight[d];
  }
  float decay = 0.f, bias = 0.f, log_rate = 0.f, omega = 0.f, noise = 0.f, old = 0.f;
  if (group == 3) {  // the gates have a group of their own, and with them the diagonal covariance
    decay = ld1<T>(a.decay_raw, (size_t)b * a.decay_stride + ch);
    bias = a.dt_bias[ch];
    log_rate = a.A_log[h];
    if (DIAG) {
      omega = ld1<T>(a.omega_raw, (size_t)b * a.omega_stride + ch);
      noise = ld1<T>(a.r_raw, (size_t)b * a.r_stride + h);
      old = a.covariance[(size_t)slot * C + ch];
    }
  }
  if (group < 3) {
    const size_t gc = (size_t)group * C + ch;
    T* win = static_cast<T*>(a.window) + (size_t)slot * 9 * C + gc;
    const T x3 = static_cast<const T*>(a.qkv)[(size_t)b * a.qkv_stride + gc];
    const T x0 = win[0], x1 = win[3 * C], x2 = win[6 * C];
    const float4 w = reinterpret_cast<const float4*>(a.conv_weight)[gc];
    float c = w.x * to_f(x0);
    c = fmaf(w.y, to_f(x1), c);
    c = fmaf(w.z, to_f(x2), c);
    c = fmaf(w.w, to_f(x3), c);
    win[0] = x1;
    win[3 * C] = x2;
    win[6 * C] = x3;
    mine = c * sigmoid_f(c);
  }
  if (group == 3) alpha = expf(-expf(log_rate) * softplus_f(decay + bias));
  if (group == 3) sh.alpha[d] = DIAG ? fmaxf(alpha, 1e-6f) : alpha;
  if (DIAG) {
    if (group == 3) {
      r = a.r_min + softplus_f(noise);
      prior = fmaf(alpha * alpha, old, a.omega_min + softplus_f(omega));
    }
  } else {
    if (tid == 3 * D) {
      sh.scalar[0] = a.omega_min + softplus_f(ld1<T>(a.omega_raw, (size_t)b * a.omega_stride + h) + a.omega_bias[h]);
      sh.scalar[1] = a.r_min + softplus_f(ld1<T>(a.r_raw, (size_t)b * a.r_stride + h) + a.r_bias[h]);
      sh.scalar[2] = a.covariance[(size_t)slot * a.H + h];
    }
  }
  if (group == 0) sh.q[d] = mine;
  if (group == 1) sh.k[d] = mine;
  if (group == 2) {
    const float s = sigmoid_f(gate);
    act = (a.swish ? gate * s : s) * weight;
  }
  {
    // row sums: q^2, k^2 and (iso) alpha^2
    const float s = warp_sum(group == 3 ? alpha * alpha : mine * mine);
    if (lane == 0 && (group < 2 || (!DIAG && group == 3))) sh.red[group == 3 ? 2 : group][warp % WG] = s;
  }
  __syncthreads();

  float ssq = 0.f, ssk = 0.f, third = 0.f;
#pragma unroll
  for (int i = 0; i < WG; ++i) {
    ssq += sh.red[0][i];
    ssk += sh.red[1][i];
    if (!DIAG) third += sh.red[2][i];
  }
  float rq, rk, kn = 0.f;
  if (DIAG) {  // the diagonal boundary's norm: x / max(|x|, 1e-12)
    rq = 1.f / fmaxf(sqrtf(ssq), 1e-12f);
    rk = 1.f / fmaxf(sqrtf(ssk), 1e-12f);
    if (group == 3) {  // sum z k^2: published by the next barrier, the gain by the one after it
      kn = sh.k[d] * rk;
      const float zk = warp_sum(prior * kn * kn);
      if (lane == 0) sh.red[2][warp % WG] = zk;
    }
  } else {  // x / sqrt(|x|^2 + 1e-6)
    rq = rsqrtf(ssq + 1e-6f);
    rk = rsqrtf(ssk + 1e-6f);
    const float om = sh.scalar[0], rr = sh.scalar[1];
    const float z = fmaf(third * (1.f / (float)D), sh.scalar[2], om);
    if (group == 1) sh.kappa[d] = z / (rr + z) * (mine * rk);
    if (tid == 0) a.covariance[(size_t)slot * a.H + h] = rr * z / fmaf(a.posterior_scale, z, rr);
  }

  // ---- one pass over the state: S^ = alpha S, u = S^T k, w = S^T q ----
  cp_async_wait_all();
  float4 u = make_float4(0.f, 0.f, 0.f, 0.f), w = u;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = rg * ROWS + i;
    const float4 st = held[i * 4 * D];
    const float al = sh.alpha[row], kk = sh.k[row] * al, qq = sh.q[row] * al;
    u.x = fmaf(kk, st.x, u.x); u.y = fmaf(kk, st.y, u.y);
    u.z = fmaf(kk, st.z, u.z); u.w = fmaf(kk, st.w, u.w);
    w.x = fmaf(qq, st.x, w.x); w.y = fmaf(qq, st.y, w.y);
    w.z = fmaf(qq, st.z, w.z); w.w = fmaf(qq, st.w, w.w);
  }
  // D / 8 warps: the upper half leaves its sums, the lower half adds its own
  // (D = 64: a warp holds two row groups, joined first)
  if (D == 64) {
    u.x += __shfl_xor_sync(0xffffffffu, u.x, 16); u.y += __shfl_xor_sync(0xffffffffu, u.y, 16);
    u.z += __shfl_xor_sync(0xffffffffu, u.z, 16); u.w += __shfl_xor_sync(0xffffffffu, u.w, 16);
    w.x += __shfl_xor_sync(0xffffffffu, w.x, 16); w.y += __shfl_xor_sync(0xffffffffu, w.y, 16);
    w.z += __shfl_xor_sync(0xffffffffu, w.z, 16); w.w += __shfl_xor_sync(0xffffffffu, w.w, 16);
  }
  float4* pu = reinterpret_cast<float4*>(sh.part[0][warp % HALF]) + c4;
  float4* pw = reinterpret_cast<float4*>(sh.part[1][warp % HALF]) + c4;
  if (warp >= HALF && lane < D / 4) {
    *pu = u;
    *pw = w;
  }
  __syncthreads();
  if (DIAG && group == 3) {
#pragma unroll
    for (int i = 0; i < WG; ++i) third += sh.red[2][i];
    sh.kappa[d] = prior * kn / (r + third);
    a.covariance[(size_t)slot * C + ch] = prior / (1.f + (float)D * kn * kn / r * prior);
  }
  if (warp < HALF && lane < D / 4) {
    const float4 x = *pu, z = *pw;
    *pu = make_float4(u.x + x.x, u.y + x.y, u.z + x.z, u.w + x.w);
    *pw = make_float4(w.x + z.x, w.y + z.y, w.z + z.z, w.w + z.w);
  }
  __syncthreads();
  if (group >= 2) {  // the v threads finish u and delta, the gate threads w; a column's threads own it
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < HALF; ++i) s += sh.part[group - 2][i][d];
    if (group == 2) mine -= s * rk;  // delta
    sh.part[group - 2][0][d] = group == 2 ? mine : s * rq;
  }
  if (warp == 0) {  // q . kappa
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < WG; ++i) s = fmaf(sh.q[lane + 32 * i], sh.kappa[lane + 32 * i], s);
    s = warp_sum(s);
    if (lane == 0) sh.scalar[3] = s * rq;
  }
  __syncthreads();
  const float4 dl = reinterpret_cast<const float4*>(sh.part[0][0])[c4];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = rg * ROWS + i;
    const float al = sh.alpha[row], ka = sh.kappa[row];
    float4 st = held[i * 4 * D];
    st.x = fmaf(ka, dl.x, al * st.x); st.y = fmaf(ka, dl.y, al * st.y);
    st.z = fmaf(ka, dl.z, al * st.z); st.w = fmaf(ka, dl.w, al * st.w);
    S[i * (D / 4)] = st;
  }
  if (group == 2) {
    const float o = a.scale * fmaf(sh.scalar[3], mine, sh.part[1][0][d]);
    const float s = warp_sum(o * o);
    if (lane == 0) sh.out[warp % WG] = s;
    bar_sync(1, D);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < WG; ++i) ss += sh.out[i];
    *y = from_f<T>(o * rsqrtf(ss * (1.f / (float)D) + a.eps) * act);
  }
}

template <int D, bool DIAG, class T>
int launch_step(const StepParams& p, unsigned grid, cudaStream_t st) {
  constexpr size_t smem = sizeof(StepShared<D>);
  if (int rc = allow_smem<step_kernel<D, DIAG, T>>(smem, "step_kernel")) return rc;
  step_kernel<D, DIAG, T><<<grid, 4 * D, smem, st>>>(p);
  return check_launch("step_kernel");
}

template <int D, class T>
int launch_step(const StepParams& p, unsigned grid, cudaStream_t st) {
  return p.a.variant == KDN_DIAG ? launch_step<D, true, T>(p, grid, st) : launch_step<D, false, T>(p, grid, st);
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
  if (a.D == 128) return a.act_bf16 ? launch_step<128, bf16>(p, grid, st) : launch_step<128, float>(p, grid, st);
  return a.act_bf16 ? launch_step<64, bf16>(p, grid, st) : launch_step<64, float>(p, grid, st);
}
