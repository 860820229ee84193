// Forward of the norms around a block (mathematics and layout: kdn_block_norm.cuh).
#include "kdn_block_norm.cuh"

namespace kdn {
namespace {

constexpr int kBnGroups = kBnFwdWarps / 2;  // row groups of two warps or more in a CTA

// FULL: y comes with a norm, gate or scale (else plainly, or not at all).
template <class TX, class TY, int SLOTS, bool FULL, BnRows ROWS>
__global__ void __launch_bounds__(32 * kBnFwdWarps, 1) block_norm_fwd_kernel(const __grid_constant__ BnParams prm) {
  const KdnBlockNormArgs& a = prm.a;
  constexpr int PX = Raw<TX>::kPlanes, PY = Raw<TY>::kPlanes;
  __shared__ __align__(16) float red_all[kBnGroups][2 * kBnRed];
  extern __shared__ uint4 smem[];  // the weights, then the ring: [stages][groups][planes][nv + 1]
  const int tpr = prm.tpr, group = threadIdx.x / tpr, t = threadIdx.x - group * tpr, rpb = blockDim.x / tpr;
  const int D = (int)a.D, nv = bn_vectors(D, ROWS == kBnPacked), places = nv + 1;
  // packed rows: the shift of this CTA's, and their vectors
  const int turn = ROWS == kBnPacked ? (int)(blockIdx.x % prm.period) : 0, shift = ROWS == kBnPacked ? turn * D % kBnVec : 0;
  const int own = ROWS == kBnPacked ? (shift + D + kBnVec - 1) / kBnVec : nv;
  const float inv_D = 1.f / (float)D;
  const bool has_y = a.y != nullptr;
  const int gate = !(FULL && a.gate) ? kBnOpen : a.swish ? kBnSwish : kBnSigmoid;
  float* red = red_all[group < kBnGroups ? group : 0];  // groups of one warp need none
  for (int i = threadIdx.x; i < kBnGroups * 2 * kBnRed; i += blockDim.x) red_all[0][i] = 0.f;
  float4* kept = reinterpret_cast<float4*>(smem);
  stage_weights<ROWS, FULL>(kept, a, nv, shift);
  const BnSource<TX, ROWS> X(a.x, a.x_stride, a.rows, D);
  const BnSource<TY, ROWS> Y(a.y, a.y_stride, a.rows, D), G(gate ? a.gate : nullptr, a.gate_stride, a.rows, D);
  const int stage_size = rpb * prm.planes * places;
  uint4* ring = smem + kWeightPlanes<FULL> * places + group * prm.planes * places;
  // lanes past the row read vector nv, which stays zero (aligned and packed rows)
  auto clear = [&](int plane, int pieces) {
    for (int k = 0; k < prm.stages; ++k)
      for (int i = pieces * own + t; i < pieces * places; i += tpr)
        ring[k * stage_size + plane * places + i] = make_uint4(0, 0, 0, 0);
  };
  clear(0, PX);
  if (FULL || has_y) clear(PX, PY);
  if (G) clear(PX + PY, PY);
  __syncthreads();
  auto vec = [&](int s) { return s < SLOTS - 1 ? t + s * tpr : min(t + s * tpr, nv); };
  // the row's values of a vector: from lowest(s) to width(s)
  auto width = [&](int s) {
    return ROWS == kBnAligned && s < SLOTS - 1 ? kBnVec : min(max(shift + D - (t + s * tpr) * kBnVec, 0), kBnVec);
  };
  auto lowest = [&](int s) { return ROWS == kBnPacked && s == 0 && t == 0 ? shift : 0; };
  auto copy = [&](int64_t r, int stage) {
    if (r >= a.rows) return;
    uint4* d = ring + stage * stage_size;
    X.template copy<SLOTS>(r, d, t, tpr, own, shift);
    if (FULL || has_y) Y.template copy<SLOTS>(r, d + PX * places, t, tpr, own, shift);
    if (G) G.template copy<SLOTS>(r, d + (PX + PY) * places, t, tpr, own, shift);
  };
  int phase = 0;
  const int64_t step = (int64_t)gridDim.x * rpb;
  int64_t row = (int64_t)blockIdx.x * rpb + group;
  if (ROWS == kBnPacked) row = turn + prm.period * ((int64_t)(blockIdx.x / prm.period) * rpb + group);
  BnRing<ROWS != kBnLoose> rows_in(prm.stages, row, step, copy);
  for (; row < a.rows; row += step) {
    const uint4* here = ring + rows_in.next(row, step, group, tpr, copy) * stage_size;
    if (ROWS == kBnPacked)
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {
        const int v = vec(s), n = width(s), lo = lowest(s);
        if (n == 0 || (n == kBnVec && lo == 0)) continue;
        clear_outer<TX>(here + PX * v, lo, n);
        if (FULL || has_y) clear_outer<TY>(here + PX * places + PY * v, lo, n);
        if (G) clear_outer<TY>(here + (PX + PY) * places + PY * v, lo, n);
      }
    Raw<TY> y[SLOTS];
    if (FULL || has_y) {
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) Y.take(y[s], row, here + PX * places, vec(s), width(s));
    } else {
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) y[s].zero();
    }
    float sum[1], ry = 1.f;
    float2 z[SLOTS][4], ss = both(0.f);
    if (FULL && a.post_weight) {
#pragma unroll
      for (int s = 0; s < SLOTS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) ss = fma2(y[s][i], y[s][i], ss);
      sum[0] = ss.x + ss.y;
      group_sum<1>(sum, red, phase, tpr, group);
      ry = rsqrtf(fmaf(sum[0], inv_D, a.eps));
      ss = both(0.f);
    }
    by_gate<FULL>(gate, [&](auto kind) {
      constexpr int GATE = decltype(kind)::value;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {
        Raw<TX> x;
        Raw<TY> g;
        float2 m[4];
        X.take(x, row, here, vec(s), width(s));
        if (GATE != kBnOpen) G.take(g, row, here + (PX + PY) * places, vec(s), width(s));
        if (FULL) recall(m, kept + 2 * places + vec(s), places);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float2 u = y[s][i];
          if (FULL) {
            u = mul2(mul2(u, both(ry)), m[i]);
            if (GATE != kBnOpen) u = mul2(u, sigmoid2(g[i]));
            if (GATE == kBnSwish) u = mul2(u, g[i]);
          }
          z[s][i] = fma2(both(a.alpha), x[i], u);
          ss = fma2(z[s][i], z[s][i], ss);
        }
      }
    });
    sum[0] = ss.x + ss.y;
    group_sum<1>(sum, red, phase, tpr, group);
    const float rz = rsqrtf(fmaf(sum[0], inv_D, a.eps));
    if (a.rstd && t == 0) {
      a.rstd[row] = ry;
      a.rstd[a.rows + row] = rz;
    }
    const size_t at = (size_t)row * D - shift + t * kBnVec;
    if (has_y)
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) put<ROWS>(static_cast<TX*>(a.z) + at + s * tpr * kBnVec, z[s], width(s), lowest(s));
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      float2 w[4];
      recall(w, kept + vec(s), places);
#pragma unroll
      for (int i = 0; i < 4; ++i) z[s][i] = mul2(mul2(z[s][i], both(rz)), w[i]);
      put<ROWS>(static_cast<TY*>(a.h) + at + s * tpr * kBnVec, z[s], width(s), lowest(s));
    }
  }
}

template <class TX, class TY, bool FULL, BnRows ROWS>
int fwd_sizes(const BnParams& p, const BnGeom& g, cudaStream_t st) {
  const char* what = "block_norm_fwd_kernel";
  constexpr size_t fixed = sizeof(float) * kBnGroups * 2 * kBnRed;
  if (g.slots == 1) return bn_start<block_norm_fwd_kernel<TX, TY, 1, FULL, ROWS>>(p, g, ROWS, kWeightPlanes<FULL>, fixed, what, st);
  if (g.slots == 2) return bn_start<block_norm_fwd_kernel<TX, TY, 2, FULL, ROWS>>(p, g, ROWS, kWeightPlanes<FULL>, fixed, what, st);
  return bn_start<block_norm_fwd_kernel<TX, TY, 3, FULL, ROWS>>(p, g, ROWS, kWeightPlanes<FULL>, fixed, what, st);
}

template <class TX, class TY, BnRows ROWS>
int fwd_rows(const BnParams& p, const BnGeom& g, cudaStream_t st) {
  const bool full = p.a.post_weight || p.a.gate || p.a.scale;
  return full ? fwd_sizes<TX, TY, true, ROWS>(p, g, st) : fwd_sizes<TX, TY, false, ROWS>(p, g, st);
}

template <class TX, class TY>
int fwd_types(const BnParams& p, const BnGeom& g, BnRows kind, cudaStream_t st) {
  if (kind == kBnAligned) return fwd_rows<TX, TY, kBnAligned>(p, g, st);
  if (kind == kBnPacked) return fwd_rows<TX, TY, kBnPacked>(p, g, st);
  return fwd_rows<TX, TY, kBnLoose>(p, g, st);
}

}  // namespace

int block_norm_check(const char* what, const KdnBlockNormArgs* p) {
  if (!p) return set_error(KDN_ERR_INVALID, "%s: null args", what);
  const KdnBlockNormArgs& a = *p;
  if (a.rows < 0 || a.D < kBnMinD || a.D > kBnMaxD)
    return set_error(KDN_ERR_INVALID, "%s: rows >= 0 and D in [%d, %d] required", what, kBnMinD, kBnMaxD);
  if (a.stream_bf16 && !a.act_bf16)
    return set_error(KDN_ERR_INVALID, "%s: fp32 activations need an fp32 residual stream", what);
  if (a.rows == 0) return KDN_OK;
  if (!a.x || !a.weight) return set_error(KDN_ERR_INVALID, "%s: null pointer", what);
  if (!a.y && (a.gate || a.post_weight || a.scale || a.alpha != 1.f))
    return set_error(KDN_ERR_INVALID, "%s: gate, post_weight, scale and alpha need a block output y", what);
  auto bad = [&](int64_t stride) { return stride < a.D && stride != 0; };  // 0: one row for all
  if (a.rows > 1 && (bad(a.x_stride) || (a.y && bad(a.y_stride)) || (a.gate && bad(a.gate_stride))))
    return set_error(KDN_ERR_INVALID, "%s: row strides smaller than the rows", what);
  return KDN_OK;
}

}  // namespace kdn

using namespace kdn;

extern "C" int kdn_block_norm_fwd(const KdnBlockNormArgs* args, kdn_stream_t stream) {
  if (int rc = block_norm_check("kdn_block_norm_fwd", args)) return rc;
  const KdnBlockNormArgs& a = *args;
  if (a.rows == 0) return KDN_OK;
  if (!a.h || (a.y && !a.z)) return set_error(KDN_ERR_INVALID, "kdn_block_norm_fwd: null output");
  const BnRows kind = bn_rows(a);
  const BnGeom g = bn_geom(a.rows, a.D, kind == kBnLoose ? kBnFwdWarps : kBnBwdWarps, kind, false);
  const int ex = a.stream_bf16 ? 1 : 2, ey = a.act_bf16 ? 1 : 2;
  const BnParams p{a, nullptr, g.tpr, g.period, ex + (a.y ? ey : 0) + (a.gate ? ey : 0), 0};
  cudaStream_t st = (cudaStream_t)stream;
  if (a.act_bf16 && a.stream_bf16) return fwd_types<bf16, bf16>(p, g, kind, st);
  if (a.act_bf16) return fwd_types<float, bf16>(p, g, kind, st);
  return fwd_types<float, float>(p, g, kind, st);
}
