// Backward of the norms around a block (mathematics and layout: kdn_block_norm.cuh).
#include <algorithm>

#include "kdn_block_norm.cuh"

namespace kdn {

int block_norm_check(const char* what, const KdnBlockNormArgs* p);  // kdn_block_norm.cu

namespace {

constexpr int kBnGroups = kBnBwdWarps / 2;  // row groups of two warps or more in a CTA

// The three row sums come from one pass and one reduction: with
// m = s scale post and e = dz + rz w dh, Z = e - rz c1 zh, so
//   mean(t yh) = mean(e m yh) - rz c1 mean(zh m yh),  c1 = mean(w dh zh).
template <class TX, class TY, int SLOTS, bool FULL, BnRows ROWS>
__global__ void __launch_bounds__(32 * kBnBwdWarps, 1) block_norm_bwd_kernel(const __grid_constant__ BnParams prm) {
  const KdnBlockNormArgs& a = prm.a;
  constexpr int PX = Raw<TX>::kPlanes, PY = Raw<TY>::kPlanes;
  constexpr int NS = FULL ? 3 : 1;  // row sums
  constexpr int NW = FULL ? 2 : 1;  // column sums
  __shared__ __align__(16) float red_all[kBnGroups][2 * NS * kBnRed];
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
  for (int i = threadIdx.x; i < kBnGroups * 2 * NS * kBnRed; i += blockDim.x) red_all[0][i] = 0.f;
  float4* kept = reinterpret_cast<float4*>(smem);
  stage_weights<ROWS, FULL>(kept, a, nv, shift);
  const BnSource<TX, ROWS> X(a.x, a.x_stride, a.rows, D), DZ(a.dz, D, a.rows, D);
  const BnSource<TY, ROWS> DH(a.dh, D, a.rows, D), Y(a.y, a.y_stride, a.rows, D),
      G(gate ? a.gate : nullptr, a.gate_stride, a.rows, D);
  const int stage_size = rpb * prm.planes * places;
  constexpr int kDZ = PX, kDH = 2 * PX, kY = 2 * PX + PY, kG = 2 * PX + 2 * PY;  // planes
  uint4* ring = smem + kWeightPlanes<FULL> * places + group * prm.planes * places;
  // lanes past the row read vector nv, which stays zero (aligned and packed rows); absent cotangents are zero
  auto clear = [&](int plane, int pieces, int from) {
    for (int k = 0; k < prm.stages; ++k)
      for (int i = pieces * from + t; i < pieces * places; i += tpr)
        ring[k * stage_size + plane * places + i] = make_uint4(0, 0, 0, 0);
  };
  clear(0, PX, own);
  clear(kDZ, PX, DZ ? own : 0);
  clear(kDH, PY, DH ? own : 0);
  if (FULL || has_y) clear(kY, PY, own);
  if (G) clear(kG, PY, own);
  __syncthreads();
  auto vec = [&](int s) { return s < SLOTS - 1 ? t + s * tpr : min(t + s * tpr, nv); };
  // the row's values of a vector: from lowest(s) to width(s)
  auto width = [&](int s) {
    return ROWS == kBnAligned && s < SLOTS - 1 ? kBnVec : min(max(shift + D - (t + s * tpr) * kBnVec, 0), kBnVec);
  };
  auto lowest = [&](int s) { return ROWS == kBnPacked && s == 0 && t == 0 ? shift : 0; };
  // A warp past the row leaves a slot out (16384 x 2304 bf16, all parts: 113.5 us, without 117; 8192 x 2312: 80, 82.5).
  // Packed rows lose what they gain by it (8192 x 2305 bf16 98 us against 97, fp32 136 against 138).
  auto idle = [&](int s) { return ROWS == kBnAligned && s == SLOTS - 1 && (t & ~31) + s * tpr >= nv; };
  auto copy = [&](int64_t r, int stage) {
    if (r >= a.rows) return;
    uint4* d = ring + stage * stage_size;
    X.template copy<SLOTS>(r, d, t, tpr, own, shift);
    if (DZ) DZ.template copy<SLOTS>(r, d + kDZ * places, t, tpr, own, shift);
    if (DH) DH.template copy<SLOTS>(r, d + kDH * places, t, tpr, own, shift);
    if (FULL || has_y) Y.template copy<SLOTS>(r, d + kY * places, t, tpr, own, shift);
    if (G) G.template copy<SLOTS>(r, d + kG * places, t, tpr, own, shift);
  };
  float2 acc[SLOTS][NW][4];  // this thread's column sums
#pragma unroll
  for (int s = 0; s < SLOTS; ++s)
#pragma unroll
    for (int k = 0; k < NW; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[s][k][i] = both(0.f);
  int phase = 0;
  const int64_t step = (int64_t)gridDim.x * rpb;
  int64_t row = (int64_t)blockIdx.x * rpb + group;
  if (ROWS == kBnPacked) row = turn + prm.period * ((int64_t)(blockIdx.x / prm.period) * rpb + group);
  BnRing<ROWS != kBnLoose> rows_in(prm.stages, row, step, copy);
  float next_ry = 0.f, next_rz = 0.f;  // the coming row's statistics, requested a row ahead
  if (row < a.rows) {
    next_ry = a.rstd[row];
    next_rz = a.rstd[a.rows + row];
  }
  for (; row < a.rows; row += step) {
    const float ry = next_ry, rz = next_rz;
    if (row + step < a.rows) {
      next_ry = a.rstd[row + step];
      next_rz = a.rstd[a.rows + row + step];
    }
    const uint4* here = ring + rows_in.next(row, step, group, tpr, copy) * stage_size;
    if (ROWS == kBnPacked)
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {
        const int v = vec(s), n = width(s), lo = lowest(s);
        if (n == 0 || (n == kBnVec && lo == 0)) continue;
        clear_outer<TX>(here + PX * v, lo, n);
        if (DZ) clear_outer<TX>(here + kDZ * places + PX * v, lo, n);
        if (DH) clear_outer<TY>(here + kDH * places + PY * v, lo, n);
        if (FULL || has_y) clear_outer<TY>(here + kY * places + PY * v, lo, n);
        if (G) clear_outer<TY>(here + kG * places + PY * v, lo, n);
      }
    float2 zh[SLOTS][4], ss[NS];
#pragma unroll
    for (int k = 0; k < NS; ++k) ss[k] = both(0.f);
    by_gate<FULL>(gate, [&](auto kind) {
      constexpr int GATE = decltype(kind)::value;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {
        if (idle(s)) continue;
        const int v = vec(s), n = width(s);
        Raw<TX> x, dz;
        Raw<TY> y, g, dh;
        float2 w[4], m[4];
        if (FULL || has_y) Y.take(y, row, here + kY * places, v, n);
        else y.zero();
        if (GATE != kBnOpen) G.take(g, row, here + kG * places, v, n);
        X.take(x, row, here, v, n);
        DH.take(dh, row, here + kDH * places, v, n);
        recall(w, kept + v, places);
        if (FULL) {
          DZ.take(dz, row, here + kDZ * places, v, n);
          recall(m, kept + 2 * places + v, places);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float2 u = y[i];
          if (FULL) {
            u = mul2(mul2(u, both(ry)), m[i]);
            if (GATE != kBnOpen) u = mul2(u, sigmoid2(g[i]));
            if (GATE == kBnSwish) u = mul2(u, g[i]);
          }
          zh[s][i] = mul2(fma2(both(a.alpha), x[i], u), both(rz));
          const float2 wd = mul2(w[i], dh[i]);
          ss[0] = fma2(wd, zh[s][i], ss[0]);
          if constexpr (FULL) {  // u = m yh
            ss[1] = fma2(fma2(both(rz), wd, dz[i]), u, ss[1]);
            ss[2] = fma2(zh[s][i], u, ss[2]);
          }
        }
      }
    });
    float sum[NS];
#pragma unroll
    for (int k = 0; k < NS; ++k) sum[k] = ss[k].x + ss[k].y;
    group_sum<NS>(sum, red, phase, tpr, group);
    const float c1 = rz * sum[0] * inv_D;
    float c2 = 0.f;
    if constexpr (FULL) c2 = a.post_weight ? sum[1] * inv_D - c1 * (sum[2] * inv_D) : 0.f;
    const size_t at = (size_t)row * D - shift + t * kBnVec;
    by_gate<FULL>(gate, [&](auto kind) {
      constexpr int GATE = decltype(kind)::value;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {  // everything but zh again from the ring: no registers held over the reduction
        if (idle(s)) continue;
        const int v = vec(s), n = width(s);
        const size_t o = at + s * tpr * kBnVec;
        Raw<TX> dz;
        Raw<TY> y, g, dh;
        float2 w[4], Z[4], out[4];
        DZ.take(dz, row, here + kDZ * places, v, n);
        DH.take(dh, row, here + kDH * places, v, n);
        recall(w, kept + v, places);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[s][0][i] = fma2(dh[i], zh[s][i], acc[s][0][i]);
          Z[i] = fma2(both(-c1), zh[s][i], fma2(both(rz), mul2(w[i], dh[i]), dz[i]));
          out[i] = mul2(both(a.alpha), Z[i]);
        }
        if (a.dx) put<ROWS>(static_cast<TX*>(a.dx) + o, out, n, lowest(s));
        if constexpr (!FULL) {
          if (a.dy) put<ROWS>(static_cast<TY*>(a.dy) + o, Z, n, lowest(s));
        } else {
          float2 m[4], dg[4];
          Y.take(y, row, here + kY * places, v, n);
          if (GATE != kBnOpen) G.take(g, row, here + kG * places, v, n);
          recall(m, kept + 2 * places + v, places);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 yh = mul2(y[i], both(ry)), Zy = mul2(Z[i], yh);
            float2 am = m[i], flow = Zy;  // act m and Z yh act
            if (GATE == kBnSigmoid) {     // act' = act (1 - act)
              const float2 open = sigmoid2(g[i]);
              am = mul2(m[i], open);
              flow = mul2(Zy, open);
              dg[i] = mul2(flow, fma2(both(-1.f), am, m[i]));
            } else if (GATE == kBnSwish) {  // act = g s, act' = s + act (1 - s)
              const float2 open = sigmoid2(g[i]), act = mul2(g[i], open);
              am = mul2(m[i], act);
              flow = mul2(Zy, act);
              dg[i] = mul2(mul2(Zy, m[i]), fma2(act, fma2(both(-1.f), open, both(1.f)), open));
            }
            acc[s][NW - 1][i] = add2(acc[s][NW - 1][i], flow);
            out[i] = mul2(both(ry), fma2(both(-c2), yh, mul2(Z[i], am)));
          }
          if (GATE != kBnOpen && a.dgate) put<ROWS>(static_cast<TY*>(a.dgate) + o, dg, n, lowest(s));
          if (a.dy) put<ROWS>(static_cast<TY*>(a.dy) + o, out, n, lowest(s));
        }
      }
    });
  }
  if (!prm.partial) return;
  // the row groups' sums, added up in the ring's memory (at most 12 * 32 * 24 columns in all)
  cp_async_wait_group<0>();
  __syncthreads();
  float* all = reinterpret_cast<float*>(smem);  // [groups][NW][D]
#pragma unroll
  for (int s = 0; s < SLOTS; ++s)
#pragma unroll
    for (int k = 0; k < NW; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i >= lowest(s) && i < width(s))
          all[(group * NW + k) * D + (t + s * tpr) * kBnVec - shift + i] = i & 1 ? acc[s][k][i / 2].y : acc[s][k][i / 2].x;
  __syncthreads();
  float* partial = prm.partial + (size_t)blockIdx.x * 2 * D;
  for (int i = threadIdx.x; i < NW * D; i += blockDim.x) {
    float s = all[i];
    for (int g = 1; g < rpb; ++g) s += all[g * NW * D + i];
    partial[i] = s;
  }
}

// Weight gradients: column sums of the CTAs' partial rows in a fixed order (32
// columns x 16 chains of four loads in flight per CTA); the second sum times scale is dpost, times
// post_weight dscale.
constexpr int kBnChains = 16;
__global__ void __launch_bounds__(32 * kBnChains) block_norm_weights_kernel(const __grid_constant__ BnParams prm,
                                                                             int parts) {
  const KdnBlockNormArgs& a = prm.a;
  __shared__ float red[kBnChains][33];
  if (blockIdx.y == 0 ? !a.dweight : !a.dpost && !a.dscale) return;
  const int D = (int)a.D, lane = threadIdx.x & 31, chain = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (col < D)
    for (int p0 = chain; p0 < parts; p0 += 4 * kBnChains) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int p = p0 + j * kBnChains;
        v[j] = p < parts ? prm.partial[((size_t)p * 2 + blockIdx.y) * D + col] : 0.f;
      }
      s += (v[0] + v[1]) + (v[2] + v[3]);
    }
  red[chain][lane] = s;
  __syncthreads();
  if (chain != 0 || col >= D) return;
#pragma unroll
  for (int c = 1; c < kBnChains; ++c) s += red[c][lane];
  const bool wb = a.weights_bf16 != 0;
  auto weight = [&](const void* p) {
    return !p ? 1.f : wb ? to_f(static_cast<const bf16*>(p)[col]) : static_cast<const float*>(p)[col];
  };
  auto store = [&](void* p, float v) {
    if (!p) return;
    if (wb) static_cast<bf16*>(p)[col] = from_f<bf16>(v);
    else static_cast<float*>(p)[col] = v;
  };
  if (blockIdx.y == 0) {
    store(a.dweight, s);
  } else {
    store(a.dpost, s * weight(a.scale));
    store(a.dscale, s * weight(a.post_weight));
  }
}

template <class TX, class TY, bool FULL, BnRows ROWS>
int bwd_sizes(const BnParams& p, const BnGeom& g, cudaStream_t st) {
  const char* what = "block_norm_bwd_kernel";
  constexpr size_t fixed = sizeof(float) * kBnGroups * 2 * (FULL ? 3 : 1) * kBnRed;
  if (g.slots == 1) return bn_start<block_norm_bwd_kernel<TX, TY, 1, FULL, ROWS>>(p, g, ROWS, kWeightPlanes<FULL>, fixed, what, st);
  if (g.slots == 2) return bn_start<block_norm_bwd_kernel<TX, TY, 2, FULL, ROWS>>(p, g, ROWS, kWeightPlanes<FULL>, fixed, what, st);
  return bn_start<block_norm_bwd_kernel<TX, TY, 3, FULL, ROWS>>(p, g, ROWS, kWeightPlanes<FULL>, fixed, what, st);
}

template <class TX, class TY, BnRows ROWS>
int bwd_rows(const BnParams& p, const BnGeom& g, cudaStream_t st) {
  const bool full = p.a.post_weight || p.a.gate || p.a.scale;
  return full ? bwd_sizes<TX, TY, true, ROWS>(p, g, st) : bwd_sizes<TX, TY, false, ROWS>(p, g, st);
}

template <class TX, class TY>
int bwd_types(const BnParams& p, const BnGeom& g, BnRows kind, cudaStream_t st) {
  if (kind == kBnAligned) return bwd_rows<TX, TY, kBnAligned>(p, g, st);
  if (kind == kBnPacked) return bwd_rows<TX, TY, kBnPacked>(p, g, st);
  return bwd_rows<TX, TY, kBnLoose>(p, g, st);
}

BnGeom bwd_geom(int64_t rows, int64_t D, BnRows kind) {
  return bn_geom(rows, D, kBnBwdWarps, kind, kind == kBnLoose);
}

}  // namespace
}  // namespace kdn

using namespace kdn;

extern "C" {

size_t kdn_block_norm_workspace_bytes(int64_t rows, int64_t D) {
  if (rows <= 0 || D < kBnMinD || D > kBnMaxD) return 0;
  unsigned most = 0;  // of the grids
  for (const BnRows kind : {kBnLoose, kBnAligned, kBnPacked}) most = std::max(most, bwd_geom(rows, D, kind).grid);
  return align_up(sizeof(float) * 2 * (size_t)D * most, 256);
}

int kdn_block_norm_bwd(const KdnBlockNormArgs* args, kdn_stream_t stream) {
  if (int rc = block_norm_check("kdn_block_norm_bwd", args)) return rc;
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
  const BnRows kind = bn_rows(a);
  const BnGeom g = bwd_geom(a.rows, a.D, kind);
  const int ex = a.stream_bf16 ? 1 : 2, ey = a.act_bf16 ? 1 : 2;
  const BnParams p{a, weights ? static_cast<float*>(a.workspace) : nullptr, g.tpr, g.period,
                   2 * ex + (a.y ? 2 : 1) * ey + (a.gate ? ey : 0), 0};
  if (int rc = a.act_bf16 && a.stream_bf16 ? bwd_types<bf16, bf16>(p, g, kind, st)
               : a.act_bf16               ? bwd_types<float, bf16>(p, g, kind, st)
                                          : bwd_types<float, float>(p, g, kind, st))
    return rc;
  if (!weights) return KDN_OK;
  block_norm_weights_kernel<<<dim3((unsigned)((a.D + 31) / 32), 2), 32 * kBnChains, 0, st>>>(p, (int)g.grid);
  return check_launch("block_norm_weights_kernel");
}

}  // extern "C"
