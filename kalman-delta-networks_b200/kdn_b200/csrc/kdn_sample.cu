// One token per row of logits under temperature, top-k, top-p and min-p, from
// given Exp(1) random numbers.  With e_i = exp((l_i - max) / T), Z = sum e and
// the order "larger logit first, then lower index", the filters keep a prefix
// of the order: rank < top_k, (sum of e ahead) < top_p Z, e >= min_p.  The
// token is the kept one with the largest e_i / noise_i: with independent
// exponential noise it is drawn with probability e_i / (sum of the kept e).
//
// No sort is needed, because the kept set is a prefix.  A cluster of CTAs
// holds a row in shared memory (read once) and
//  1. finds the maximum,
//  2. sums Z and fills a histogram over 1/16-octave bins of e, whose integer
//     entries bound the count and the mass ahead of every bin from both sides:
//     tokens from bin `cut` on are certainly dropped, those before bin `safe`
//     are certainly within top-k and top-p,
//  3. races the tokens before `cut` (only their random numbers are read).  A
//     winner before `safe` is the answer.  Otherwise the exact count and mass
//     ahead of it are taken; if it is not kept, the tokens ahead of it race.
// Every race lost drops the winner and what is behind it; after kRaces of them
// (noise that follows the logits) the end of the kept prefix is bisected
// instead, so that no row takes more than kRaces + 64 turns.  Sums have a fixed
// order or are integers.
#include <cooperative_groups.h>

#include "kdn_common.cuh"

namespace kdn {
namespace {

namespace cg = cooperative_groups;

constexpr int kSmThreads = 512, kSmWarps = kSmThreads / 32;
constexpr int kSmChunk = 16384;     // tokens per CTA before a row gets another one
constexpr int kSmHeld = 192 * 1024;  // bytes of shared memory for them; what a chunk has beyond is read again in every pass
constexpr int kSmCluster = 8;
constexpr int kRaces = 12;
constexpr int kBins = 1024;       // of 1/16 octave: e down to 2^-64
constexpr float kPerOctave = 16.f;
constexpr float kBinLow = 0.957f;  // 2^(-1/16), rounded down: the smallest e of a bin over its largest

struct Best {  // a race's leader: the larger score, then the earlier in the order
  float score, logit;
  int index;
};
__device__ __forceinline__ bool ahead(float la, int ia, float lb, int ib) { return la > lb || (la == lb && ia < ib); }
__device__ __forceinline__ bool beats(const Best& a, const Best& b) {
  return a.score > b.score || (a.score == b.score && ahead(a.logit, a.index, b.logit, b.index));
}
__device__ __forceinline__ Best shuffle(const Best& b, int o) {
  return Best{__shfl_xor_sync(~0u, b.score, o), __shfl_xor_sync(~0u, b.logit, o), __shfl_xor_sync(~0u, b.index, o)};
}
__device__ __forceinline__ Best warp_best(Best b) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Best c = shuffle(b, o);
    if (beats(c, b)) b = c;
  }
  return b;
}
__device__ __forceinline__ float clean(float l) { return isnan(l) ? -INFINITY : l; }

// Whole-number keys in the order of the logits.
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t u = __float_as_uint(l);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// The part of a row that one CTA works on: tokens [begin, end), the first
// `held` of them in shared memory, where every thread keeps its own.  VEC: 8
// neighbouring tokens per thread and group (rows that start on 16-byte
// boundaries), else one by one, 512 apart.
template <class T, bool VEC>
struct Chunk {
  static constexpr int kPer = VEC ? 8 : 1;
  const T* row;
  int begin, end, groups;  // groups of kSmThreads * kPer tokens in shared memory
  T* held;

  __device__ __forceinline__ int first(int j) const { return begin + (j * kSmThreads + (int)threadIdx.x) * kPer; }
  // place of this thread's group j; fp32 vectors are split over two planes
  __device__ __forceinline__ T* place(int j) const {
    return held + (size_t)(VEC && sizeof(T) == 4 ? 2 * j * kSmThreads * 4 + threadIdx.x * 4
                                                 : (j * kSmThreads + threadIdx.x) * kPer);
  }
  __device__ __forceinline__ void load() {
#pragma unroll 4
    for (int j = 0; j < groups; ++j) {
      const int i = first(j);
      T* to = place(j);
      if constexpr (!VEC) {
        if constexpr (sizeof(T) == 4) {
          if (i < end) cp_async4(to, row + i);
          else *to = -INFINITY;
        } else {
          *to = i < end ? row[i] : from_f<T>(-INFINITY);
        }
      } else if (i + 8 <= end) {
        cp_async16(to, row + i);
        if constexpr (sizeof(T) == 4) cp_async16(to + kSmThreads * 4, row + i + 4);
      } else {
        for (int k = 0; k < 8; ++k)
          to[sizeof(T) == 4 && k >= 4 ? kSmThreads * 4 + k - 4 : k] = i + k < end ? row[i + k] : from_f<T>(-INFINITY);
      }
    }
    cp_async_commit();
    cp_async_wait_all();
  }
  // f(logit, index) for this thread's tokens, in a fixed order (past the end: -inf)
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
#pragma unroll 1
    for (int j = 0; j < groups; ++j) {
      const int i = first(j);
      const T* at = place(j);
      if constexpr (!VEC) {
        f(clean(to_f(*at)), i);
      } else {
        float v[8];
        if constexpr (sizeof(T) == 2) {
          ld8(v, at);
        } else {
          const float4 p = *reinterpret_cast<const float4*>(at), q = *reinterpret_cast<const float4*>(at + kSmThreads * 4);
          v[0] = p.x; v[1] = p.y; v[2] = p.z; v[3] = p.w; v[4] = q.x; v[5] = q.y; v[6] = q.z; v[7] = q.w;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) f(clean(v[k]), i + k);
      }
    }
    for (int i = begin + groups * kSmThreads * kPer + (int)threadIdx.x; i < end; i += kSmThreads) f(clean(to_f(row[i])), i);
  }
};

struct Shared {
  float top[kSmWarps], mass[2][kSmWarps];
  int first[kSmWarps], count[2][kSmWarps];
  Best best[2][kSmWarps];
  uint32_t hist[kBins];
  unsigned long long scan_s[kSmWarps];
  float scan_m[kSmWarps];
  int cut[kSmWarps], safe[kSmWarps];
};

// f(value) over the warps' entries of every CTA of the cluster: lane by lane, then `join` over the warp
template <class V, class J>
__device__ __forceinline__ V gather(cg::cluster_group& cluster, V* mine, int ctas, V none, J&& join) {
  const int lane = threadIdx.x & 31;
  V v = none;
  for (int e = lane; e < ctas * kSmWarps; e += 32) {
    V* at = mine + e % kSmWarps;
    v = join(v, ctas == 1 ? *at : *cluster.map_shared_rank(at, e / kSmWarps));
  }
  return v;
}

template <class T, bool VEC>
__global__ void __launch_bounds__(kSmThreads, 3) sample_kernel(const __grid_constant__ KdnSampleArgs a, int ctas,
                                                              int chunk, int groups, float fraction) {
  __shared__ __align__(16) Shared sh;
  extern __shared__ uint4 held[];
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = (int)a.V;
  const int64_t row = blockIdx.x / ctas;
  const int rank = (int)(blockIdx.x % ctas);
  auto meet = [&] {
    if (ctas == 1) __syncthreads();
    else cluster.sync();
  };
  const float temp = a.temperature ? a.temperature[row] : a.temperature_all;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_all, min_p = a.min_p ? a.min_p[row] : a.min_p_all;
  int64_t top_k = !a.top_k ? a.top_k_all
                  : a.top_k_i64 ? static_cast<const int64_t*>(a.top_k)[row]
                                : (int64_t) static_cast<const int32_t*>(a.top_k)[row];
  if (top_k <= 0 || top_k > V) top_k = V;
  const bool greedy = !(temp > 0.f), by_rank = !greedy && (top_k < V || top_p < 1.f);
  const float* E = a.noise + row * a.noise_stride;

  Chunk<T, VEC> c;
  c.row = static_cast<const T*>(a.logits) + row * a.logits_stride;
  c.begin = min((int64_t)rank * chunk, (int64_t)V);
  c.end = min((int64_t)c.begin + chunk, (int64_t)V);
  c.groups = groups;
  c.held = reinterpret_cast<T*>(held);
  c.load();
  if (by_rank)
    for (int i = tid; i < kBins; i += kSmThreads) sh.hist[i] = 0;

  // ---- 1: the maximum ----
  float m = -INFINITY;
  c.each([&](float l, int) { m = fmaxf(m, l); });
  m = warp_max(m);
  if (lane == 0) sh.top[warp] = m;
  meet();
  const float top = warp_max(gather(cluster, sh.top, ctas, -INFINITY, [](float x, float y) { return fmaxf(x, y); }));
  if (top == -INFINITY) {
    if (rank == 0 && tid == 0) a.token[row] = -1, a.prob[row] = 0.f;
    meet();  // nobody leaves while its memory may be read
    return;
  }

  // ---- 2: Z, the order's first token, the histogram or the only race ----
  // octaves below the maximum, the product kept exact enough by a second term
  const float scale = 1.4426950408889634f / temp, rest = fmaf(-scale, temp, 1.4426950408889634f) / temp;
  auto octaves = [&](float l) {
    const float d = top - l;  // inf or (two infinities) NaN for infinite logits
    return l == top ? 0.f : d < INFINITY ? fmaf(d, scale, d * rest) : INFINITY;
  };
  auto score = [&](float e, int i) { return __fdividef(e, E[i]); };
  float z = 0.f;
  int first = INT32_MAX;
  Best best{-1.f, -INFINITY, INT32_MAX};
  auto enter = [&](float e, float l, int i) {
    const Best b{score(e, i), l, i};
    if (beats(b, best)) best = b;
  };
  if (greedy) {
    c.each([&](float l, int i) {
      if (l == top) first = min(first, i);
    });
  } else {
    c.each([&](float l, int i) {
      if (l == top) first = min(first, i);
      const float t = octaves(l), e = ex2a(-t);
      z += e;
      if (by_rank) {
        const float bin = floorf(t * kPerOctave);
        if (bin < (float)kBins)
          atomicAdd(&sh.hist[(int)bin], (uint32_t)(ex2a(bin * (1.f / kPerOctave) - t) * fraction));
      } else if (e > 0.f && e >= min_p) {
        enter(e, l, i);
      }
    });
  }
  z = warp_sum(z);
  first = __reduce_min_sync(~0u, first);
  best = warp_best(best);
  if (lane == 0) sh.mass[0][warp] = z, sh.first[warp] = first, sh.best[0][warp] = best;
  meet();
  // the CTAs' sums one after the other: the same order in every thread
  const float Z = warp_sum(gather(cluster, sh.mass[0], ctas, 0.f, [](float x, float y) { return x + y; }));
  first = __reduce_min_sync(~0u, gather(cluster, sh.first, ctas, INT32_MAX, [](int x, int y) { return min(x, y); }));
  auto faster = [](const Best& x, const Best& y) { return beats(y, x) ? y : x; };
  const Best nobody{-1.f, -INFINITY, INT32_MAX};
  Best win = greedy ? nobody : warp_best(gather(cluster, sh.best[0], ctas, nobody, faster));

  // ---- 3: races among the tokens before `cut` ----
  if (by_rank) {
    // bins 2 tid and 2 tid + 1 over the cluster
    unsigned long long s[2] = {0, 0};
    for (int r = 0; r < ctas; ++r) {
      const uint2 u = *reinterpret_cast<const uint2*>((ctas == 1 ? sh.hist : cluster.map_shared_rank(sh.hist, r)) + 2 * tid);
      s[0] += u.x;
      s[1] += u.y;
    }
    const float unit = 1.f / fraction;
    const float mass0 = (float)s[0] * unit * ex2a(-(float)(2 * tid) * (1.f / kPerOctave));
    const float mass1 = (float)s[1] * unit * ex2a(-(float)(2 * tid + 1) * (1.f / kPerOctave));
    unsigned long long ps = s[0] + s[1];  // inclusive scans over the threads
    float pm = mass0 + mass1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long us = __shfl_up_sync(~0u, ps, o);
      const float um = __shfl_up_sync(~0u, pm, o);
      if (lane >= o) ps += us, pm += um;
    }
    if (lane == 31) sh.scan_s[warp] = ps, sh.scan_m[warp] = pm;
    __syncthreads();
    for (int w = 0; w < warp; ++w) ps += sh.scan_s[w], pm += sh.scan_m[w];
    // before this thread's bins (a lower bound of what is ahead of them), after the first, after the second.
    // Entries are rounded down by less than one in 0.95 `fraction`; 1e-5 covers the sums' own rounding.
    const double k_units = (double)top_k * fraction;
    const float goal = top_p < 1.f ? top_p * Z : INFINITY;
    int cut = kBins + 1, safe = 0;
    const float over = 1.f + 2.f / (kBinLow * fraction) + 1e-5f;
#pragma unroll
    for (int b = 1; b >= 0; --b) {
      const unsigned long long sb = b ? ps - s[1] : ps - s[1] - s[0];
      const float mb = b ? pm - mass1 : pm - mass1 - mass0;
      if ((double)sb >= k_units || mb * (1.f - 1e-5f) >= goal) cut = 2 * tid + b;
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const unsigned long long sb = b ? ps : ps - s[1];
      const float mb = b ? pm : pm - mass1;
      if ((double)sb <= 0.95 * k_units && mb * over < goal) safe = 2 * tid + b + 1;
    }
    cut = __reduce_min_sync(~0u, cut);
    safe = __reduce_max_sync(~0u, safe);
    if (lane == 0) sh.cut[warp] = cut, sh.safe[warp] = safe;
    __syncthreads();
    cut = __reduce_min_sync(~0u, sh.cut[lane % kSmWarps]);
    safe = __reduce_max_sync(~0u, sh.safe[lane % kSmWarps]);
    const float cut_t = cut > kBins ? INFINITY : (float)cut, safe_t = fminf((float)safe, cut_t);

    // What a turn looks at lies ahead of (pl, pi) in the order.
    const Best leader{0.f, top, first};
    float pl = -INFINITY;
    int pi = INT32_MAX;
    // bisection: the last kept logit is in [lo, hi] (keys), then the last kept index of it
    enum { kRace, kLogit, kIndex, kLast } what = kRace;
    uint32_t lo = 0, hi = 0;
    for (int turn = 0;; ++turn) {
      best = nobody;
      float mass = 0.f;
      int count = 0;
      c.each([&](float l, int i) {
        if (!ahead(l, i, pl, pi)) return;
        const float t = octaves(l);
        if (!(t * kPerOctave < cut_t)) return;
        const float e = ex2a(-t);
        mass += e;
        ++count;
        if (e > 0.f && e >= min_p) enter(e, l, i);
      });
      mass = warp_sum(mass);
      count = __reduce_add_sync(~0u, count);
      best = warp_best(best);
      const int buf = 1 - (turn & 1);
      if (lane == 0) sh.mass[buf][warp] = mass, sh.count[buf][warp] = count, sh.best[buf][warp] = best;
      meet();
      mass = warp_sum(gather(cluster, sh.mass[buf], ctas, 0.f, [](float x, float y) { return x + y; }));
      count = __reduce_add_sync(~0u, gather(cluster, sh.count[buf], ctas, 0, [](int x, int y) { return x + y; }));
      best = warp_best(gather(cluster, sh.best[buf], ctas, nobody, faster));
      // whether a token at (pl, pi) is within top-k and top-p (the order's first always is)
      const bool kept = turn > 0 && (count == 0 || (count < top_k && (top_p >= 1.f || mass < top_p * Z)));
      if (what == kRace) {
        if (kept) break;  // (pl, pi) is the winner
        win = best.index == INT32_MAX ? leader : best;  // none: no score compares
        if (win.index == first || octaves(win.logit) * kPerOctave < safe_t) break;
        if (turn < kRaces) {
          pl = win.logit;
          pi = win.index;
          continue;
        }
        what = kLogit;
        lo = key_of(pl);
        hi = key_of(top);
      } else if (what == kLogit) {
        if (kept) hi = lo + (hi - lo) / 2;  // the position before every token of this logit
        else lo += (hi - lo) / 2 + 1;
      } else if (what == kIndex) {
        if (kept) lo += (hi - lo + 1) / 2;
        else hi = lo + (hi - lo + 1) / 2 - 1;
      } else {
        win = best.index == INT32_MAX ? leader : best;
        break;
      }
      if (what == kLogit && lo == hi) {  // every token before the first of this logit is kept
        what = kIndex;
        pl = logit_of(lo);
        lo = 0;
        hi = (uint32_t)V - 1;
      }
      if (what == kIndex && lo == hi) what = kLast;
      if (what == kLogit) pl = logit_of(lo + (hi - lo) / 2), pi = -1;
      if (what == kIndex) pi = (int)(lo + (hi - lo + 1) / 2);
      if (what == kLast) pi = (int)lo + 1;  // up to and with index lo
    }
  }
  if (rank == 0 && tid == 0) {
    if (win.index == INT32_MAX) win = Best{0.f, top, first};  // greedy, or no score compares
    a.token[row] = win.index;
    a.prob[row] = greedy ? 1.f : (win.logit == top ? 1.f : expf((win.logit - top) / temp)) / Z;
  }
  meet();
}

template <class T, bool VEC>
int sample_launch(const KdnSampleArgs& a, cudaStream_t st) {
  // A CTA per 16384 tokens; more while the rows alone leave SMs idle and every
  // CTA still has 2048 tokens.
  int64_t ctas = (a.V + kSmChunk - 1) / kSmChunk;
  while (2 * ctas <= kSmCluster && 2 * ctas * a.rows <= 296 && a.V / (2 * ctas) >= 2048) ctas *= 2;
  if (ctas > kSmCluster) ctas = kSmCluster;
  const int64_t chunk = ((a.V + ctas - 1) / ctas + 7) / 8 * 8;
  const int64_t group = kSmThreads * Chunk<T, VEC>::kPer, most = kSmHeld / (group * (int64_t)sizeof(T));
  const int64_t need = (chunk + group - 1) / group, groups = need < most ? need : most;
  const size_t smem = (size_t)(groups * group) * sizeof(T);
  if (smem > 40 * 1024) {
    const cudaError_t err = cudaFuncSetAttribute(sample_kernel<T, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (err != cudaSuccess) {
      cudaGetLastError();
      return set_error(KDN_ERR_CUDA, "sample_kernel: %s", cudaGetErrorString(err));
    }
  }
  float fraction = 32768.f;  // units of the histogram: a bin of a CTA's tokens fits 31 bits
  while (fraction > 1.f && fraction * (float)chunk > 2147483648.f) fraction *= 0.5f;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.rows * ctas));
  cfg.blockDim = dim3(kSmThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, sample_kernel<T, VEC>, a, (int)ctas, (int)chunk, (int)groups, fraction);
  if (err != cudaSuccess) {
    cudaGetLastError();
    return set_error(KDN_ERR_CUDA, "sample_kernel: %s", cudaGetErrorString(err));
  }
  return KDN_OK;
}

}  // namespace
}  // namespace kdn

using namespace kdn;

extern "C" {

size_t kdn_sample_workspace_bytes(int64_t rows, int64_t V) {
  (void)rows;
  (void)V;
  return 0;
}

int kdn_sample(const KdnSampleArgs* args, kdn_stream_t stream) {
  if (!args) return set_error(KDN_ERR_INVALID, "kdn_sample: null args");
  const KdnSampleArgs& a = *args;
  if (a.rows < 0 || a.rows > INT32_MAX / kSmCluster || a.V < 1 || a.V > INT32_MAX - (1 << 16))
    return set_error(KDN_ERR_INVALID, "kdn_sample: 0 <= rows < 2^28 and 1 <= V < 2^31 - 2^16 required");
  if (a.rows == 0) return KDN_OK;
  if (!a.logits || !a.noise || !a.token || !a.prob) return set_error(KDN_ERR_INVALID, "kdn_sample: null pointer");
  if (a.rows > 1 && (a.logits_stride < a.V || a.noise_stride < a.V))
    return set_error(KDN_ERR_INVALID, "kdn_sample: row strides smaller than the rows");
  const int64_t elem = a.logits_bf16 ? 2 : 4;
  const bool vec = ((reinterpret_cast<uintptr_t>(a.logits) | (uintptr_t)(a.rows > 1 ? a.logits_stride * elem : 0)) & 15) == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (a.logits_bf16) return vec ? sample_launch<bf16, true>(a, st) : sample_launch<bf16, false>(a, st);
  return vec ? sample_launch<float, true>(a, st) : sample_launch<float, false>(a, st);
}

}  // extern "C"
