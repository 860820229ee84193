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
//  2. sums Z and fills a histogram of e over 1/16 octaves (the bins are the
//     leading bits of the float e).  A bin's entry is the whole-number sum of
//     its tokens' mantissas: it bounds their count from both sides and gives
//     their mass, so that tokens behind `cut` are certainly dropped and those
//     before `safe` certainly within top-k and top-p,
//  3. races the tokens before `cut` (only their random numbers are read).  A
//     winner before `safe` is the answer.  Otherwise the exact count and mass
//     ahead of it are taken; if it is not kept, the tokens ahead of it race.
// Every race lost drops the winner and what is behind it; after kRaces of them
// (noise that follows the logits) the end of the kept prefix is bisected
// instead, so that no row takes more than kRaces + 64 turns.  Rows without
// top-k and top-p race in step 2.  Sums have a fixed order or are integers, so
// that equal calls give equal results; the order of Z follows the split into
// CTAs, which the number of rows decides, and the rows' alignment.
//
// One row of 32000 bf16 logits 10.5 us, 61 rows 16.6, 128 rows of 131072 49
// (unfiltered 35, greedy 22): the latency of the copy, of three cluster-wide
// reductions and of the random numbers, twice for large rows (two waves), and
// the passes' instructions; the logits' bytes alone would take 5 us of the 49.
// Rows of which eight CTAs hold only a part (more than 786432 bf16 or 393216
// fp32 logits) read the rest again in every pass: 32 rows of 800000 bf16 logits
// 119 us unfiltered (23 by bytes), 84 top-k 50, 186 top-p 0.9; one row 41.
#include <cooperative_groups.h>

#include "kdn_launch.cuh"

namespace kdn {
namespace {

namespace cg = cooperative_groups;

constexpr int kSmThreads = 512, kSmWarps = kSmThreads / 32;
constexpr int kSmChunk = 64 * 1024;  // bytes of a row per CTA before it gets another one
constexpr int kSmHeld = 192 * 1024;  // bytes of shared memory for them; what a chunk has beyond is read again in every pass
constexpr int kSmCluster = 8;
constexpr int kRaces = 12;
constexpr float kLargest = 3.402823466e38f;
constexpr float kColdest = 1e-37f;  // log2(e) / T is finite from here on; what is below (0, negative, NaN) is greedy
constexpr int kBins = 1024;      // e from 1 down to 2^-64
constexpr int kBinShift = 23 - 4;  // 16 bins per octave
constexpr uint32_t kOne = 0x3f800000u;  // the bits of e = 1

struct Best {  // a race's leader: the larger score, then the lower index; score 0: nobody
  float score, logit;
  int index;
};
__device__ __forceinline__ bool ahead(float la, int ia, float lb, int ib) { return la > lb || (la == lb && ia < ib); }
// over the warp's lanes; scores are not negative, so their bits are in order
__device__ __forceinline__ Best warp_best(const Best& b) {
  const uint32_t bits = __float_as_uint(b.score), most = __reduce_max_sync(~0u, bits);
  const uint32_t index = bits == most ? (uint32_t)b.index : ~0u, low = __reduce_min_sync(~0u, index);
  const int lane = __ffs(__ballot_sync(~0u, index == low)) - 1;
  return Best{__uint_as_float(most), __shfl_sync(~0u, b.logit, lane), (int)low};
}
// What a reduction carries beside it.
struct Part {
  Best best;
  float mass;
  int count;
};

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
  bool infinite = false;    // +inf is among the row's logits: it counts as the largest finite value
  T* held;

  // +inf becomes the largest finite value; NaN stays NaN (fminf would return the number beside it)
  __device__ __forceinline__ static float finite(float v) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(v), "f"(kLargest));
    return d;
  }
  __device__ __forceinline__ int first(int j) const { return begin + (j * kSmThreads + (int)threadIdx.x) * kPer; }
  // place of this thread's group j; fp32 vectors are split over two planes
  __device__ __forceinline__ T* place(int j) const {
    return held + (size_t)(VEC && sizeof(T) == 4 ? 2 * j * kSmThreads * 4 + threadIdx.x * 4
                                                 : (j * kSmThreads + threadIdx.x) * kPer);
  }
  __device__ __forceinline__ void request() {
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
  }
  // f(logits, first index) for this thread's groups, in a fixed order (past the end: -inf).  first index: begin and a
  // multiple of kPer
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
#pragma unroll 1
    for (int j = 0; j < groups; ++j) {
      const T* at = place(j);
      float v[kPer];
      if constexpr (!VEC) {
        v[0] = to_f(*at);
      } else if constexpr (sizeof(T) == 2) {
        ld8(v, at);
      } else {
        const float4 p = *reinterpret_cast<const float4*>(at), q = *reinterpret_cast<const float4*>(at + kSmThreads * 4);
        v[0] = p.x; v[1] = p.y; v[2] = p.z; v[3] = p.w; v[4] = q.x; v[5] = q.y; v[6] = q.z; v[7] = q.w;
      }
      if (infinite)
#pragma unroll
        for (int k = 0; k < kPer; ++k) v[k] = finite(v[k]);
      f(v, first(j));
    }
    // what does not fit: further groups of the same shape, so that f meets the same alignments
#pragma unroll 1
    for (int i = first(groups); i < end; i += kSmThreads * kPer) {
      float v[kPer];
      if (VEC && i + kPer <= end) {
        if constexpr (VEC) ld8(v, row + i);
      } else {
#pragma unroll
        for (int k = 0; k < kPer; ++k) v[k] = i + k < end ? to_f(row[i + k]) : -INFINITY;
      }
      if (infinite)
#pragma unroll
        for (int k = 0; k < kPer; ++k) v[k] = finite(v[k]);
      f(v, i);
    }
  }
};

// Keys of the largest logit and of two lower bounds: every thread (every warp)
// holds a token at or above the smallest of the threads' (warps') maxima.
struct Tops {
  uint32_t most, least_thread, least_warp;
};
__device__ __forceinline__ Tops warp_tops(const Tops& t) {
  return Tops{__reduce_max_sync(~0u, t.most), __reduce_min_sync(~0u, t.least_thread), __reduce_min_sync(~0u, t.least_warp)};
}

struct Shared {
  Part warps[kSmWarps], ctas[2][kSmCluster];
  Tops warp_tops[kSmWarps], cta_tops[kSmCluster];
  uint32_t hist[kBins];
  int least[kSmWarps], most[kSmWarps];  // of a scan: the counts' bounds
  float scan[kSmWarps];
  int cut[kSmWarps], safe[kSmWarps];
};

__device__ __forceinline__ Part warp_part(Part p) {
  p.best = warp_best(p.best);
  p.mass = warp_sum(p.mass);
  p.count = __reduce_add_sync(~0u, p.count);
  return p;
}

template <class T, bool VEC>
__global__ void __launch_bounds__(kSmThreads, 2) sample_kernel(const __grid_constant__ KdnSampleArgs a, int ctas,
                                                              int chunk, int groups, int down) {
  __shared__ __align__(16) Shared sh;
  extern __shared__ uint4 held[];
  cg::cluster_group cluster = cg::this_cluster();
  using Tokens = Chunk<T, VEC>;
  constexpr int PER = Tokens::kPer;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = (int)a.V;
  const int64_t row = blockIdx.x / ctas;
  const int rank = (int)(blockIdx.x % ctas);
  const Best nobody{0.f, -INFINITY, INT32_MAX};
  const Part nothing{nobody, 0.f, 0};
  int buf = 0;
  // Over all threads of the cluster, in the same order in each of them: lanes,
  // warps, then CTAs, which write their part into each other's memory.
  auto reduce = [&](Part p) {
    p = warp_part(p);
    if (lane == 0) sh.warps[warp] = p;
    __syncthreads();
    if (ctas == 1) {
      p = warp_part(lane < kSmWarps ? sh.warps[lane] : nothing);
      __syncthreads();  // the entries may be written again
      return p;
    }
    if (warp == 0) {
      p = warp_part(lane < kSmWarps ? sh.warps[lane] : nothing);
      if (lane < ctas) *cluster.map_shared_rank(&sh.ctas[buf][rank], lane) = p;
    }
    cluster.sync();
    p = warp_part(lane < ctas ? sh.ctas[buf][lane] : nothing);
    buf ^= 1;
    return p;
  };
  // The CTAs write into each other's memory: all of them have to have started.  Waited for before the first write.
  if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  Tokens c;
  c.row = static_cast<const T*>(a.logits) + row * a.logits_stride;
  c.begin = (int)min((int64_t)rank * chunk, (int64_t)V);
  c.end = (int)min((int64_t)c.begin + chunk, (int64_t)V);
  c.groups = groups;
  c.held = reinterpret_cast<T*>(held);
  c.request();
  const float temp = a.temperature ? a.temperature[row] : a.temperature_all;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_all, min_p = a.min_p ? a.min_p[row] : a.min_p_all;
  int64_t limit = !a.top_k ? a.top_k_all
                  : a.top_k_i64 ? static_cast<const int64_t*>(a.top_k)[row]
                                : (int64_t) static_cast<const int32_t*>(a.top_k)[row];
  const int top_k = limit <= 0 || limit > V ? V : (int)limit;
  const bool greedy = !(temp >= kColdest), by_rank = !greedy && (top_k < V || top_p < 1.f);
  const float* E = a.noise + row * a.noise_stride;
  for (int i = tid; i < kBins; i += kSmThreads) sh.hist[i] = 0;
  cp_async_wait_all();

  // ---- 1: the maximum ----
  float m = -INFINITY;
  c.each([&](const float (&v)[PER], int) {
#pragma unroll
    for (int k = 0; k < PER; ++k) m = fmaxf(m, v[k]);  // passes over NaN
  });
  Tops tops{key_of(m), key_of(m), ~0u};
  tops = warp_tops(tops);
  tops.least_warp = tops.most;
  if (lane == 0) sh.warp_tops[warp] = tops;
  __syncthreads();
  const Tops none{0u, ~0u, ~0u};
  if (ctas == 1) {
    tops = warp_tops(lane < kSmWarps ? sh.warp_tops[lane] : none);
  } else {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (warp == 0) {
      tops = warp_tops(lane < kSmWarps ? sh.warp_tops[lane] : none);
      if (lane < ctas) *cluster.map_shared_rank(&sh.cta_tops[rank], lane) = tops;
    }
    cluster.sync();
    tops = warp_tops(lane < ctas ? sh.cta_tops[lane] : none);
  }
  float top = logit_of(tops.most);
  // with that many threads or warps, a token below their bound is not among the first top_k
  float floor_l = by_rank && top_k <= kSmWarps * ctas     ? logit_of(tops.least_warp)
                  : by_rank && top_k <= kSmThreads * ctas ? logit_of(tops.least_thread)
                                                          : -INFINITY;
  c.infinite = top == INFINITY;
  if (c.infinite) top = kLargest, floor_l = fminf(floor_l, kLargest);

  // ---- 2: Z, and the histogram or the only race ----
  // e = 2^-t, t = (top - l) log2(e) / T in two terms, neither negative (T = inf: both 0, an even draw); -inf gives t = inf
  // or, where a term is 0, NaN: e = 0 both ways
  const float scale = __fdiv_rd(1.4426950408889634f, temp);
  const float rest = fmaxf(fmaf(-scale, temp, 1.4426950408889634f) / temp, 0.f);
  auto weight = [&](float l) { return fmaxf(ex2a(-fmaf(top - l, scale, (top - l) * rest)), 0.f); };
  // the random numbers of a group: one 32-byte sector, in one round trip (VEC: begin, and with it i, is a multiple of 8)
  const bool noise16 = (reinterpret_cast<uintptr_t>(E) & 15) == 0;
  auto draw = [&](float (&noise)[PER], int i) {
    if (PER == 8 && noise16 && i + 8 <= c.end) {
      const float4 p = __ldg(reinterpret_cast<const float4*>(E + i)), q = __ldg(reinterpret_cast<const float4*>(E + i + 4));
      noise[0] = p.x; noise[1 % PER] = p.y; noise[2 % PER] = p.z; noise[3 % PER] = p.w;
      noise[4 % PER] = q.x; noise[5 % PER] = q.y; noise[6 % PER] = q.z; noise[7 % PER] = q.w;
    } else {
#pragma unroll
      for (int k = 0; k < PER; ++k) noise[k] = i + k < c.end ? __ldg(E + i + k) : 1.f;
    }
  };
  Best best = nobody;
  auto enter = [&](float e, float noise, float l, int i) {  // a thread's indexes grow: ties stay with the first
    const float score = __fdividef(e, noise);
    if (score > best.score) best = Best{score, l, i};
  };
  float Z = 0.f;
  if (!greedy && top > -INFINITY) {
    c.each([&](const float (&v)[PER], int i) {
      float e[PER];
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        e[k] = weight(v[k]);
        Z += e[k];
      }
      if (by_rank) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const uint32_t u = __float_as_uint(e[k]) - 1, bin = (kOne - 1 - u) >> kBinShift;
          if (bin < kBins && v[k] >= floor_l) atomicAdd(&sh.hist[bin], ((u & 0x7fffffu) | 0x800000u) >> (8 + down));
        }
      } else {
        float noise[PER];
        draw(noise, i);
#pragma unroll
        for (int k = 0; k < PER; ++k)
          if (e[k] >= min_p) enter(e[k], noise[k], v[k], i + k);
      }
    });
  }
  const Part second = reduce(Part{best, Z, 0});
  Z = second.mass;
  Best win = second.best;

  // ---- 3: races among the tokens before `cut` ----
  if (by_rank && top > -INFINITY) {
    // this thread's two bins over the cluster: bounds of their counts, their mass
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int r = 0; r < kSmCluster; ++r)
      if (r < ctas) {
        const uint2 u = *reinterpret_cast<const uint2*>((ctas == 1 ? sh.hist : cluster.map_shared_rank(sh.hist, r)) + 2 * tid);
        sum[0] += (float)u.x;
        sum[1] += (float)u.y;
      }
    int least[2], most[2];
    float mass[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {  // 1e-6 covers the roundings of sum and quotient
      const uint32_t u = kOne - 1 - ((uint32_t)(2 * tid + b) << kBinShift);  // the largest of the bin
      const uint32_t high = ((u & 0x7fffffu) | 0x800000u) >> (8 + down), low = (high + 1) - (1u << (kBinShift - 8 - down));
      least[b] = (int)ceilf(__fdividef(sum[b], (float)high) * (1.f - 1e-6f));
      most[b] = (int)(__fdividef(sum[b], (float)low) * (1.f + 1e-6f));
      mass[b] = sum[b] * __uint_as_float(((u >> 23) - 15 + down) << 23);  // units of 2^(exponent - 15 + down)
    }
    int pl_ = least[0] + least[1], pm_ = most[0] + most[1];  // inclusive scans over the threads
    float ps_ = mass[0] + mass[1];
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {  // (rolled up: the code is run once, and its instructions come from memory)
      const int x = __shfl_up_sync(~0u, pl_, o), y = __shfl_up_sync(~0u, pm_, o);
      const float f = __shfl_up_sync(~0u, ps_, o);
      if (lane >= o) pl_ += x, pm_ += y, ps_ += f;
    }
    if (lane == 31) sh.least[warp] = pl_, sh.most[warp] = pm_, sh.scan[warp] = ps_;
    __syncthreads();
    const bool before = lane < warp;  // warps in front (lane < 16)
    pl_ += __reduce_add_sync(~0u, before ? sh.least[lane] : 0);
    pm_ += __reduce_add_sync(~0u, before ? sh.most[lane] : 0);
    ps_ += warp_sum(before ? sh.scan[lane] : 0.f);
    // Entries are rounded down by less than one in 2^15 >> down; 1e-5 covers the sums' own rounding.
    const float goal = top_p < 1.f ? top_p * Z : INFINITY, over = 1.f + (float)(1 << down) / 16384.f + 1e-5f;
    int cut = kBins, safe = 0;
    // least and mass ahead of the thread's first and second bin; most and mass up to and with them
    if (pl_ - least[1] >= top_k || (ps_ - mass[1]) * (1.f - 1e-5f) >= goal) cut = 2 * tid + 1;
    if (pl_ - least[1] - least[0] >= top_k || (ps_ - mass[1] - mass[0]) * (1.f - 1e-5f) >= goal) cut = 2 * tid;
    if (pm_ - most[1] <= top_k && (ps_ - mass[1]) * over < goal) safe = 2 * tid + 1;
    if (pm_ <= top_k && ps_ * over < goal) safe = 2 * tid + 2;
    cut = __reduce_min_sync(~0u, cut);
    safe = __reduce_max_sync(~0u, safe);
    if (lane == 0) sh.cut[warp] = cut, sh.safe[warp] = safe;
    __syncthreads();
    cut = __reduce_min_sync(~0u, sh.cut[lane % kSmWarps]);
    safe = __reduce_max_sync(~0u, sh.safe[lane % kSmWarps]);
    // tokens of bins before b have e above these
    // tokens below floor_l are not in the histogram: they are dropped, and nothing above it has one ahead
    const float e_floor = floor_l > -INFINITY ? weight(floor_l) : 0.f;
    const float e_cut = fmaxf(cut == kBins ? 0.f : __uint_as_float(kOne - ((uint32_t)cut << kBinShift)),
                              e_floor > 0.f ? __uint_as_float(__float_as_uint(e_floor) - 1) : 0.f);
    const float e_safe = fmaxf(__uint_as_float(kOne - ((uint32_t)safe << kBinShift)), fmaxf(e_cut, e_floor));

    // What a turn looks at lies ahead of (pl, pi) in the order.
    float pl = -INFINITY;
    int pi = INT32_MAX;
    // bisection: the last kept logit is in [lo, hi] (keys), then the last kept index of it
    enum { kRace, kLogit, kIndex, kLast } what = kRace;
    uint32_t lo = 0, hi = 0;
    for (int turn = 0;; ++turn) {
      best = nobody;
      float weights = 0.f;
      int count = 0;
      c.each([&](const float (&v)[PER], int i) {
        float most_l = v[0];
#pragma unroll
        for (int k = 1; k < PER; ++k) most_l = fmaxf(most_l, v[k]);
        if (most_l < pl || !(weight(most_l) > e_cut)) return;
        float noise[PER];
        draw(noise, i);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const float e = weight(v[k]);
          if (e > e_cut && ahead(v[k], i + k, pl, pi)) {
            weights += e;
            ++count;
            if (e >= min_p) enter(e, noise[k], v[k], i + k);
          }
        }
      });
      const Part part = reduce(Part{best, weights, count});
      best = part.best;
      weights = part.mass;
      count = part.count;
      // whether a token at (pl, pi) is within top-k and top-p (the order's first always is)
      const bool kept = turn > 0 && (count == 0 || (count < top_k && (top_p >= 1.f || weights < top_p * Z)));
      if (what == kRace) {
        if (kept) break;  // (pl, pi) is the winner
        win = best;
        if (win.score == 0.f || weight(win.logit) > e_safe) break;
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
        win = best;
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

  // greedy, or nobody's score compares: the order's first token
  if (win.score == 0.f && top > -INFINITY) {
    int first = INT32_MAX;
    c.each([&](const float (&v)[PER], int i) {
#pragma unroll
      for (int k = PER - 1; k >= 0; --k)
        if (v[k] == top) first = min(first, i + k);
    });
    win = reduce(Part{Best{first < INT32_MAX ? 1.f : 0.f, top, first}, 0.f, 0}).best;
  }
  if (rank == 0 && tid == 0) {
    const bool empty = top == -INFINITY;
    a.token[row] = empty ? -1 : win.index;
    a.prob[row] = empty ? 0.f : greedy ? 1.f : expf((win.logit - top) / temp) / Z;
  }
  if (ctas > 1) cluster.sync();  // nobody leaves while its memory may be read
}

template <class T, bool VEC>
int sample_launch(const KdnSampleArgs& a, cudaStream_t st) {
  // A CTA per 64 KB (128 rows of 131072 bf16 logits, mixed filters: 49 us, 32 KB 62 us); more while the rows alone
  // leave SMs idle and every CTA still has 2048 tokens.
  int64_t ctas = (a.V * (int64_t)sizeof(T) + kSmChunk - 1) / kSmChunk;
  while (2 * ctas <= kSmCluster && 2 * ctas * a.rows <= 296 && a.V / (2 * ctas) >= 2048) ctas *= 2;
  if (ctas > kSmCluster) ctas = kSmCluster;
  const int64_t chunk = ((a.V + ctas - 1) / ctas + 7) / 8 * 8;
  const int64_t group = kSmThreads * Chunk<T, VEC>::kPer, most = kSmHeld / (group * (int64_t)sizeof(T));
  const int64_t need = (chunk + group - 1) / group, groups = need < most ? need : most;
  const size_t smem = (size_t)(groups * group) * sizeof(T);
  if (int rc = allow_smem<sample_kernel<T, VEC>>(kSmHeld, "sample_kernel")) return rc;
  int down = 0;  // a bin's entry, below 2^16 >> down per token, fits 32 bits
  while ((chunk << 16 >> down) >> 32) ++down;
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
  const cudaError_t err = cudaLaunchKernelEx(&cfg, sample_kernel<T, VEC>, a, (int)ctas, (int)chunk, (int)groups, down);
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

int kdn_sample(const KdnSampleArgs* args, kdn_stream_t stream) {
  if (!args) return set_error(KDN_ERR_INVALID, "kdn_sample: null args");
  const KdnSampleArgs& a = *args;
  if (a.rows < 0 || a.rows > INT32_MAX / kSmCluster || a.V < 1 || a.V > (1 << 29))
    return set_error(KDN_ERR_INVALID, "kdn_sample: 0 <= rows < 2^28 and 1 <= V <= 2^29 required");
  if (a.rows == 0) return KDN_OK;
  if (!a.logits || !a.noise || !a.token || !a.prob) return set_error(KDN_ERR_INVALID, "kdn_sample: null pointer");
  auto bad = [&](int64_t stride) { return stride < a.V && stride != 0; };  // 0: one row for all
  if (a.rows > 1 && (bad(a.logits_stride) || bad(a.noise_stride)))
    return set_error(KDN_ERR_INVALID, "kdn_sample: row strides smaller than the rows");
  const int64_t elem = a.logits_bf16 ? 2 : 4;
  const bool vec = ((reinterpret_cast<uintptr_t>(a.logits) | (uintptr_t)(a.rows > 1 ? a.logits_stride * elem : 0)) & 15) == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (a.logits_bf16) return vec ? sample_launch<bf16, true>(a, st) : sample_launch<bf16, false>(a, st);
  return vec ? sample_launch<float, true>(a, st) : sample_launch<float, false>(a, st);
}

}  // extern "C"
