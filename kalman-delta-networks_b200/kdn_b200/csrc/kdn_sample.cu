// One token per row of logits under temperature, top-k, top-p and min-p, from
// given Exp(1) random numbers.  With e_i = exp((l_i - max) / T), Z = sum e and
// the order "larger logit first, then lower index", the filters keep a prefix
// of the order: rank < top_k, (sum of e ahead) < top_p Z, e >= min_p.  The
// token is the kept one with the largest e_i / noise_i: with independent
// exponential noise it is drawn with probability e_i / (sum of the kept e).
//
// Because the kept set is a prefix, no sort is needed: take the best token of
// the race, count the tokens and the mass ahead of it, and if it is not kept,
// race again among the tokens ahead of it.  Every round shortens the prefix;
// the order's first token is always kept, so the rounds end.
#include "kdn_common.cuh"

namespace kdn {
namespace {

constexpr int kSampleThreads = 1024;

struct Best {  // a race's leader: the larger score, then the earlier in the order
  float score, logit;
  int index;
};

__device__ __forceinline__ bool ahead(float la, int ia, float lb, int ib) { return la > lb || (la == lb && ia < ib); }
__device__ __forceinline__ bool beats(const Best& a, const Best& b) {
  return a.score > b.score || (a.score == b.score && ahead(a.logit, a.index, b.logit, b.index));
}

template <class T>
__device__ __forceinline__ float logit_at(const T* p, int i) {
  const float l = to_f(p[i]);
  return isnan(l) ? -INFINITY : l;
}

template <class T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const __grid_constant__ KdnSampleArgs a) {
  __shared__ float sf[2][32];
  __shared__ int si[2][32];
  __shared__ Best sb[32];
  const int64_t row = blockIdx.x;
  const int V = (int)a.V, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* L = static_cast<const T*>(a.logits) + row * a.logits_stride;
  const float* E = a.noise + row * a.noise_stride;
  const float T_ = a.temperature ? a.temperature[row] : a.temperature_all;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_all, min_p = a.min_p ? a.min_p[row] : a.min_p_all;
  int64_t top_k = !a.top_k ? a.top_k_all
                  : a.top_k_i64 ? static_cast<const int64_t*>(a.top_k)[row]
                                : (int64_t) static_cast<const int32_t*>(a.top_k)[row];
  if (top_k <= 0 || top_k > V) top_k = V;

  // the order's first token
  Best first{0.f, -INFINITY, INT32_MAX};
  for (int i = tid; i < V; i += kSampleThreads) {
    const float l = logit_at(L, i);
    if (ahead(l, i, first.logit, first.index)) first.logit = l, first.index = i;
  }
  auto reduce_best = [&](Best b) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Best c{__shfl_xor_sync(~0u, b.score, o), __shfl_xor_sync(~0u, b.logit, o), __shfl_xor_sync(~0u, b.index, o)};
      if (beats(c, b)) b = c;
    }
    __syncthreads();  // the previous reader of sb is done
    if (lane == 0) sb[warp] = b;
    __syncthreads();
    b = sb[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Best c{__shfl_xor_sync(~0u, b.score, o), __shfl_xor_sync(~0u, b.logit, o), __shfl_xor_sync(~0u, b.index, o)};
      if (beats(c, b)) b = c;
    }
    return b;
  };
  first = reduce_best(first);
  const float top = first.logit;
  if (top == -INFINITY) {
    if (tid == 0) a.token[row] = -1, a.prob[row] = 0.f;
    return;
  }
  if (!(T_ > 0.f)) {
    if (tid == 0) a.token[row] = first.index, a.prob[row] = 1.f;
    return;
  }
  auto weight = [&](float l) { return l == top ? 1.f : expf((l - top) / T_); };

  // race over the tokens ahead of (pl, pi); rounds end when the winner is kept
  float pl = -INFINITY, Z = 0.f;
  int pi = INT32_MAX;
  Best win = first;
  for (int round = 0;; ++round) {
    Best best{-1.f, -INFINITY, INT32_MAX};
    float mass = 0.f;
    int count = 0;
    for (int i = tid; i < V; i += kSampleThreads) {
      const float l = logit_at(L, i);
      if (!ahead(l, i, pl, pi)) continue;
      const float e = weight(l);
      mass += e;
      ++count;
      if (!(e > 0.f)) continue;
      const Best b{e / E[i], l, i};
      if (beats(b, best)) best = b;
    }
    mass = warp_sum(mass);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) count += __shfl_xor_sync(~0u, count, o);
    const int buf = round & 1;
    if (lane == 0) sf[buf][warp] = mass, si[buf][warp] = count;
    best = reduce_best(best);  // its barriers publish sf and si
    mass = warp_sum(sf[buf][lane]);
    count = si[buf][lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) count += __shfl_xor_sync(~0u, count, o);
    if (round == 0) {
      Z = mass;
    } else {
      // (pl, pi) = win: is it kept?
      const bool kept = (win.index == first.index && win.logit == top) ||
                        (count < top_k && (top_p >= 1.f || mass < top_p * Z) && weight(win.logit) >= min_p);
      if (kept) break;
    }
    // the next candidate; without one (no score compares) the first token
    win = best.index == INT32_MAX ? first : best;
    pl = win.logit;
    pi = win.index;
  }
  if (tid == 0) a.token[row] = win.index, a.prob[row] = weight(win.logit) / Z;
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
  if (a.rows < 0 || a.rows > INT32_MAX || a.V < 1 || a.V > INT32_MAX - kSampleThreads)
    return set_error(KDN_ERR_INVALID, "kdn_sample: rows >= 0 and 1 <= V < 2^31 - 1024 required");
  if (a.rows == 0) return KDN_OK;
  if (!a.logits || !a.noise || !a.token || !a.prob) return set_error(KDN_ERR_INVALID, "kdn_sample: null pointer");
  if (a.rows > 1 && (a.logits_stride < a.V || a.noise_stride < a.V))
    return set_error(KDN_ERR_INVALID, "kdn_sample: row strides smaller than the rows");
  cudaStream_t st = (cudaStream_t)stream;
  if (a.logits_bf16)
    sample_kernel<bf16><<<(unsigned)a.rows, kSampleThreads, 0, st>>>(a);
  else
    sample_kernel<float><<<(unsigned)a.rows, kSampleThreads, 0, st>>>(a);
  return check_launch("sample_kernel");
}

}  // extern "C"
