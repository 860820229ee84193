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
// consecutive values per thread and slot) and walks several rows, so that each
// thread keeps its columns' weight-gradient sums in registers; dscale and
// dpost share one sum, sum Z s yh, because the weights are factors of whole
// columns.  The coming rows are copied into a ring in shared memory
// (cp.async), which keeps enough bytes in flight without holding registers.
// Rows of odd widths in contiguous tensors are worked on as the aligned words
// that cover them, rows of other strides and alignments are copied so and
// shifted when they are read (BnRows).  The groups' sums are
// added in a fixed order by a second kernel.
//
// 16384 x 2304 bf16: all parts 68 us forward (5.5 TB/s) and 114 us backward
// (5.3 TB/s, the second kernel included), the plain sum 55 and 88 us; with an
// fp32 stream 99 / 153 and 85 / 126 us.  8192 x 2304 bf16 39 / 67, 8192 x 2305
// 57 / 97 (four warps a row instead of three, and the outer vectors).
#pragma once

#include "kdn_launch.cuh"

namespace kdn {
namespace {

constexpr int kBnVec = 8;       // values per thread and slot, worked on as pairs
constexpr int kBnMaxD = 8192;
constexpr int kBnMinD = 2;  // the norm of one value is its sign: fp32 cannot resolve its gradient (of the order of eps)
// A row belongs to the fewest warps whose lanes hold it in three slots each:
// what a row costs beside its values (reductions, addresses, barriers) is paid
// per warp.  The backward of loose rows (see BnRows) takes as few slots as the
// CTA's warps allow instead: every slot's shifts are code of its own, more of it
// than registers and instruction fetch bear (rows of 1155 fp32 values, 1000 of
// them: 31 us against 39; 8192 of 2305 bf16: 203 against 218; the forward loses,
// 125 us against 79).  One CTA per SM with as many rows at a time as its warps
// make: 12 warps (168 registers a thread), in the forward of loose rows, which
// wait at a barrier per row, 16.
constexpr int kBnFwdWarps = 16, kBnBwdWarps = 12, kBnSlots = 3;
constexpr size_t kBnSmem = 232448;  // a CTA's shared memory; fp32 rows of 8192 values and their weights fit once

struct BnGeom {
  int slots;  // slots per thread: 1, 2 or 3
  int tpr;    // threads per row
  int rpb;    // rows per CTA at a time
  int period;  // rows from one to the next of the same shift
  unsigned grid;
};

// How the rows of a call lie in memory.  Aligned: every row starts on a 16-byte
// boundary and is a whole number of vectors.  Packed: rows of another width, in
// tensors that are contiguous and aligned as a whole.  A row's vectors are then
// the aligned words of memory that cover it, its first column `shift` places
// into the first one, and rows a `period` apart have the same shift: a CTA takes
// rows of one shift only, so that its weights and its columns' sums are those of
// aligned rows, moved by it; only the outer vectors of a row differ (what they
// hold of the neighbours is cleared in shared memory, their values are stored
// one by one).  Loose: any other strides and alignments, every vector shifted
// when it is read and when it is stored.  8192 x 2305 bf16, all parts: packed 57
// us forward and 97 backward, loose 80 and 204; 1000 x 1155 fp32: 12.5 and 25,
// loose 12.5 and 31.
enum BnRows { kBnLoose = 0, kBnAligned = 1, kBnPacked = 2 };

// vectors of a row (packed: of the rows with the largest shift)
__host__ __device__ inline int bn_vectors(int D, bool packed) {
  return packed && D % kBnVec ? (D + 2 * kBnVec - 2) / kBnVec : (D + kBnVec - 1) / kBnVec;
}

inline BnGeom bn_geom(int64_t rows, int64_t D, int cta_warps, BnRows kind, bool few_slots) {
  BnGeom g;
  const int nv = bn_vectors((int)D, kind == kBnPacked);
  g.slots = !few_slots ? kBnSlots : (nv + 32 * cta_warps - 1) / (32 * cta_warps);
  const int warps = (nv + 32 * g.slots - 1) / (32 * g.slots);
  g.tpr = 32 * warps;
  g.slots = (nv + g.tpr - 1) / g.tpr;
  g.rpb = cta_warps / warps;
  g.period = 1;
  if (kind == kBnPacked)
    while (D * g.period % kBnVec) g.period *= 2;
  const int64_t each = (rows + g.period - 1) / g.period, want = (each + g.rpb - 1) / g.rpb, most = 148 / g.period;
  g.grid = (unsigned)(g.period * (want < most ? (want > 0 ? want : 1) : most));
  return g;
}

struct BnParams {
  KdnBlockNormArgs a;
  float* partial;  // [CTAs][2][D]: sums of dh zh and of Z s yh
  int tpr;
  int period;
  int planes;  // 16-byte pieces of the call's inputs per vector
  int stages;  // of the ring
};

// Arithmetic on pairs of values: Blackwell's packed fp32 instructions take
// half the issue slots, which is what the gated kernels run short of.
__device__ __forceinline__ unsigned long long bits2(float2 v) {
  unsigned long long u;
  asm("mov.b64 %0, {%1, %2};" : "=l"(u) : "f"(v.x), "f"(v.y));
  return u;
}
__device__ __forceinline__ float2 pair2(unsigned long long u) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(u));
  return v;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return pair2(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
  return pair2(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
  return pair2(d);
}

// 1 / (1 + 2^(-x log2 e)) with the hardware's exponential and reciprocal (a few 2^-23 over a gate's range)
__device__ __forceinline__ float2 sigmoid2(float2 x) {
  float2 t = mul2(x, both(-1.4426950408889634f));
  t = add2(make_float2(ex2a(t.x), ex2a(t.y)), both(1.f));
  float2 r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(t.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(t.y));
  return r;
}

enum BnGate { kBnOpen = 0, kBnSigmoid = 1, kBnSwish = 2 };

// f(gate kind), so that the kind is known inside the loops
template <bool FULL, class F>
__device__ __forceinline__ void by_gate(int gate, F&& f) {
  if (!FULL || gate == kBnOpen) f(std::integral_constant<int, kBnOpen>{});
  else if (gate == kBnSigmoid) f(std::integral_constant<int, kBnSigmoid>{});
  else f(std::integral_constant<int, kBnSwish>{});
}

// 8 values as they lie in memory, and the number of 16-byte pieces they fill
template <class T> struct Raw;
template <> struct Raw<bf16> {
  static constexpr int kPlanes = 1;
  uint4 u;
  __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void set(const uint32_t* w) { u = make_uint4(w[0], w[1], w[2], w[3]); }
  __device__ __forceinline__ void cut(int n) {  // values n.. become 0
    uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] &= 2 * i + 1 < n ? 0xffffffffu : 2 * i < n ? 0xffffu : 0u;
    set(w);
  }
  __device__ __forceinline__ float2 operator[](int i) const {  // values 2 i and 2 i + 1
    const uint32_t w = i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w;
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
};
template <> struct Raw<float> {
  static constexpr int kPlanes = 2;
  float v[8];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
  }
  __device__ __forceinline__ void set(const uint32_t* w) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
  }
  __device__ __forceinline__ void cut(int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i >= n) v[i] = 0.f;
  }
  __device__ __forceinline__ float2 operator[](int i) const { return make_float2(v[2 * i], v[2 * i + 1]); }
};

// 16 bytes of which at most n (0 or fewer: none) are read, zeros behind them
__device__ __forceinline__ void cp_async16_part(void* dst, const void* src, int n) {
  n = min(max(n, 0), 16);
  if (n == 0) *static_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
  else
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(n)
                 : "memory");
}
// values outside [lo, n) of a vector in shared memory become 0
template <class T>
__device__ __forceinline__ void clear_outer(const uint4* vector, int lo, int n) {
  T* v = reinterpret_cast<T*>(const_cast<uint4*>(vector));
#pragma unroll
  for (int i = 0; i < kBnVec; ++i)
    if (i < lo || i >= n) v[i] = from_f<T>(0.f);
}

// One input tensor of a call: rows of D values, `stride` apart.  The pieces of
// a row are the 16-byte words of memory that cover it; piece 0 starts up to 15
// bytes before the row.
template <class T, BnRows ROWS>
struct BnSource {
  static constexpr bool ALIGNED = ROWS != kBnLoose;
  const char* base;
  int64_t stride;  // bytes
  int64_t rows;
  int bytes;  // of a row
  __device__ __forceinline__ BnSource(const void* p, int64_t s, int64_t n, int D)
      : base(static_cast<const char*>(p)), stride(s * (int64_t)sizeof(T)), rows(n), bytes(D * (int)sizeof(T)) {}
  __device__ __forceinline__ explicit operator bool() const { return base != nullptr; }
  __device__ __forceinline__ const char* row(int64_t r) const { return base + r * stride; }
  __device__ __forceinline__ static int lead(const char* p) {
    return ALIGNED ? 0 : (int)(reinterpret_cast<uintptr_t>(p) & 15);
  }
  // piece k of the row at p, or what of it belongs to the tensor
  __device__ __forceinline__ bool whole(const char* p, int k) const {
    const char* q = p - lead(p) + 16 * k;
    return ALIGNED || (q >= base && q + 16 <= base + (rows - 1) * stride + bytes);
  }
  __device__ __forceinline__ uint4 part(const char* p, int k) const {
    const char* q = p - lead(p) + 16 * k;
    uint32_t w[4] = {0, 0, 0, 0};
    for (int i = 0; i < 16; i += (int)sizeof(T))
      if (q + i >= base && q + i < base + (rows - 1) * stride + bytes)
        w[i >> 2] |= sizeof(T) == 4 ? *reinterpret_cast<const uint32_t*>(q + i)
                                    : (uint32_t) * reinterpret_cast<const unsigned short*>(q + i) << (8 * (i & 2));
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // Copies this thread's pieces of row r into the ring at dst, piece after
  // piece.  Only the last slot can reach past the row's nv vectors; unaligned
  // rows may reach one piece past them.  Packed rows: from `shift` values before the row, and zeros past the tensor.
  template <int SLOTS>
  __device__ __forceinline__ void copy(int64_t r, uint4* dst, int t, int tpr, int nv, int shift) const {
    constexpr int P = Raw<T>::kPlanes;
    const char* p = row(r) - (ROWS == kBnPacked ? shift * (int)sizeof(T) : 0);
    if (ROWS == kBnPacked && p + 16 * P * nv > base + rows * bytes) {
      const int first = P * (t & ~31) + (t & 31), inside = (int)(base + rows * bytes - p);
#pragma unroll 1
      for (int s = 0; s < SLOTS; ++s)
        for (int k = 0; k < P; ++k) {
          const int piece = first + P * s * tpr + 32 * k;
          if (piece < P * nv) cp_async16_part(dst + piece, p + 16 * piece, inside - 16 * piece);
        }
    } else if (ALIGNED) {
      // a warp's vectors of a slot are 32 P neighbouring pieces: lane by lane, so that each request is one run of memory
      const int first = P * (t & ~31) + (t & 31);
      const char* q = p + 16 * first;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s)
#pragma unroll
        for (int k = 0; k < P; ++k) {
          const int at = P * s * tpr + 32 * k;
          if (s == SLOTS - 1 && first + at >= P * nv) break;
          cp_async16(dst + first + at, q + 16 * at);
        }
    } else {
      const int end = lead(p) + bytes;
      const char* q = p - lead(p);
      // rows whose outer pieces lie inside the tensor: less than 16 bytes outside the row, where its neighbours' starts are
      // 16 or more away (not so with one row for all, stride 0, or rows of a few values)
      const bool inner = stride >= 16 && r > 0 && r < rows - 1;
#pragma unroll
      for (int s = 0; s < P * SLOTS + 1; ++s) {
        const int piece = t + s * tpr;
        if (16 * piece >= end) break;
        if (inner || whole(p, piece)) cp_async16(dst + piece, q + 16 * piece);
        else dst[piece] = part(p, piece);
      }
    }
  }
  // The 8 values of vector v of a row in the ring; n of them are the row's.
  __device__ __forceinline__ void take(Raw<T>& out, int64_t r, const uint4* src, int v, int n) const {
    constexpr int P = Raw<T>::kPlanes;
    uint32_t w[4 * P + 4];
#pragma unroll
    for (int k = 0; k < (ALIGNED ? P : P + 1); ++k) {
      const uint4 q = src[P * v + (k < P || n > 0 ? k : 0)];
      w[4 * k] = q.x;
      w[4 * k + 1] = q.y;
      w[4 * k + 2] = q.z;
      w[4 * k + 3] = q.w;
    }
    if (!ALIGNED) {
      const int b = lead(row(r));
#pragma unroll
      for (int i = 0; i < 4 * P + 2; ++i) w[i] = b & 8 ? w[i + 2] : w[i];
#pragma unroll
      for (int i = 0; i < 4 * P + 1; ++i) w[i] = b & 4 ? w[i + 1] : w[i];
      if (sizeof(T) == 2)
#pragma unroll
        for (int i = 0; i < 4 * P; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 8 * (b & 2));
    }
    out.set(w);
    if (!ALIGNED && n < 8) out.cut(n);
  }
};

// 8 values to an aligned row: one whole 32-byte sector per thread for fp32
__device__ __forceinline__ void st_row(bf16* p, const float (&s)[8]) { st8(p, s); }
__device__ __forceinline__ void st_row(float* p, const float (&s)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(s[0]), "f"(s[1]), "f"(s[2]),
               "f"(s[3]), "f"(s[4]), "f"(s[5]), "f"(s[6]), "f"(s[7])
               : "memory");
}

// The 8 values (n at a row's end) of a vector, as pairs, to an output row.
// Rows of any alignment: a lane stores the aligned 8-value word of memory that
// its values begin in, with the last values of the lane before; what no lane
// holds whole (at a warp's ends and the row's) is stored value by value.  Every
// lane of the warp calls; neighbouring lanes hold neighbouring vectors.
__device__ __forceinline__ void words_of(uint32_t (&w)[4], const float2 (&v)[4], bf16*) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[i].x, v[i].y);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
}
__device__ __forceinline__ void words_of(uint32_t (&w)[8], const float2 (&v)[4], float*) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(i & 1 ? v[i / 2].y : v[i / 2].x);
}
template <BnRows ROWS, class T>
__device__ __forceinline__ void put(T* p, const float2 (&v)[4], int n, int lo) {
  if (ROWS != kBnLoose) {
    const float s[8] = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
    if (ROWS == kBnAligned ? n > 0 : lo == 0 && n == 8) {
      st_row(p, s);
    } else if (ROWS == kBnPacked && n > 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i >= lo && i < n) p[i] = from_f<T>(s[i]);
    }
    return;
  }
  constexpr int W = 2 * sizeof(T);  // 32-bit words of 8 values
  const int lane = threadIdx.x & 31;
  const int e = (int)(reinterpret_cast<uintptr_t>(p) / sizeof(T) & 7);  // values of the word before this vector's
  uint32_t own[W], w[2 * W];
  words_of(own, v, p);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    w[i] = __shfl_up_sync(0xffffffffu, own[i], 1);
    w[W + i] = own[i];
  }
  const int next_n = __shfl_down_sync(0xffffffffu, n, 1);
  const bool whole = n >= 8 - e && (lane > 0 || e == 0), next_whole = lane < 31 && next_n >= 8 - e;
  // the 8 values from position 8 - e of (the lane before's, this lane's)
  const int q = (8 - e) * (int)sizeof(T);  // bytes
#pragma unroll
  for (int k = 16; k >= 4; k /= 2)
    if (k < 4 * W)
#pragma unroll
      for (int i = 0; i < 2 * W - k / 4; ++i) w[i] = q & k ? w[i + k / 4] : w[i];
  if (sizeof(T) == 2)
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 8 * (q & 2));
  if (whole) {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = e ? w[i] : own[i];
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(p - e) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      float s[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = __uint_as_float(w[i]);
      st_row(p - e, s);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n && !(i < 8 - e ? whole : next_whole)) p[i] = from_f<T>(i & 1 ? v[i / 2].y : v[i / 2].x);
}

// weights of 8 columns, those from lo to n (absent: 1; outside the row: 0)
template <BnRows ROWS>
__device__ __forceinline__ void ldw(float2 (&out)[4], const void* p, int col, int n, int lo, bool bf) {
  float d[8];
  if (!p || n <= 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = i >= lo && i < n ? 1.f : 0.f;
  } else if ((ROWS == kBnAligned || (ROWS == kBnLoose && n == 8)) && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    if (bf) ld8(d, static_cast<const bf16*>(p) + col);
    else ld8(d, static_cast<const float*>(p) + col);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      d[i] = i < lo || i >= n ? 0.f : bf ? to_f(static_cast<const bf16*>(p)[col + i]) : static_cast<const float*>(p)[col + i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = make_float2(d[2 * i], d[2 * i + 1]);
}

// The weights of the call in shared memory: [2 or 4][nv + 1] float4, weight first,
// scale * post_weight next (FULL), zero at vector nv.  All row groups of a CTA share them.
template <bool FULL>
constexpr int kWeightPlanes = FULL ? 4 : 2;
template <BnRows ROWS, bool FULL>
__device__ __forceinline__ void stage_weights(float4* dst, const KdnBlockNormArgs& a, int nv, int shift) {
  const bool wb = a.weights_bf16 != 0;
  const int plane = nv + 1;
  for (int v = threadIdx.x; v <= nv; v += blockDim.x) {
    const int col = v * kBnVec - shift, n = min(max((int)a.D - col, 0), kBnVec), lo = max(-col, 0);
    float2 w[4], sc[4];
    ldw<ROWS>(w, a.weight, col, n, lo, wb);
    dst[v] = make_float4(w[0].x, w[0].y, w[1].x, w[1].y);
    dst[plane + v] = make_float4(w[2].x, w[2].y, w[3].x, w[3].y);
    if (!FULL) continue;
    ldw<ROWS>(sc, a.scale, col, n, lo, wb);
    ldw<ROWS>(w, a.post_weight, col, n, lo, wb);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = mul2(w[i], sc[i]);
    dst[2 * plane + v] = make_float4(w[0].x, w[0].y, w[1].x, w[1].y);
    dst[3 * plane + v] = make_float4(w[2].x, w[2].y, w[3].x, w[3].y);
  }
}
__device__ __forceinline__ void recall(float2 (&v)[4], const float4* src, int plane) {
  const float4 p = src[0], q = src[plane];
  v[0] = make_float2(p.x, p.y);
  v[1] = make_float2(p.z, p.w);
  v[2] = make_float2(q.x, q.y);
  v[3] = make_float2(q.z, q.w);
}

// Sums of N values over the threads of a row group (tpr threads, its own
// named barrier); `red` alternates between two buffers from call to call, so
// one barrier per call is enough.  A buffer holds [N][kBnRed] warp sums, zero
// past the group's warps.
constexpr int kBnRed = 16;
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* red, int& phase, int tpr, int group) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if (tpr == 32) return;
  const int t = threadIdx.x - group * tpr, warp = t >> 5;
  float* r = red + phase * N * kBnRed;
  phase ^= 1;
  if ((t & 31) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) r[i * kBnRed + warp] = v[i];
  bar_sync(1 + group, tpr);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = 0.f;
#pragma unroll
    for (int q = 0; q < kBnRed / 4; ++q) {
      const float4 f = reinterpret_cast<const float4*>(r + i * kBnRed)[q];
      v[i] += (f.x + f.y) + (f.z + f.w);
    }
  }
}

__device__ __forceinline__ void ring_wait(int newer) {  // all but the newest groups have landed
  if (newer == 3) cp_async_wait_group<3>();
  else if (newer == 2) cp_async_wait_group<2>();
  else if (newer == 1) cp_async_wait_group<1>();
  else cp_async_wait_group<0>();
}

// Fetches the rows of a group in order through the ring.  F(r, stage) copies
// a thread's pieces.  Aligned rows: a warp reads only what it copied itself,
// so that no barrier is needed.  Otherwise a thread also reads its
// neighbour's piece: a barrier publishes the copies, and only behind it is the
// stage of the row before reused.
template <bool ALIGNED>
struct BnRing {
  int stages, stage = 0;
  template <class F>
  __device__ __forceinline__ BnRing(int n, int64_t row, int64_t step, F&& copy) : stages(n) {
    for (int s = 0; s < n - 1; ++s) {
      copy(row + s * step, s);
      cp_async_commit();
    }
  }
  // brings in the current row; returns its stage
  template <class F>
  __device__ __forceinline__ int next(int64_t row, int64_t step, int group, int tpr, F&& copy) {
    const int here = stage, spare = stage == 0 ? stages - 1 : stage - 1;
    stage = stage == stages - 1 ? 0 : stage + 1;
    if (ALIGNED || stages == 1) {
      sync(group, ALIGNED ? 32 : tpr);  // its readers are done with the stage's last row
      copy(row + (stages - 1) * step, spare);
      cp_async_commit();
      ring_wait(stages - 1);
      sync(group, ALIGNED ? 32 : tpr);
    } else {
      ring_wait(stages - 2);
      sync(group, tpr);
      copy(row + (stages - 1) * step, spare);
      cp_async_commit();
    }
    return here;
  }
  __device__ __forceinline__ static void sync(int group, int tpr) {
    if (tpr == 32) __syncwarp();
    else bar_sync(1 + group, tpr);
  }
};

template <auto Kernel>
int bn_start(BnParams p, const BnGeom& g, BnRows kind, int weight_planes, size_t fixed, const char* what,
             cudaStream_t st) {
  const size_t threads = (size_t)g.tpr * g.rpb, places = (size_t)bn_vectors((int)p.a.D, kind == kBnPacked) + 1;
  const size_t plane = sizeof(uint4) * places * g.rpb, weights = sizeof(float4) * weight_planes * places;
  p.stages = (int)((kBnSmem - fixed - weights) / (plane * p.planes));
  if (p.stages < 1) return set_error(KDN_ERR_INVALID, "%s: a row does not fit shared memory", what);
  if (p.stages > 4) p.stages = 4;
  const size_t smem = weights + p.stages * p.planes * plane;
  if (int rc = allow_smem<Kernel>(kBnSmem - fixed, what)) return rc;
  Kernel<<<g.grid, (unsigned)threads, smem, st>>>(p);
  return check_launch(what);
}

// Aligned: every row of every tensor of the call starts on a 16-byte boundary
// (fp32 outputs: 32) and is a whole number of vectors (absent tensors are).
inline BnRows bn_rows(const KdnBlockNormArgs& a) {
  const int64_t ex = a.stream_bf16 ? 2 : 4, ey = a.act_bf16 ? 2 : 4;
  uintptr_t bits = 0, weights = 0, strides = (uintptr_t)(a.D % kBnVec);
  for (const void* p : {a.x, a.y, a.gate, a.dz, a.dh}) bits |= reinterpret_cast<uintptr_t>(p) & 15;
  for (const void* p : {a.weight, a.post_weight, a.scale}) weights |= reinterpret_cast<uintptr_t>(p) & 15;
  for (const void* p : {a.z, a.dx}) bits |= reinterpret_cast<uintptr_t>(p) & (8 * ex - 1);
  for (const void* p : {a.h, a.dy, a.dgate}) bits |= reinterpret_cast<uintptr_t>(p) & (8 * ey - 1);
  strides |= (uintptr_t)(a.x_stride * ex) & 15;
  if (a.y) strides |= (uintptr_t)(a.y_stride * ey) & 15;
  if (a.gate) strides |= (uintptr_t)(a.gate_stride * ey) & 15;
  if ((bits | weights | strides) == 0) return kBnAligned;
  const bool packed = a.x_stride == a.D && (!a.y || a.y_stride == a.D) && (!a.gate || a.gate_stride == a.D);
  return bits == 0 && packed ? kBnPacked : kBnLoose;
}

}  // namespace
}  // namespace kdn
