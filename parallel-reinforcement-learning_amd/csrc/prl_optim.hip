// prl_optim.hip — optimizer operators over lists of tensors (include/prl_optim.h): the global
// gradient norm and one clipped AdamW step with 32-bit or 8-bit moments.
//
// The tensors' descriptors travel in the kernels' arguments, a batch of 48 to 256 tensors per launch:
// a captured graph then holds them itself, and no table on the device has to outlive a call.  Every
// tensor is cut into chunks of one workgroup each; a workgroup finds its tensor by comparing its
// index with the batch's chunk prefix, 64 entries per ballot.  Fields that a uniform index reads
// from the arguments are 4 or 8 bytes wide: of a byte array and a pointer array with one index the
// compiler once formed a scalar load from two unaligned parts, whose low bits the hardware drops.
//
// One call: list_norm_kernel (per batch; one float64 partial sum per chunk), then list_begin_kernel
// (one workgroup: folds the partials into the norm and the clip coefficient, advances every
// tensor's step count and forms its bias corrections in float64), then list_adam32_kernel /
// list_adam8_kernel per batch.  A short list takes all of that in list_small_kernel's one launch.
//
// Everything here is bound by memory but the shortest lists (launches) and 8-bit moments of 16-bit
// weights (instructions).  MI355X, 3 states in turn, so that nothing comes from the caches:
//   norm of 126 M bfloat16 values               40 us  6.2 TB/s
//   step of 126 M float32 values (28 B each)   560 us  6.3 TB/s  (list_adam32; 655 us with norm and begin)
//   8-bit moments, 126 M float32 (16 B)        339 us  6.0 TB/s  (list_adam8)
//   8-bit moments, 126 M bfloat16 (10 B)   226 - 239 us  5.3 - 5.6 TB/s (two cards)
// (a 2 GiB tensor multiplied in place by torch: 5.9 TB/s).
#include "prl_common.h"
#include "../../include/prl_optim.h"

namespace prl {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
// tensors may start at any element (views of a flat buffer): the types' alignment is one element's,
// the accesses still are 16 / 8 / 4 bytes wide
typedef f32x4 f32x4_u __attribute__((aligned(4)));
typedef u16x4 u16x4_u __attribute__((aligned(2)));
typedef unsigned u32_u __attribute__((aligned(1)));
#define PRL_GLOBAL __attribute__((address_space(1)))

constexpr int L_THREADS = 256;
constexpr int L_BATCH_NORM = 128;     // tensors per launch of the norm,
constexpr int L_BATCH = 64;           // of the 32-bit step,
constexpr int L_BATCH8 = 48;          // of the 8-bit step (more pointers each),
constexpr int L_BATCH_BEGIN = 256;    // of list_begin_kernel: as many as 4 KB of arguments hold
constexpr int L_GROUPS = 16;
// Values per workgroup of a step.  32 bits: 2,048 (50 M bfloat16 values with masters, clipped, 255 us; 4,096: 260,
// 8,192: 266).  8 bits: 2,048 of float32 weights or masters (126 M values 336 us; 1,024: 351, 4,096: 350),
// 4,096 of 16-bit weights alone, where the instructions count and with them what a workgroup
// does once (126 M values, clipped, 256 us; 2,048: 286, 8,192: 258).
constexpr int L_CHUNK32 = 2048, L_CHUNK8 = 2048, L_CHUNK8_16 = 4096;
constexpr int L_COEF = 12;            // floats per tensor in the workspace
constexpr int L_NORM_BLOCKS = 2048;   // partial sums of a norm, besides one per tensor

// per-tensor scalars of a step, formed by list_begin_kernel
struct Coef {
  float clip, decay, step_size, inv_bc2_sqrt, omb1, omb2, beta2, eps;
  unsigned seed, pad[3];
};
static_assert(sizeof(Coef) == 4 * L_COEF, "Coef layout");

template <typename T>
__device__ inline const PRL_GLOBAL T* gptr(const void* p) { return (const PRL_GLOBAL T*)p; }
template <typename T>
__device__ inline PRL_GLOBAL T* gptr(void* p) { return (PRL_GLOBAL T*)p; }

// Everything a step touches is touched once: its loads and stores are marked nontemporal, so that they
// pass the caches without displacing each other (126 M float32 values: 789 -> 679 us; loads alone
// 761, stores alone 789).  The norm that goes before a step reads its gradients plainly: the step
// then finds part of them in the Infinity Cache (nontemporal: 706 us); a norm by itself does not
// (126 M bfloat16 values: plain 52 us, nontemporal 47.5).
#define PRL_LOAD_NT(Q, p) __builtin_nontemporal_load((const PRL_GLOBAL Q*)(p))
#define PRL_STORE_NT(Q, p, x) __builtin_nontemporal_store(x, (PRL_GLOBAL Q*)(p))

// the batch's tensor that workgroup `b` works on: the last one whose first chunk is <= b
__device__ inline int find_entry(const unsigned* start, int count, unsigned b) {
  int before = 0;
  for (int k = 0; k < count; k += 64) {
    const int i = k + (int)(threadIdx.x & 63);
    before += __popcll(__ballot(i < count && start[i] <= b));
  }
  return __builtin_amdgcn_readfirstlane(before - 1);
}

// ---- element types ---------------------------------------------------------------------------
struct F32 {
  typedef f32x4_u Quad;
  typedef float One;
  static __device__ inline f32x4 widen(f32x4 q) { return q; }
  static __device__ inline f32x4 narrow(f32x4 x) { return x; }
  static __device__ inline float widen1(float x) { return x; }
  static __device__ inline float narrow1(float x) { return x; }
};
template <typename H>
struct Half {   // __bf16 / _Float16: conversions round to nearest even
  typedef u16x4_u Quad;
  typedef unsigned short One;
  static __device__ inline float widen1(unsigned short x) { return (float)__builtin_bit_cast(H, x); }
  static __device__ inline unsigned short narrow1(float x) {
    asm("" : "+v"(x));   // of the float32 value: a float16 one would be formed with the sum before it (v_fma_mix)
    return __builtin_bit_cast(unsigned short, (H)x);
  }
  static __device__ inline f32x4 widen(u16x4 q) {
    return f32x4{widen1(q.x), widen1(q.y), widen1(q.z), widen1(q.w)};
  }
  static __device__ inline u16x4 narrow(f32x4 x) {
    return u16x4{narrow1(x.x), narrow1(x.y), narrow1(x.z), narrow1(x.w)};
  }
};
typedef Half<__bf16> BF16;
typedef Half<_Float16> F16;

// ---- norm ------------------------------------------------------------------------------------
// At most L_NORM_BLOCKS chunks and one more per tensor, 8 workgroups per CU with 64 bytes per thread in
// flight.  Squares are summed in float64 (a float32 square overflows from 1.8e19 on; the additions cost
// nothing beside the loads), each chunk's in a fixed order, so a list's norm repeats bit for bit.
struct NormArgs {
  const void* x[L_BATCH_NORM];
  int64_t n[L_BATCH_NORM];
  unsigned start[L_BATCH_NORM];
  unsigned dtype[L_BATCH_NORM];
  int64_t chunk;
  int count;
};
static_assert(sizeof(NormArgs) <= 4096, "kernel arguments");

// up to 4 values from x[0 .. left), zeros behind: the loads are issued together, then converted
template <typename T>
__device__ inline f32x4 load_part(const PRL_GLOBAL typename T::One* x, int left) {
  typename T::One q[3] = {};
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (e < left) q[e] = x[e];
  return f32x4{T::widen1(q[0]), T::widen1(q[1]), T::widen1(q[2]), 0.0f};
}
template <typename T>
__device__ inline void store_part(PRL_GLOBAL typename T::One* x, int left, f32x4 f) {
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (e < left) x[e] = T::narrow1(f[e]);
}

template <typename T, bool ONCE>
__device__ inline double norm_chunk(const void* px, int64_t lo, int64_t hi) {
  typedef typename T::Quad Quad;
  const PRL_GLOBAL typename T::One* x = gptr<typename T::One>(px);
  constexpr int U = 16 / sizeof(Quad) * 4;   // 64 bytes in flight per thread
  double acc = 0.0;
  const auto add = [&](f32x4 f) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = fma((double)f[e], (double)f[e], acc);
  };
  int64_t base = lo;
  for (; base + 4 * L_THREADS * U <= hi; base += 4 * L_THREADS * U) {
    Quad q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const PRL_GLOBAL typename T::One* at = x + base + 4 * (L_THREADS * u + (int)threadIdx.x);
      if (ONCE) q[u] = PRL_LOAD_NT(Quad, at);
      else q[u] = *(const PRL_GLOBAL Quad*)at;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) add(T::widen(q[u]));
  }
  if (base < hi) {
    Quad q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = base + 4 * (L_THREADS * u + (int)threadIdx.x);
      q[u] = Quad{};
      if (i + 4 <= hi) q[u] = *(const PRL_GLOBAL Quad*)(x + i);
    }
    const int64_t part = hi & ~(int64_t)3;   // chunks start at multiples of 4
    if (part < hi && threadIdx.x == 0) add(load_part<T>(x + part, (int)(hi - part)));
#pragma unroll
    for (int u = 0; u < U; ++u) add(T::widen(q[u]));
  }
  return acc;
}

// ONCE: no step of the same gradients follows
template <bool ONCE>
__global__ __launch_bounds__(L_THREADS) void list_norm_kernel(const NormArgs a, double* partial) {
  __shared__ double s_part[L_THREADS / 64];
  const int e = find_entry(a.start, a.count, blockIdx.x);
  const int64_t n = a.n[e], lo = (int64_t)(blockIdx.x - a.start[e]) * a.chunk;
  const int64_t hi = lo + a.chunk < n ? lo + a.chunk : n;
  double acc;
  if (a.dtype[e] == PRL_LIST_F32) acc = norm_chunk<F32, ONCE>(a.x[e], lo, hi);
  else if (a.dtype[e] == PRL_LIST_BF16) acc = norm_chunk<BF16, ONCE>(a.x[e], lo, hi);
  else acc = norm_chunk<F16, ONCE>(a.x[e], lo, hi);
  acc = wave_sum_f64_to63(acc);
  if ((threadIdx.x & 63) == 63) s_part[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0.0;
    for (int w = 0; w < L_THREADS / 64; ++w) sum += s_part[w];
    partial[blockIdx.x] = sum;
  }
}

// ---- the clip coefficient, and a tensor's scalars --------------------------------------------------
__device__ inline float clip_coef(float norm, float max_norm) {
  const float clip = max_norm / (norm + 1e-6f);
  return clip > 1.0f ? 1.0f : clip;   // a NaN stays
}
// b^t by squaring; its relative error grows to t * 2^-53, below float32's rounding up to t = 2^28 (b^t is
// below 2^-23 there for any b up to 1 - 2^-24).  Latency before a step: the CartPole policy's one launch takes
// 7.8 us, 8.5 with pow().
__device__ inline double power(double b, float t) {
  double r = 1.0;
  for (unsigned k = (unsigned)fminf(t, 0xffffff00p0f); k != 0; k >>= 1) {
    if (k & 1) r *= b;
    b *= b;
  }
  return r;
}
// Advances the step count.  float32 counts whole steps up to 2^24 and stays there.  That is well for 32-bit
// moments; with 8-bit ones (coded) the draws would be the same at every step from then on, and a second moment
// beside a block's decaying largest one fall to half of what it should be.  Theirs goes on by the next float32, whose
// bits are hashed in the count's place.
__device__ inline Coef next_coef(const prl_list_group& g, float* count, bool coded, float clip) {
  const double lr = g.lr_dev != nullptr ? (double)g.lr_dev[0] : g.lr;
  float step = count[0] + 1.0f;
  if (coded && step == count[0] && step < 0x1.fffffep127f) step = __uint_as_float(__float_as_uint(step) + 1);
  count[0] = step;
  Coef c{};
  c.clip = clip;
  c.decay = (float)(1.0 - lr * g.weight_decay);
  c.step_size = (float)(lr / (1.0 - power(g.beta1, step)));
  c.inv_bc2_sqrt = (float)(1.0 / sqrt(1.0 - power(g.beta2, step)));
  c.omb1 = (float)(1.0 - g.beta1);
  c.omb2 = (float)(1.0 - g.beta2);
  c.beta2 = (float)g.beta2;
  c.eps = (float)g.eps;
  c.seed = (step <= 0x1p24f ? (unsigned)step : __float_as_uint(step)) * 0x9E3779B1u;
  return c;
}

// ---- once per call: the norm's fold, the step counts, the per-tensor scalars -------------------
constexpr unsigned CODED = 0x80;
struct BeginArgs {
  float* step[L_BATCH_BEGIN];
  unsigned char group[L_BATCH_BEGIN];   // and CODED: moments in 8 bits
  prl_list_group groups[L_GROUPS];
  const double* partial;   // n_partial sums to fold into *norm, or n_partial < 0: *norm is ready
  float* norm;             // or NULL: no clipping
  Coef* coef;              // of the batch's first tensor
  int64_t n_partial;
  float max_norm;
  int count;
};
static_assert(sizeof(BeginArgs) <= 4096, "kernel arguments");

__global__ __launch_bounds__(1024) void list_begin_kernel(const BeginArgs a) {
  __shared__ double s_part[1024 / 64];
  __shared__ float s_norm;
  const int t = threadIdx.x;
  if (a.norm != nullptr) {
    if (a.n_partial >= 0) {
      double acc = 0.0;
      for (int64_t i = t; i < a.n_partial; i += 1024) acc += a.partial[i];
      acc = wave_sum_f64_to63(acc);
      if ((t & 63) == 63) s_part[t >> 6] = acc;
      __syncthreads();
      if (t == 0) {
        double sum = 0.0;
        for (int w = 0; w < 1024 / 64; ++w) sum += s_part[w];
        s_norm = (float)sqrt(sum);
        a.norm[0] = s_norm;
      }
    } else if (t == 0) {
      s_norm = a.norm[0];
    }
    __syncthreads();
  }
  if (t >= a.count) return;
  const float clip = a.norm != nullptr ? clip_coef(s_norm, a.max_norm) : 1.0f;
  const unsigned group = a.group[t];
  a.coef[t] = next_coef(a.groups[group & ~CODED], a.step[t], (group & CODED) != 0, clip);
}

// ---- the step, 32-bit moments ------------------------------------------------------------------
// 28 bytes per float32 value against some 40 instructions: memory's.  Two quads of everything per
// thread are loaded ahead of the arithmetic (one or four: the same times).  Moments are float32 for
// every parameter type; a 16-bit parameter is widened, stepped in float32 and rounded once.
struct Adam32Args {
  void* param[L_BATCH];
  const void* grad[L_BATCH];
  float* master[L_BATCH];
  float* m[L_BATCH];
  float* v[L_BATCH];
  int64_t n[L_BATCH];
  unsigned start[L_BATCH];
  unsigned which[L_BATCH];   // the tensor's place in the call (its Coef), dtype in the top bits
  const Coef* coef;
  int count;
};
static_assert(sizeof(Adam32Args) <= 4096, "kernel arguments");

__device__ inline float adam_weight(const Coef& c, float w, float m, float rms) {
  return fmaf(-c.step_size, m * __builtin_amdgcn_rcpf(fmaf(rms, c.inv_bc2_sqrt, c.eps)), w * c.decay);
}
// one rounding per operation, as written: the 8-bit moments' codes follow from these bits
__device__ inline void adam_moments(const Coef& c, float g, float& m, float& v) {
  g = g * c.clip;
  m = m + (g - m) * c.omb1;
  v = v * c.beta2 + (g * g) * c.omb2;
}

__device__ inline void adam32_quad(const Coef& c, f32x4 g, f32x4& x, f32x4& m, f32x4& v) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float me = m[e], ve = v[e];
    adam_moments(c, g[e], me, ve);
    x[e] = adam_weight(c, x[e], me, sqrtf(ve));
    m[e] = me;
    v[e] = ve;
  }
}
// 1 .. 3 values
template <typename T, bool MASTER>
__device__ inline void adam32_part(const Coef& c, PRL_GLOBAL typename T::One* p, const PRL_GLOBAL typename T::One* g,
                                   PRL_GLOBAL float* w, PRL_GLOBAL float* m, PRL_GLOBAL float* v, int left) {
  const f32x4 gr = load_part<T>(g, left);
  f32x4 mq = load_part<F32>(m, left), vq = load_part<F32>(v, left);
  f32x4 x = MASTER ? load_part<F32>(w, left) : load_part<T>(p, left);
  adam32_quad(c, gr, x, mq, vq);
  store_part<F32>(m, left, mq);
  store_part<F32>(v, left, vq);
  if (MASTER) store_part<F32>(w, left, x);
  store_part<T>(p, left, x);
}

template <typename T, bool MASTER>
__device__ inline void adam32_chunk(const Coef& c, void* pp, const void* pg, float* pw, float* pm,
                                    float* pv, int64_t lo, int64_t hi) {
  PRL_GLOBAL typename T::One* p = gptr<typename T::One>(pp);
  const PRL_GLOBAL typename T::One* g = gptr<typename T::One>(pg);
  PRL_GLOBAL float* w = gptr<float>(pw);
  PRL_GLOBAL float* m = gptr<float>(pm);
  PRL_GLOBAL float* v = gptr<float>(pv);
  typedef typename T::Quad Quad;
  constexpr int U = 2;
  for (int64_t base = lo; base < hi; base += 4 * L_THREADS * U) {
    Quad pq[U], gq[U];
    f32x4 wq[U], mq[U], vq[U];
    const int64_t k0 = base + 4 * (int)threadIdx.x;
    const bool whole = base + 4 * L_THREADS * U <= hi;   // of the workgroup: no bounds in the usual case
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = k0 + 4 * L_THREADS * u;
      if (whole || k + 4 <= hi) {
        if (MASTER) wq[u] = PRL_LOAD_NT(f32x4_u, w + k);
        else pq[u] = PRL_LOAD_NT(Quad, p + k);
        gq[u] = PRL_LOAD_NT(Quad, g + k);
        mq[u] = PRL_LOAD_NT(f32x4_u, m + k);
        vq[u] = PRL_LOAD_NT(f32x4_u, v + k);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = k0 + 4 * L_THREADS * u;
      if (whole || k + 4 <= hi) {
        f32x4 x = MASTER ? wq[u] : T::widen(pq[u]);
        adam32_quad(c, T::widen(gq[u]), x, mq[u], vq[u]);
        PRL_STORE_NT(f32x4_u, m + k, mq[u]);
        PRL_STORE_NT(f32x4_u, v + k, vq[u]);
        if (MASTER) PRL_STORE_NT(f32x4_u, w + k, x);
        PRL_STORE_NT(Quad, p + k, T::narrow(x));
      }
    }
  }
  const int64_t part = hi & ~(int64_t)3;   // a tensor's last 1 .. 3 values: one thread's
  if (part < hi && threadIdx.x == L_THREADS - 1)
    adam32_part<T, MASTER>(c, p + part, g + part, w + (MASTER ? part : 0), m + part, v + part, (int)(hi - part));
}

__global__ __launch_bounds__(L_THREADS) void list_adam32_kernel(const Adam32Args a) {
  const int e = find_entry(a.start, a.count, blockIdx.x);
  const int64_t n = a.n[e], lo = (int64_t)(blockIdx.x - a.start[e]) * L_CHUNK32;
  const int64_t hi = lo + L_CHUNK32 < n ? lo + L_CHUNK32 : n;
  const unsigned which = a.which[e], dtype = which >> 30;
  const Coef c = a.coef[which & 0x3fffffffu];
  void* p = a.param[e];
  const void* g = a.grad[e];
  float *w = a.master[e], *m = a.m[e], *v = a.v[e];
  if (dtype == PRL_LIST_F32) adam32_chunk<F32, false>(c, p, g, w, m, v, lo, hi);
  else if (dtype == PRL_LIST_BF16) {
    if (w) adam32_chunk<BF16, true>(c, p, g, w, m, v, lo, hi);
    else adam32_chunk<BF16, false>(c, p, g, w, m, v, lo, hi);
  } else {
    if (w) adam32_chunk<F16, true>(c, p, g, w, m, v, lo, hi);
    else adam32_chunk<F16, false>(c, p, g, w, m, v, lo, hi);
  }
}

// ---- the step, 8-bit moments -------------------------------------------------------------------
// A block of 256 values is one wave's: 4 consecutive values per lane, so a code quad is one 32-bit
// word, the block's largest magnitude a wave reduction, and nothing crosses waves.  Some 60 issue slots
// per value: beside 16 bytes (float32 weights) the loads bound it, beside 10 (16-bit weights) the
// instructions do.  Rounding r to 8 bits to the nearest would leave it in place for good: a step moves it
// by 0.05 % at beta2 = 0.999, codes lie 6 to 12 % apart, so it is rounded stochastically.
struct Adam8Args {
  void* param[L_BATCH8];
  const void* grad[L_BATCH8];
  float* master[L_BATCH8];
  void* m[L_BATCH8];
  void* r[L_BATCH8];
  float* m_scale[L_BATCH8];
  float* r_scale[L_BATCH8];
  int64_t n[L_BATCH8];
  unsigned start[L_BATCH8];
  unsigned which[L_BATCH8];
  const Coef* coef;
  int count;
};
static_assert(sizeof(Adam8Args) <= 4096, "kernel arguments");

// the largest of x and of y over the wave: one swap of halves (x's in lanes 0 - 31, y's in 32 - 63), then
// five DPP steps for both (xor 1, xor 2, half-row mirror, row mirror, row 0 / 2's lane 15 broadcast)
__device__ inline void wave_max_pair(unsigned& x, unsigned& y) {
  const auto moved = [](unsigned v, int m) { return v > (unsigned)m ? v : (unsigned)m; };
  const auto s = __builtin_amdgcn_permlane32_swap(x, y, false, false);
  unsigned v = s[0] > s[1] ? s[0] : s[1];
  v = moved(v, __builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
  v = moved(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
  v = moved(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));
  v = moved(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false));
  v = moved(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false));
  x = (unsigned)__builtin_amdgcn_readlane((int)v, 31);
  y = (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}

// The mixing of the bits is published: C. Wellons' search for 32-bit integer hashes of low bias found this pair of
// multipliers for the shifts 16, 15, 16.  0x9E3779B1 and 0x85EBCA77 (a step count's and an index's high word's
// factor) are primes that xxHash's specification lists.
// A value's two 16-bit draws at this step are the halves of h ^ (h >> 16), h = draw_bits(its index
// folded to 32 bits, ..): the low one for the first moment, the high one for the second
__device__ inline unsigned draw_bits(unsigned at, unsigned seed) {
  unsigned h = at ^ seed;
  h = (h ^ (h >> 16)) * 0x7FEB352Du;
  h = (h ^ (h >> 15)) * 0x846CA68Bu;
  asm("" : "+v"(h));   // opaque: the compiler would form h << 16 by a third multiplication (quarter rate)
  return h;
}

// the largest of the four magnitudes, as bits (a NaN is larger than an infinity); the roots are
// positive, or a NaN of either sign: larger than an infinity too
template <bool SIGNED>
__device__ inline unsigned max_bits(const float (&x)[4]) {
  unsigned most = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const unsigned b = __float_as_uint(x[e]) & (SIGNED ? 0x7fffffffu : 0xffffffffu);
    most = most > b ? most : b;
  }
  return most;
}

// The root of v >= 0 by one step of Newton's method on v_rsq_f32, half the instructions of sqrtf():
// within 2^-44 of the root before its last rounding.  Below 2^-126 it comes out small (a positive v
// still gives a positive root), and an infinite v gives NaN: a block is taken again with sqrtf() unless its
// largest root lies from 2^-40 to the largest finite number.  In such a block a root below 2^-63 is the
// smallest code, right or small, and vanishes beside an eps of 2^-30 or more in the denominator (beta2 up
// to 1 - 2^-16); a smaller eps takes sqrtf() throughout.
constexpr unsigned QUICK_FROM = 0x2b800000u;   // 2^-40
__device__ inline float quick_root(float v) {
  const float y = __builtin_amdgcn_rsqf(fmaxf(v, 0x1p-126f));
  const float s = v * y;
  return fmaf(fmaf(-s, s, v), 0.5f * y, s);
}

// 256 / A for a block's largest magnitude A given as its bits, by v_rcp_f32 and one step of Newton's
// method (both operands' sizes stay normal); 0: the block is held as zeros
__device__ inline float block_factor(unsigned max_bits) {
  const float A = __uint_as_float(max_bits), a = A * 0x1p-8f;
  const float x = __builtin_amdgcn_rcpf(a);
  return max_bits < 0x7f800000u && A >= 0x1p-118f ? fmaf(fmaf(-a, x, 1.0f), x, x) : 0.0f;
}
// A as stored: NaN where a value of the block is not finite
__device__ inline float block_store(unsigned max_bits, float k) {
  return max_bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : k > 0.0f ? __uint_as_float(max_bits) : 0.0f;
}

// The pointers are the block's own (uniform over the wave); left: its values, 256 but for a tensor's
// last block (WHOLE: known to be 256); at: the first value's index folded to 32 bits.
template <typename T, bool MASTER, bool WHOLE>
__device__ inline void adam8_block(const Coef& c, PRL_GLOBAL typename T::One* p, const PRL_GLOBAL typename T::One* g,
                                   PRL_GLOBAL float* w, PRL_GLOBAL unsigned char* mc, PRL_GLOBAL unsigned char* rc,
                                   PRL_GLOBAL float* ms, PRL_GLOBAL float* rs, unsigned at, int left) {
  typedef typename T::Quad Quad;
  const int lane = threadIdx.x & 63;
  const unsigned i = 4 * lane;
  left = WHOLE ? 4 : left - (int)i;   // this lane's values: 4 or more, 1 .. 3, or none
  f32x4 x, gr;
  unsigned mq = 0, rq = 0;
  if (left >= 4) {
    gr = T::widen(PRL_LOAD_NT(Quad, g + i));
    if (MASTER) x = PRL_LOAD_NT(f32x4_u, w + i);
    else x = T::widen(PRL_LOAD_NT(Quad, p + i));
    mq = PRL_LOAD_NT(u32_u, mc + i);
    rq = PRL_LOAD_NT(u32_u, rc + i);
  } else {
    gr = load_part<T>(g + i, left);
    x = MASTER ? load_part<F32>(w + i, left) : load_part<T>(p + i, left);
    for (int e = 0; e < 3; ++e)
      if (e < left) {
        mq |= (unsigned)mc[i + e] << (8 * e);
        rq |= (unsigned)rc[i + e] << (8 * e);
      }
  }
  const float ma = ms[0] * 0x1p-8f, ra = rs[0] * 0x1p-8f;
  const auto m01 = __builtin_amdgcn_cvt_pk_f32_fp8(mq, false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8(mq, true);
  const auto r01 = __builtin_amdgcn_cvt_pk_f32_fp8(rq, false), r23 = __builtin_amdgcn_cvt_pk_f32_fp8(rq, true);
  float m[4] = {m01[0], m01[1], m23[0], m23[1]}, r[4] = {r01[0], r01[1], r23[0], r23[1]};
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    m[e] = m[e] * ma;
    r[e] = r[e] * ra;
    v[e] = r[e] * r[e];
    adam_moments(c, gr[e], m[e], v[e]);
    if (!WHOLE && e >= left) m[e] = v[e] = 0.0f;   // past the tensor's end nothing counts (a NaN clip would)
    r[e] = quick_root(v[e]);
  }
  unsigned m_max = max_bits<true>(m), r_max = max_bits<false>(r);
  wave_max_pair(m_max, r_max);
  // not the quick root's range (see there)
  if (r_max - QUICK_FROM >= 0x7f800000u - QUICK_FROM || c.eps < 0x1p-30f) {
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = sqrtf(v[e]);
    unsigned again = m_max;
    r_max = max_bits<false>(r);
    wave_max_pair(again, r_max);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = adam_weight(c, x[e], m[e], r[e]);
  if (left >= 4) {
    if (MASTER) PRL_STORE_NT(f32x4_u, w + i, x);
    PRL_STORE_NT(Quad, p + i, T::narrow(x));
  } else {
    if (MASTER) store_part<F32>(w + i, left, x);
    store_part<T>(p + i, left, x);
  }
  // both factors at once: the first moment's in lane 0, the second's in lane 1
  const float k = block_factor(lane & 1 ? r_max : m_max);
  const float km = __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(k), 0));
  const float kr = __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(k), 1));
  // stochastic rounding to e4m3: the conversion adds its random bits below the mantissa bits it keeps
  // and truncates, the sign aside; 16 of the 20 are drawn, the rest are 0.  (A * k may come out an ulp
  // above 256: no draw carries that over 16 ulps to the next code.)
  unsigned d[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) d[e] = draw_bits(at + i + e, c.seed);
  int mw = 0, rw = 0;
  if (km > 0.0f) {
    const auto y = [&](int e) { return m[e] * km; };
    const auto draw = [&](int e) { return (d[e] << 16) ^ (d[e] & 0xffff0000u); };
    mw = __builtin_amdgcn_cvt_sr_fp8_f32(y(0), draw(0), mw, 0);
    mw = __builtin_amdgcn_cvt_sr_fp8_f32(y(1), draw(1), mw, 1);
    mw = __builtin_amdgcn_cvt_sr_fp8_f32(y(2), draw(2), mw, 2);
    mw = __builtin_amdgcn_cvt_sr_fp8_f32(y(3), draw(3), mw, 3);
  }
  if (kr > 0.0f) {
    float y[4] = {r[0] * kr, r[1] * kr, r[2] * kr, r[3] * kr};
    // an r above 0 stays above 0: 2^-9 is the smallest code.  Few blocks hold one that small.
    if (__ballot(fminf(fminf(y[0], y[1]), fminf(y[2], y[3])) < 0x1p-9f) != 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = r[e] > 0.0f ? fmaxf(y[e], 0x1p-9f) : 0.0f;
    }
    const auto draw = [&](int e) { return d[e] & 0xffff0000u; };
    rw = __builtin_amdgcn_cvt_sr_fp8_f32(y[0], draw(0), rw, 0);
    rw = __builtin_amdgcn_cvt_sr_fp8_f32(y[1], draw(1), rw, 1);
    rw = __builtin_amdgcn_cvt_sr_fp8_f32(y[2], draw(2), rw, 2);
    rw = __builtin_amdgcn_cvt_sr_fp8_f32(y[3], draw(3), rw, 3);
  }
  if (left >= 4) {
    PRL_STORE_NT(u32_u, mc + i, (unsigned)mw);
    PRL_STORE_NT(u32_u, rc + i, (unsigned)rw);
  } else {
    for (int e = 0; e < 3; ++e)
      if (e < left) {
        mc[i + e] = (unsigned char)((unsigned)mw >> (8 * e));
        rc[i + e] = (unsigned char)((unsigned)rw >> (8 * e));
      }
  }
  if (lane == 0) {
    ms[0] = block_store(m_max, km);
    rs[0] = block_store(r_max, kr);
  }
}

__host__ __device__ inline int adam8_chunk_of(unsigned dtype, bool master) {
  return dtype == PRL_LIST_F32 || master ? L_CHUNK8 : L_CHUNK8_16;
}
template <typename T, bool MASTER>
__device__ inline void adam8_chunk(const Coef& c, const Adam8Args& a, int e, int64_t lo, int64_t hi, int64_t n) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int64_t base = lo + wave * PRL_LIST_BLOCK; base < hi; base += L_THREADS / 64 * PRL_LIST_BLOCK) {
    const int64_t b = base / PRL_LIST_BLOCK;
    const unsigned at = (unsigned)base + (unsigned)((uint64_t)base >> 32) * 0x85EBCA77u;
    PRL_GLOBAL typename T::One* p = gptr<typename T::One>(a.param[e]) + base;
    const PRL_GLOBAL typename T::One* g = gptr<typename T::One>(a.grad[e]) + base;
    PRL_GLOBAL float* w = gptr<float>(a.master[e]) + (MASTER ? base : 0);
    PRL_GLOBAL unsigned char *mc = gptr<unsigned char>(a.m[e]) + base, *rc = gptr<unsigned char>(a.r[e]) + base;
    PRL_GLOBAL float *ms = gptr<float>(a.m_scale[e]) + b, *rs = gptr<float>(a.r_scale[e]) + b;
    if (base + PRL_LIST_BLOCK <= n) adam8_block<T, MASTER, true>(c, p, g, w, mc, rc, ms, rs, at, PRL_LIST_BLOCK);
    else adam8_block<T, MASTER, false>(c, p, g, w, mc, rc, ms, rs, at, (int)(n - base));
  }
}

__global__ __launch_bounds__(L_THREADS) void list_adam8_kernel(const Adam8Args a) {
  const int e = find_entry(a.start, a.count, blockIdx.x);
  const unsigned which = a.which[e], dtype = which >> 30;
  const int chunk = adam8_chunk_of(dtype, a.master[e] != nullptr);
  const int64_t n = a.n[e], lo = (int64_t)(blockIdx.x - a.start[e]) * chunk;
  const int64_t hi = lo + chunk < n ? lo + chunk : n;
  const Coef c = a.coef[which & 0x3fffffffu];
  const bool master = a.master[e] != nullptr;
  if (dtype == PRL_LIST_F32) adam8_chunk<F32, false>(c, a, e, lo, hi, n);
  else if (dtype == PRL_LIST_BF16) {
    if (master) adam8_chunk<BF16, true>(c, a, e, lo, hi, n);
    else adam8_chunk<BF16, false>(c, a, e, lo, hi, n);
  } else {
    if (master) adam8_chunk<F16, true>(c, a, e, lo, hi, n);
    else adam8_chunk<F16, false>(c, a, e, lo, hi, n);
  }
}

// ---- a short list in one launch ------------------------------------------------------------------
// Up to L_SMALL_ITEMS blocks of 256 values in L_SMALL tensors: one workgroup of 16 waves, a block per
// wave at a time, takes the norm, the scalars and the step.  Both ways, us per clipped step of 16 tensors as a call /
// on the GPU alone (50 steps in one graph), one launch and three:
//   blocks   float32 weights, 32 bits    bfloat16 weights, 8 bits
//      48    18.6 /  7.8  26.7 /  7.8    20.9 / 10.5  29.9 /  8.9
//     112    18.8 / 13.1  27.0 /  8.3    20.9 / 19.7  29.8 /  9.6
//     160    18.7 / 17.6  26.9 /  8.4    27.9 / 26.7  29.9 / 10.5
//     176    19.3 / 18.7  26.9 /  8.3    29.6 / 28.7  29.7 / 10.4
//     304    30.2 / 29.8  26.8 /  8.4    47.6 / 46.8  29.7 / 11.1
// (the norm alone: 160 blocks 14.4 / 4.4 and 19.4 / 4.1, 1,008 blocks 18.5 / 17.7 and 19.6 / 3.9.)  One bound for
// all, just below where the slowest form's calls are level.  It is a bound for calls, whose time is mostly the
// host's: on the GPU alone (a captured step, a stream that is behind) three launches are level at some 45 blocks
// and ahead beyond.
constexpr int L_SMALL = 32;
constexpr int L_SMALL_ITEMS = 160;
constexpr int L_SMALL_WAVES = 16;
struct SmallArgs {
  void* param[L_SMALL];
  const void* grad[L_SMALL];
  float* master[L_SMALL];
  void* m[L_SMALL];
  void* r[L_SMALL];
  float* m_scale[L_SMALL];
  float* r_scale[L_SMALL];
  float* step[L_SMALL];
  int n[L_SMALL];
  unsigned start[L_SMALL];
  unsigned kind[L_SMALL];    // dtype | bits << 8 | group << 16
  prl_list_group groups[L_GROUPS];
  float* norm;
  float max_norm;
  int count, items;
};
static_assert(sizeof(SmallArgs) <= 4096, "kernel arguments");

template <typename T>
__device__ inline f32x4 load_quad(const void* px, int i, int left) {
  const PRL_GLOBAL typename T::One* x = gptr<typename T::One>(px) + i;
  return left >= 4 ? T::widen(*(const PRL_GLOBAL typename T::Quad*)x) : load_part<T>(x, left);
}

template <typename T, bool MASTER>
__device__ inline void small_item(const Coef& c, const SmallArgs& a, int e, int base) {
  PRL_GLOBAL typename T::One* p = gptr<typename T::One>(a.param[e]) + base;
  const PRL_GLOBAL typename T::One* g = gptr<typename T::One>(a.grad[e]) + base;
  PRL_GLOBAL float* w = gptr<float>(a.master[e]) + (MASTER ? base : 0);
  const int left = a.n[e] - base;
  if ((a.kind[e] >> 8 & 0xff) == 8) {
    PRL_GLOBAL unsigned char *mc = gptr<unsigned char>(a.m[e]) + base, *rc = gptr<unsigned char>(a.r[e]) + base;
    PRL_GLOBAL float* ms = gptr<float>(a.m_scale[e]) + base / PRL_LIST_BLOCK;
    PRL_GLOBAL float* rs = gptr<float>(a.r_scale[e]) + base / PRL_LIST_BLOCK;
    adam8_block<T, MASTER, false>(c, p, g, w, mc, rc, ms, rs, (unsigned)base, left);
    return;
  }
  PRL_GLOBAL float *m = gptr<float>(a.m[e]) + base, *v = gptr<float>(a.r[e]) + base;
  const int i = 4 * (int)(threadIdx.x & 63);
  if (i + 4 <= left) {
    f32x4 mq = *(const PRL_GLOBAL f32x4_u*)(m + i), vq = *(const PRL_GLOBAL f32x4_u*)(v + i);
    const f32x4 gr = T::widen(*(const PRL_GLOBAL typename T::Quad*)(g + i));
    f32x4 x;
    if (MASTER) x = *(const PRL_GLOBAL f32x4_u*)(w + i);
    else x = T::widen(*(const PRL_GLOBAL typename T::Quad*)(p + i));
    adam32_quad(c, gr, x, mq, vq);
    *(PRL_GLOBAL f32x4_u*)(m + i) = mq;
    *(PRL_GLOBAL f32x4_u*)(v + i) = vq;
    if (MASTER) *(PRL_GLOBAL f32x4_u*)(w + i) = x;
    *(PRL_GLOBAL typename T::Quad*)(p + i) = T::narrow(x);
  } else if (i < left) {
    adam32_part<T, MASTER>(c, p + i, g + i, MASTER ? w + i : w, m + i, v + i, left - i);
  }
}

// STEP: the whole step; otherwise the norm alone
template <bool STEP>
__global__ __launch_bounds__(64 * L_SMALL_WAVES) void list_small_kernel(const SmallArgs a) {
  __shared__ double s_part[L_SMALL_WAVES];
  __shared__ Coef s_coef[L_SMALL];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const unsigned first = lane < a.count ? a.start[lane] : 0xffffffffu;   // of tensor `lane`
  const auto entry = [&](int item) { return __popcll(__ballot(first <= (unsigned)item)) - 1; };
  // the scalars beside the norm's loads, by the wave with the fewest blocks
  if (STEP && wave == L_SMALL_WAVES - 1 && lane < a.count)
    s_coef[lane] = next_coef(a.groups[a.kind[lane] >> 16], a.step[lane], (a.kind[lane] >> 8 & 0xff) == 8, 1.0f);
  if (a.norm != nullptr) {
    double acc = 0.0;
    for (int b = wave; b < a.items; b += 4 * L_SMALL_WAVES) {
      f32x4 f[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        f[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int item = b + L_SMALL_WAVES * u;
        if (item < a.items) {
          const int e = entry(item), i = (item - (int)a.start[e]) * PRL_LIST_BLOCK + 4 * lane, left = a.n[e] - i;
          const unsigned dtype = a.kind[e] & 0xff;
          if (dtype == PRL_LIST_F32) f[u] = load_quad<F32>(a.grad[e], i, left);
          else if (dtype == PRL_LIST_BF16) f[u] = load_quad<BF16>(a.grad[e], i, left);
          else f[u] = load_quad<F16>(a.grad[e], i, left);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = fma((double)f[u][e], (double)f[u][e], acc);
    }
    acc = wave_sum_f64_to63(acc);
    if (lane == 63) s_part[wave] = acc;
  }
  __syncthreads();
  float clip = 1.0f;
  if (a.norm != nullptr) {
    double sum = 0.0;
    for (int w = 0; w < L_SMALL_WAVES; ++w) sum += s_part[w];
    const float norm = (float)sqrt(sum);
    if (t == 0) a.norm[0] = norm;
    clip = clip_coef(norm, a.max_norm);
  }
  if (!STEP) return;
  for (int item = wave; item < a.items; item += L_SMALL_WAVES) {
    const int e = entry(item), base = (item - (int)a.start[e]) * PRL_LIST_BLOCK;
    Coef c = s_coef[e];
    c.clip = clip;
    const bool master = a.master[e] != nullptr;
    const unsigned dtype = a.kind[e] & 0xff;
    if (dtype == PRL_LIST_F32) small_item<F32, false>(c, a, e, base);
    else if (dtype == PRL_LIST_BF16) {
      if (master) small_item<BF16, true>(c, a, e, base);
      else small_item<BF16, false>(c, a, e, base);
    } else {
      if (master) small_item<F16, true>(c, a, e, base);
      else small_item<F16, false>(c, a, e, base);
    }
  }
}

// ---- host --------------------------------------------------------------------------------------
inline int64_t list_total(const prl_list_entry* e, int64_t count) {
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) total += e[i].numel;
  return total;
}

// the partial sums of all grads' squares into partial[0 .. *n_partial)
int launch_norm(const prl_list_entry* e, int64_t count, bool once, double* partial, int64_t* n_partial, hipStream_t st) {
  const int64_t tile = 4 * L_THREADS * 4;
  NormArgs a{};
  a.chunk = tile * (1 + list_total(e, count) / (tile * L_NORM_BLOCKS));
  int64_t done = 0, blocks = 0;
  for (int64_t i = 0; i <= count; ++i) {
    if (a.count == L_BATCH_NORM || (i == count && a.count > 0)) {
      if (once) hipLaunchKernelGGL(list_norm_kernel<true>, dim3((unsigned)blocks), dim3(L_THREADS), 0, st, a, partial + done);
      else hipLaunchKernelGGL(list_norm_kernel<false>, dim3((unsigned)blocks), dim3(L_THREADS), 0, st, a, partial + done);
      PRL_LAUNCH_CHECK("list_norm");
      done += blocks;
      blocks = 0;
      a.count = 0;
    }
    if (i == count || e[i].numel == 0) continue;
    a.x[a.count] = e[i].grad;
    a.n[a.count] = e[i].numel;
    a.start[a.count] = (unsigned)blocks;
    a.dtype[a.count] = (unsigned)e[i].dtype;
    ++a.count;
    blocks += cdiv(e[i].numel, a.chunk);
  }
  *n_partial = done;
  return PRL_OK;
}

// list_begin_kernel over all tensors: batches of at most L_BATCH_BEGIN tensors and L_GROUPS groups
int launch_begin(const prl_list_entry* e, int64_t count, const prl_list_group* groups, float max_norm,
                 float* norm, const double* partial, int64_t n_partial, Coef* coef, hipStream_t st) {
  BeginArgs a{};
  a.partial = partial;
  a.norm = norm;
  a.n_partial = n_partial;
  a.max_norm = max_norm;
  int64_t first = 0, of[L_GROUPS];
  int n_of = 0;
  for (int64_t i = 0;; ++i) {
    int g = 0;
    if (i < count) {
      while (g < n_of && of[g] != e[i].group) ++g;
    }
    if (i == count || a.count == L_BATCH_BEGIN || g == L_GROUPS) {
      a.coef = coef + first;
      hipLaunchKernelGGL(list_begin_kernel, dim3(1), dim3(1024), 0, st, a);
      PRL_LAUNCH_CHECK("list_begin");
      a.n_partial = -1;   // later batches read the norm that the first one folded
      first = i;
      a.count = n_of = g = 0;
      if (i == count) return PRL_OK;
    }
    if (g == n_of) {
      of[n_of] = e[i].group;
      a.groups[n_of++] = groups[e[i].group];
    }
    a.step[a.count] = e[i].step;
    a.group[a.count] = (unsigned char)(g | (e[i].bits == 8 ? CODED : 0));
    ++a.count;
  }
}

// a launch has fewer than 2^32 threads: a batch ends before its workgroups pass this
constexpr int64_t L_MAX_BLOCKS = (int64_t)1 << 23;

int launch_adam32(const prl_list_entry* e, int64_t count, const Coef* coef, hipStream_t st) {
  Adam32Args a{};
  a.coef = coef;
  int64_t blocks = 0;
  for (int64_t i = 0; i <= count; ++i) {
    const int64_t more = i < count && e[i].bits == 32 ? cdiv(e[i].numel, L_CHUNK32) : 0;
    if (a.count > 0 && (a.count == L_BATCH || i == count || blocks + more > L_MAX_BLOCKS)) {
      hipLaunchKernelGGL(list_adam32_kernel, dim3((unsigned)blocks), dim3(L_THREADS), 0, st, a);
      PRL_LAUNCH_CHECK("list_adam32");
      blocks = 0;
      a.count = 0;
    }
    if (more == 0) continue;
    const int k = a.count++;
    a.param[k] = e[i].param;
    a.grad[k] = e[i].grad;
    a.master[k] = e[i].master;
    a.m[k] = static_cast<float*>(e[i].exp_avg);
    a.v[k] = static_cast<float*>(e[i].second);
    a.n[k] = e[i].numel;
    a.start[k] = (unsigned)blocks;
    a.which[k] = (unsigned)i | (unsigned)e[i].dtype << 30;
    blocks += more;
  }
  return PRL_OK;
}

int launch_adam8(const prl_list_entry* e, int64_t count, const Coef* coef, hipStream_t st) {
  Adam8Args a{};
  a.coef = coef;
  int64_t blocks = 0;
  for (int64_t i = 0; i <= count; ++i) {
    const int64_t more = i < count && e[i].bits == 8 ? cdiv(e[i].numel, adam8_chunk_of((unsigned)e[i].dtype, e[i].master != nullptr)) : 0;
    if (a.count > 0 && (a.count == L_BATCH8 || i == count || blocks + more > L_MAX_BLOCKS)) {
      hipLaunchKernelGGL(list_adam8_kernel, dim3((unsigned)blocks), dim3(L_THREADS), 0, st, a);
      PRL_LAUNCH_CHECK("list_adam8");
      blocks = 0;
      a.count = 0;
    }
    if (more == 0) continue;
    const int k = a.count++;
    a.param[k] = e[i].param;
    a.grad[k] = e[i].grad;
    a.master[k] = e[i].master;
    a.m[k] = e[i].exp_avg;
    a.r[k] = e[i].second;
    a.m_scale[k] = e[i].exp_avg_scale;
    a.r_scale[k] = e[i].second_scale;
    a.n[k] = e[i].numel;
    a.start[k] = (unsigned)blocks;
    a.which[k] = (unsigned)i | (unsigned)e[i].dtype << 30;
    blocks += more;
  }
  return PRL_OK;
}

// whether one launch of list_small_kernel takes the list
bool is_small(const prl_list_entry* e, int64_t count, int64_t n_groups) {
  if (count > L_SMALL || n_groups > L_GROUPS) return false;
  int64_t items = 0;
  for (int64_t i = 0; i < count; ++i) {
    items += cdiv(e[i].numel, PRL_LIST_BLOCK);
    if (items > L_SMALL_ITEMS) return false;
  }
  return true;
}

template <bool STEP>
int launch_small(const prl_list_entry* e, int64_t count, const prl_list_group* groups, int64_t n_groups,
                 float max_norm, float* norm, hipStream_t st) {
  SmallArgs a{};
  int64_t items = 0;
  for (int64_t i = 0; i < count; ++i) {
    a.start[i] = (unsigned)items;
    items += cdiv(e[i].numel, PRL_LIST_BLOCK);
    a.grad[i] = e[i].grad;
    a.n[i] = (int)e[i].numel;
    a.kind[i] = (unsigned)e[i].dtype;
    if (!STEP) continue;
    a.param[i] = e[i].param;
    a.master[i] = e[i].master;
    a.m[i] = e[i].exp_avg;
    a.r[i] = e[i].second;
    a.m_scale[i] = e[i].exp_avg_scale;
    a.r_scale[i] = e[i].second_scale;
    a.step[i] = e[i].step;
    a.kind[i] |= (unsigned)e[i].bits << 8 | (unsigned)e[i].group << 16;
  }
  for (int64_t g = 0; g < n_groups; ++g) a.groups[g] = groups[g];
  a.norm = norm;
  a.max_norm = max_norm;
  a.count = (int)count;
  a.items = (int)items;
  hipLaunchKernelGGL(list_small_kernel<STEP>, dim3(1), dim3(64 * L_SMALL_WAVES), 0, st, a);
  PRL_LAUNCH_CHECK("list_small");
  return PRL_OK;
}

constexpr int64_t L_MAX_COUNT = 1 << 24, L_MAX_NUMEL = (int64_t)1 << 40;
// sizes and types; a list's total stays below 2^40 values, so every launch's grid fits
int check_list(const char* what, const prl_list_entry* e, int64_t count) {
  PRL_REQUIRE(count >= 0 && count < L_MAX_COUNT, "%s: %lld tensors", what, (long long)count);
  PRL_REQUIRE(count == 0 || e != nullptr, "%s: null entries", what);
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) {
    PRL_REQUIRE(e[i].numel >= 0 && e[i].numel < L_MAX_NUMEL, "%s: tensor %lld: bad size %lld", what,
                (long long)i, (long long)e[i].numel);
    total += e[i].numel;
    PRL_REQUIRE(total < L_MAX_NUMEL, "%s: list too large", what);
    PRL_REQUIRE(e[i].dtype >= PRL_LIST_F32 && e[i].dtype <= PRL_LIST_F16, "%s: tensor %lld: unknown type %d", what,
                (long long)i, (int)e[i].dtype);
    PRL_REQUIRE(e[i].numel == 0 || e[i].grad, "%s: tensor %lld: null grad", what, (long long)i);
    PRL_REQUIRE((reinterpret_cast<uintptr_t>(e[i].grad) & (e[i].dtype == PRL_LIST_F32 ? 3u : 1u)) == 0,
                "%s: tensor %lld: grad not aligned to its type", what, (long long)i);
  }
  return PRL_OK;
}

}  // namespace prl

using namespace prl;

extern "C" int64_t prl_list_workspace_bytes(const prl_list_entry* entries, int64_t count, int64_t n_groups) {
  if (count < 0 || count >= L_MAX_COUNT || (count > 0 && entries == nullptr)) return -1;
  for (int64_t i = 0; i < count; ++i)
    if (entries[i].numel < 0 || entries[i].numel >= L_MAX_NUMEL) return -1;
  if (is_small(entries, count, n_groups)) return 0;
  return (int64_t)sizeof(Coef) * count + 8 * (L_NORM_BLOCKS + count);
}

extern "C" int prl_list_norm(const prl_list_entry* entries, int64_t count, float* norm, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  if (int rc = check_list("prl_list_norm", entries, count)) return rc;
  PRL_REQUIRE(norm, "prl_list_norm: null norm");
  PRL_REQUIRE((reinterpret_cast<uintptr_t>(norm) & 3u) == 0, "prl_list_norm: norm not aligned to its type");
  if (is_small(entries, count, 0)) return launch_small<false>(entries, count, nullptr, 0, 0.0f, norm, as_stream(stream));
  PRL_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= prl_list_workspace_bytes(entries, count, 0),
              "prl_list_norm: workspace null, too small or not 16-B aligned");
  Coef* coef = static_cast<Coef*>(workspace);
  double* partial = reinterpret_cast<double*>(coef + count);
  int64_t n_partial = 0;
  if (int rc = launch_norm(entries, count, true, partial, &n_partial, as_stream(stream))) return rc;
  return launch_begin(entries, 0, nullptr, 0.0f, norm, partial, n_partial, coef, as_stream(stream));
}

extern "C" int prl_list_adamw(const prl_list_entry* entries, int64_t count, const prl_list_group* groups,
                              int64_t n_groups, float max_norm, float* norm, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  if (int rc = check_list("prl_list_adamw", entries, count)) return rc;
  if (count == 0 && norm == nullptr) return PRL_OK;
  PRL_REQUIRE(norm == nullptr || max_norm >= 0.0f, "prl_list_adamw: max_norm %g", (double)max_norm);
  PRL_REQUIRE((reinterpret_cast<uintptr_t>(norm) & 3u) == 0, "prl_list_adamw: norm not aligned to its type");
  PRL_REQUIRE(n_groups >= 0 && (n_groups == 0 || groups), "prl_list_adamw: null groups");
  for (int64_t g = 0; g < n_groups; ++g) {
    const prl_list_group& h = groups[g];
    PRL_REQUIRE(h.beta1 >= 0.0 && h.beta1 < 1.0 && h.beta2 >= 0.0 && h.beta2 < 1.0 && h.eps >= 0.0 &&
                    h.weight_decay >= 0.0 && (h.lr_dev != nullptr || h.lr >= 0.0),
                "prl_list_adamw: group %lld: lr, eps and weight_decay must not be negative, betas lie in [0, 1)", (long long)g);
    PRL_REQUIRE((reinterpret_cast<uintptr_t>(h.lr_dev) & 3u) == 0, "prl_list_adamw: group %lld: lr_dev not aligned to its type",
                (long long)g);
  }
  for (int64_t i = 0; i < count; ++i) {
    const prl_list_entry& e = entries[i];
    PRL_REQUIRE(e.numel <= L_MAX_BLOCKS * L_CHUNK8, "prl_list_adamw: tensor %lld: bad size %lld", (long long)i, (long long)e.numel);
    PRL_REQUIRE(e.bits == 32 || e.bits == 8, "prl_list_adamw: tensor %lld: moments in %d bits", (long long)i, (int)e.bits);
    PRL_REQUIRE(e.group >= 0 && e.group < n_groups, "prl_list_adamw: tensor %lld: group %lld of %lld", (long long)i,
                (long long)e.group, (long long)n_groups);
    PRL_REQUIRE(e.step, "prl_list_adamw: tensor %lld: null step", (long long)i);
    PRL_REQUIRE(e.master == nullptr || e.dtype != PRL_LIST_F32, "prl_list_adamw: tensor %lld: a float32 param has no master",
                (long long)i);
    if (e.numel == 0) continue;
    PRL_REQUIRE(e.param && e.exp_avg && e.second && (e.bits == 32 || (e.exp_avg_scale && e.second_scale)),
                "prl_list_adamw: tensor %lld: null pointer", (long long)i);
    const uintptr_t p = reinterpret_cast<uintptr_t>(e.param);
    const uintptr_t s = reinterpret_cast<uintptr_t>(e.exp_avg) | reinterpret_cast<uintptr_t>(e.second);
    const uintptr_t f = reinterpret_cast<uintptr_t>(e.master) | reinterpret_cast<uintptr_t>(e.exp_avg_scale) |
                        reinterpret_cast<uintptr_t>(e.second_scale) | reinterpret_cast<uintptr_t>(e.step);
    PRL_REQUIRE((p & (e.dtype == PRL_LIST_F32 ? 3u : 1u)) == 0 && (e.bits == 8 || (s & 3u) == 0) && (f & 3u) == 0,
                "prl_list_adamw: tensor %lld: a pointer not aligned to its type", (long long)i);
  }
  hipStream_t st = as_stream(stream);
  if (is_small(entries, count, n_groups)) return launch_small<true>(entries, count, groups, n_groups, max_norm, norm, st);
  PRL_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= prl_list_workspace_bytes(entries, count, n_groups),
              "prl_list_adamw: workspace null, too small or not 16-B aligned");
  Coef* coef = static_cast<Coef*>(workspace);
  double* partial = reinterpret_cast<double*>(coef + count);
  int64_t n_partial = 0;
  if (norm) {
    if (int rc = launch_norm(entries, count, false, partial, &n_partial, st)) return rc;
  }
  if (int rc = launch_begin(entries, count, groups, max_norm, norm, partial, n_partial, coef, st)) return rc;
  if (int rc = launch_adam32(entries, count, coef, st)) return rc;
  return launch_adam8(entries, count, coef, st);
}
