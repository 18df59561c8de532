// AdamW over many tensors at once, moments in 32 or 8 bits, with the global gradient norm, clipping and the skip of a
// step whose gradients are not finite.  See include/srx.h (srx_adamw_step) for the formulas and the buffers.
//
// Launches of one step: [norm pass over the gradients, 448 tensors a launch, or 896 whose gradients lie near each other] + one
// "prepare" workgroup (finishes the norm, advances the step counts, computes each tensor's bias-corrected constants) + the
// update, in as many launches, or one where the norm pass has left the addresses in device memory.  A small step without a
// norm is one launch in all.
// The gradients' addresses travel in the kernel arguments: they change from step to step (autograd allocates new
// gradients), and a table in device memory would need a host-to-device copy that a captured graph could not repeat.
//
// Bound: HBM.  702 tensors of together 16.9 M fp32 elements: norm pass 13 us, prepare 5 us, update 73 us (6.5 TB/s: part
// of the 474 MB stays in the last-level cache) with 32-bit moments, 50 us (5.4 TB/s) with 8-bit ones rounded to nearest, 62 us
// rounded at random (the hash and a division for each code).
#include <type_traits>
#include "srx_common.h"

namespace {

constexpr int BLOCK = SRX_ADAMW_BLOCK;          // elements that share one scale in the 8-bit moments
constexpr int CHUNK = SRX_ADAMW_CHUNK;          // elements of one tensor that one workgroup updates
constexpr int TPB = 256;
constexpr int MAX_GRADS = 448;                  // addresses per launch: 3.6 KB of the 4 KB of kernel arguments
constexpr int NEAR_GRADS = 896;                 // the same as 32-bit distances from the first in memory
constexpr int SMALL_GRADS = 128;                // addresses beside 32 groups of constants
constexpr int FLAT = 0, TABLE = -1;             // the other places of the gradients' addresses
constexpr int PREP_TENSORS = 16384;             // tensors per prepare launch: one bit each, 2 KB of kernel arguments
constexpr int PREP_TPB = 1024;
// Up to here a step without a norm is one launch.  Measured from the host, one launch against two: 12 tensors of 64 elements
// 9.0 us against 12.4, 100 chunks 11.0 against 14.1, 200 chunks 12.8 against 14.3, 400 chunks 20.7 against 14.0; replayed in a
// graph 5.1 against 5.9, 9.3 against 8.2, 12.6 against 8.9 (every workgroup adds to one counter).
constexpr int SMALL_CHUNKS = 64;

// The top 12 bits of a float are its exponent and three mantissa bits; 1.0 has 1016 there.  Code c > 0 stands for the
// float with base + c there: 127 signed codes reach from 1 down to 1.25 * 2^-16, 255 unsigned ones to 1.25 * 2^-32.
constexpr unsigned M_BASE = 889, V_BASE = 761;

struct Ctl { float factor; int skip; int arrived; int pad; };    // first 16 bytes of the coefficient workspace
struct Coef { float decay, step_size, root, eps, b1, ob1, b2, ob2; };

struct PrepArgs {
  const srx_adamw_tensor* tensors;
  int32_t* steps;
  float* coef;
  const double* partial;
  float* norm;
  double grad_scale, max_norm;
  int ntensors, t0, nchunks;
  int norm_mode;             // 0 none, 1 finish the norm here, 2 already finished by an earlier launch
  int skip_nonfinite;
  srx_adamw_group groups[SRX_ADAMW_MAX_GROUPS];
  uint32_t has_grad[PREP_TENSORS / 32];
};

// What the small form adds: the groups' constants, and who moves the step counts.
struct SmallArgs {
  int* arrived;
  double grad_scale;
  int ntensors;              // of this launch
  srx_adamw_group groups[SRX_ADAMW_MAX_GROUPS];
};
struct NoArgs {};
constexpr uint32_t NO_GRAD = ~0u;

template <int NG, bool SMALL = false> struct StepArgs {
  const srx_adamw_tensor* tensors;
  const srx_adamw_chunk* chunks;
  const float* coef;
  double* partial;
  void* m; void* v;
  float* m_scale; float* v_scale;
  int32_t* steps;            // step counts: moved by the prepare launch, or by the small form itself
  const void* flat;          // NG == FLAT: the flat gradient
  uint64_t* table;           // addresses in device memory, bit 0 set for bf16 (NG == TABLE: read; else written, if there)
  int chunk0, t0;
  int flat_dtype;
  uint64_t is_bf16[(NG + 63) / 64 + (NG <= 0)];
  uint64_t near_base;        // NG == NEAR_GRADS: gradient k is at near_base + (g[k] << near_shift), NO_GRAD: there is none
  int near_shift;
  std::conditional_t<NG == NEAR_GRADS, uint32_t, const void*> g[NG > 0 ? NG : 1];
  std::conditional_t<SMALL, SmallArgs, NoArgs> small;
};

static_assert(sizeof(StepArgs<MAX_GRADS>) <= 4096 && sizeof(StepArgs<NEAR_GRADS>) <= 4096 && sizeof(StepArgs<SMALL_GRADS, true>) <= 4096, "");

struct Grad { const void* p; bool bf; };
template <int NG, bool SMALL> __device__ __forceinline__ Grad grad_of(const StepArgs<NG, SMALL>& a, const srx_adamw_tensor& t, int ti) {
  Grad r;
  if constexpr (NG == FLAT) {
    r.bf = a.flat_dtype == SRX_BF16;
    r.p = static_cast<const char*>(a.flat) + t.g_off * (r.bf ? 2 : 4);
  } else if constexpr (NG == TABLE) {
    const uint64_t p = a.table[ti];
    r.bf = p & 1;
    r.p = reinterpret_cast<const void*>(p & ~1ull);
  } else {
    const int k = ti - a.t0;
    if constexpr (NG == NEAR_GRADS) r.p = a.g[k] == NO_GRAD ? nullptr : reinterpret_cast<const void*>(a.near_base + ((uint64_t)a.g[k] << a.near_shift));
    else r.p = a.g[k];
    r.bf = (a.is_bf16[k >> 6] >> (k & 63)) & 1;
  }
  return r;
}
// Four elements at any address that is a multiple of the element's size (views of a flat buffer start anywhere): global
// memory takes wide accesses there.
struct __attribute__((packed, aligned(4))) F4 { float e[4]; };
struct __attribute__((packed, aligned(2))) H4 { uint16_t e[4]; };
__device__ __forceinline__ float from_bf16(uint16_t h) { return __uint_as_float((uint32_t)h << 16); }
__device__ __forceinline__ uint16_t to_bf16(float f) { return __builtin_bit_cast(uint16_t, (bf16)f); }
// elements i .. i + 3 of a tensor (i < n; `full`: all of a wave's are there); zeros behind the end
__device__ __forceinline__ F4 load4(const float* p, int64_t i, int64_t n, bool full) {
  if (full) return *reinterpret_cast<const F4*>(p + i);
  F4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r.e[j] = i + j < n ? p[i + j] : 0.f;
  return r;
}
__device__ __forceinline__ F4 load4(const uint16_t* p, int64_t i, int64_t n, bool full) {
  F4 r;
  if (full) {
    const H4 h = *reinterpret_cast<const H4*>(p + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) r.e[j] = from_bf16(h.e[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) r.e[j] = i + j < n ? from_bf16(p[i + j]) : 0.f;
  }
  return r;
}
__device__ __forceinline__ F4 grad4(const Grad& g, int64_t i, int64_t n, bool full) {
  return g.bf ? load4(static_cast<const uint16_t*>(g.p), i, n, full) : load4(static_cast<const float*>(g.p), i, n, full);
}
__device__ __forceinline__ void store4(float* p, int64_t i, int64_t n, bool full, const F4& v) {
  if (full) {
    *reinterpret_cast<F4*>(p + i) = v;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < n) p[i + j] = v.e[j];
  }
}
__device__ __forceinline__ void store4(uint16_t* p, int64_t i, int64_t n, bool full, const F4& v) {
  if (full) {
    H4 h;
#pragma unroll
    for (int j = 0; j < 4; ++j) h.e[j] = to_bf16(v.e[j]);
    *reinterpret_cast<H4*>(p + i) = h;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < n) p[i + j] = to_bf16(v.e[j]);
  }
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// Non-negative floats order like their bits, and a NaN's bits are above every number's: one NaN or infinity in a
// block makes its scale, and with it the whole block, NaN, as it would make the 32-bit moments it touches.
template <int CTRL> __device__ __forceinline__ unsigned dpp_max(unsigned v) {
  const unsigned w = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
  return w > v ? w : v;
}
__device__ __forceinline__ unsigned wave_max_u(unsigned v) {
  v = dpp_max<0xB1>(v);          // quad_perm 1,0,3,2
  v = dpp_max<0x4E>(v);          // quad_perm 2,3,0,1
  v = dpp_max<0x141>(v);         // row_half_mirror
  v = dpp_max<0x140>(v);         // row_mirror
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = r[0] > r[1] ? r[0] : r[1];
  const auto q = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return q[0] > q[1] ? q[0] : q[1];
}

__device__ __forceinline__ float decode(unsigned k, unsigned base) { return k ? __uint_as_float((k + base) << 20) : 0.f; }
// |x| / s in [0, 1] -> nearest code (ties to even); below code 1: `least` (0 stays 0).  The second moment takes least = 1:
// a moment rounded down to 0 would leave only eps in the denominator of its update.
__device__ __forceinline__ unsigned encode(float t, unsigned base, unsigned least) {
  if (!(t > 0.f)) return 0;
  const unsigned b = __float_as_uint(t);
  const int c = (int)((b + 0x7FFFFu + ((b >> 20) & 1u)) >> 20) - (int)base;
  return c < (int)least ? least : (unsigned)c;
}

// sum of squares of one chunk of gradients, in 64 bits (a square can leave 32 bits' range, and the sum runs over
// millions of terms); a fixed order, so the norm is the same every time
template <int NG> __global__ __launch_bounds__(TPB) void adamw_norm_kernel(const StepArgs<NG> a) {
  const int c = a.chunk0 + blockIdx.x;
  const srx_adamw_chunk ch = a.chunks[c];
  const srx_adamw_tensor t = a.tensors[ch.tensor];
  const Grad g = grad_of(a, t, ch.tensor);
  if (NG != FLAT && a.table && ch.index == 0 && threadIdx.x == 0) a.table[ch.tensor] = reinterpret_cast<uint64_t>(g.p) | (g.bf ? 1 : 0);
  double s = 0;
  if (g.p) {
    const int64_t lo = (int64_t)ch.index * CHUNK + threadIdx.x * 4;
    const bool full = (int64_t)(ch.index + 1) * CHUNK <= t.n;
    F4 x[CHUNK / TPB / 4];
#pragma unroll
    for (int k = 0; k < CHUNK / TPB / 4; ++k) x[k] = grad4(g, lo + k * TPB * 4, t.n, full);
#pragma unroll
    for (int k = 0; k < CHUNK / TPB / 4; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) s = fma((double)x[k].e[j], (double)x[k].e[j], s);
  }
  __shared__ double part[TPB / 64];
  s = wave_sum_d(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) a.partial[c] = part[0] + part[1] + part[2] + part[3];
}

__device__ __forceinline__ double int_pow(double b, int n) {
  double r = 1;
  for (; n > 0; n >>= 1, b *= b)
    if (n & 1) r *= b;
  return r;
}

__device__ __forceinline__ Coef coef_of(const srx_adamw_group& g, int step) {
  Coef r;
  r.decay = (float)(1 - g.lr * g.weight_decay);
  r.step_size = (float)(g.lr / (1 - int_pow(g.beta1, step)));
  r.root = (float)(1 / sqrt(1 - int_pow(g.beta2, step)));
  r.eps = (float)g.eps;
  r.b1 = (float)g.beta1;
  r.ob1 = (float)(1 - g.beta1);
  r.b2 = (float)g.beta2;
  r.ob2 = (float)(1 - g.beta2);
  return r;
}

__global__ __launch_bounds__(PREP_TPB) void adamw_prepare_kernel(const PrepArgs a) {
  Ctl* ctl = reinterpret_cast<Ctl*>(a.coef);
  Coef* coef = reinterpret_cast<Coef*>(a.coef + 4);
  __shared__ double part[PREP_TPB / 64];
  __shared__ int skip_s;
  // everything that does not need the norm comes first, beside its loads: the thread's first tensor
  const int left = a.ntensors - a.t0 < PREP_TENSORS ? a.ntensors - a.t0 : PREP_TENSORS;
  const auto has = [&](int k) { return k < left && ((a.has_grad[k >> 5] >> (k & 31)) & 1); };
  const bool mine = has(threadIdx.x);
  int step = 0, group = 0;
  if (mine) {
    step = a.steps[a.t0 + threadIdx.x] + 1;
    group = a.tensors[a.t0 + threadIdx.x].group;
  }
  int skip = 0;
  if (a.norm_mode == 1) {
    // eight loads in flight: the sums come from other dies
    double s = 0;
    for (int i0 = threadIdx.x; i0 < a.nchunks; i0 += 8 * PREP_TPB) {
      double v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = i0 + j * PREP_TPB < a.nchunks ? a.partial[i0 + j * PREP_TPB] : 0.0;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      double total = 0;
      for (int i = 0; i < PREP_TPB / 64; ++i) total += part[i];
      total = sqrt(total) * fabs(a.grad_scale);
      double c = 1;
      if (a.max_norm > 0) {
        c = a.max_norm / (total + 1e-6);
        c = c > 1 ? 1 : c;                       // a NaN norm stays NaN and reaches every parameter, as in torch
      }
      const bool finite = total - total == 0;
      skip_s = a.skip_nonfinite && !finite;
      ctl->factor = (float)(a.grad_scale * c);
      ctl->skip = skip_s;
      a.norm[0] = (float)total;
    }
  } else if (a.norm_mode == 2) {
    skip = ctl->skip;
  } else if (threadIdx.x == 0) {
    ctl->factor = (float)a.grad_scale;
    ctl->skip = 0;
  }
  Coef first;
  if (mine) first = coef_of(a.groups[group], step);
  if (a.norm_mode == 1) {
    __syncthreads();
    skip = skip_s;
  }
  if (skip) return;
  if (mine) {
    a.steps[a.t0 + threadIdx.x] = step;
    coef[a.t0 + threadIdx.x] = first;
  }
  for (int k = threadIdx.x + PREP_TPB; k < left; k += PREP_TPB) {
    if (!has(k)) continue;
    const int i = a.t0 + k;
    const int n = a.steps[i] + 1;
    a.steps[i] = n;
    coef[i] = coef_of(a.groups[a.tensors[i].group], n);
  }
}

// The moments' new values, each operation rounded on its own: the 8-bit codes are then the same whatever code computes
// them (a fused multiply-add would move one value in ten million to the neighbouring code, a tenth away).
__device__ __forceinline__ void moments(float& m, float& v, float g, const Coef& c) {
#pragma clang fp contract(off)
  const float mg = g * c.ob1, gg = g * g;
  m = m * c.b1;
  m = m + mg;
  const float vg = gg * c.ob2;
  v = v * c.b2;
  v = v + vg;
}
// The hardware's square root and reciprocal are within 2^-23 of the value: 2^-21 of the update at most, which is itself
// far below the parameter.  The root takes a denormal for zero: 2^-63 root of the denominator, below 2^-21 of it where eps is at
// least 2^-42 root (2.3e-13, 7.2e-12 at a first step with beta2 = 0.999); a smaller eps gets the exact forms.
__device__ __forceinline__ float updated(float w, float m, float v, const Coef& c, bool fast) {
  const float u = fast ? m * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v) * c.root + c.eps) : m / (sqrtf(v) * c.root + c.eps);
  return w * c.decay - c.step_size * u;
}
// Codes of four values x against a block's largest, s: the nearest code of the correctly rounded quotient |x| / s.  The
// reciprocal's product is within 3 units of it, so it gives the same code unless it lies that close to the middle
// between two codes (about one block in 500): then the divisions are made.
template <bool SIGNED> __device__ __forceinline__ uint32_t encode4(const float* x, float s) {
  constexpr unsigned base = SIGNED ? M_BASE : V_BASE, least = SIGNED ? 0 : 1;
  const float r = __builtin_amdgcn_rcpf(s);
  unsigned t[4], middle = ~0u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    t[j] = __float_as_uint(fabsf(x[j]) * r);
    const unsigned d = (t[j] << 12) + (0x80004u << 12);      // distance from four units below the middle, in the top 20 bits
    middle = d < middle ? d : middle;
  }
  uint32_t out = 0;
  if (__any(!(s > 1e-30f && s < 1e30f) || middle < (8u << 12))) {           // (or a reciprocal that is no normal number)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      unsigned c = encode(fabsf(x[j]) / s, base, least);
      if (SIGNED) c |= c && x[j] < 0 ? 128u : 0u;   // a first moment that rounds to 0 loses its sign: one code for each value
      out |= c << (8 * j);
    }
    return out;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    int c = (int)(t[j] + (0x80000u - (base << 20))) >> 20;   // no ties here
    c = c > (int)least ? c : (int)least;
    if (SIGNED) c |= (c + 127) & (__float_as_uint(x[j]) >> 24) & 128;       // the sign, where c > 0
    else c = t[j] ? c : 0;
    out |= (unsigned)c << (8 * j);
  }
  return out;
}

// 32 bits that depend on every bit of a quad of elements (its number in the whole state), a step count and a salt: rounds of
// a shift, an exclusive or and a product, with the odd numbers at 2^32 times the fractional parts of the roots of 3, 5 and 7.
__device__ __forceinline__ uint32_t random_word(int64_t quad, uint32_t step, uint32_t salt) {
  uint32_t h = (uint32_t)quad ^ ((uint32_t)(quad >> 32) * 0xA54FF53Bu) ^ ((4 * step + salt) * 0xBB67AE85u);
  h = (h ^ (h >> 16)) * 0x3C6EF373u;
  h = (h ^ (h >> 15)) * 0xBB67AE85u;
  h = (h ^ (h >> 16)) * 0xA54FF53Bu;
  return h ^ (h >> 15);
}
// Codes of four values, rounded up or down at random with the mean that the value has: 16 random bits, in the middle of the 20
// that a code drops, are added to the correctly rounded quotient before they go.  Between two codes a float's bits are
// linear in its value, and no quotient is above 1, so nothing carries past the last code.
template <bool SIGNED> __device__ __forceinline__ uint32_t encode4_random(const float* x, float s, int64_t quad, uint32_t step) {
  constexpr unsigned base = SIGNED ? M_BASE : V_BASE;
  constexpr float smallest = SIGNED ? 1.25f * 0x1p-16f : 1.25f * 0x1p-32f;
  const uint32_t r[2] = {random_word(quad, step, SIGNED ? 0 : 2), random_word(quad, step, SIGNED ? 1 : 3)};
  uint32_t out = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float t = fabsf(x[j]) / s;
    const uint32_t add = ((r[j / 2] >> (16 * (j & 1))) & 0xFFFFu) << 4 | 8u;
    unsigned c = ((__float_as_uint(t) + add) >> 20) - base;
    if (t < smallest) c = !SIGNED || (float)add < t * (0x1p20f / smallest);
    if (!(t > 0.f)) c = 0;
    if (SIGNED) c |= c && x[j] < 0 ? 128u : 0u;
    out |= c << (8 * j);
  }
  return out;
}

// A wave takes whole blocks of 256, four elements a lane, so that a block's largest is a wave's.  All of a wave's four
// blocks are read before the first is computed: a workgroup's only other wait is for the tables in front of them.
template <int BITS, int NG, bool SMALL, bool RANDOM> __device__ __forceinline__ void update_chunk(const StepArgs<NG, SMALL>& a) {
  const Ctl* ctl = reinterpret_cast<const Ctl*>(a.coef);
  if (!SMALL && ctl->skip) return;
  const srx_adamw_chunk ch = a.chunks[a.chunk0 + blockIdx.x];
  const srx_adamw_tensor t = a.tensors[ch.tensor];
  const Grad g = grad_of(a, t, ch.tensor);
  if (!g.p) return;
  Coef c;
  float factor;
  if constexpr (SMALL) {
    factor = (float)a.small.grad_scale;
    c = coef_of(a.small.groups[t.group], a.steps[ch.tensor] + 1);
  } else {
    factor = ctl->factor;
    c = reinterpret_cast<const Coef*>(a.coef + 4)[ch.tensor];
  }
  const uint32_t step = RANDOM ? (uint32_t)a.steps[ch.tensor] + SMALL : 0;       // of this step
  const bool fast = c.eps >= 0x1p-42f * c.root;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int NB = CHUNK / BLOCK / (TPB / 64);
  const int64_t lo = (int64_t)ch.index * CHUNK + wave * NB * BLOCK;        // the wave's first element in its tensor
  const int64_t blk = t.first_block + lo / BLOCK;
  F4 w[NB], gr[NB], m[NB], v[NB];
  uint32_t mc[NB], vc[NB];
  float ms[NB], vs[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int64_t i = lo + b * BLOCK + lane * 4, s = (blk + b) * BLOCK + lane * 4;
    if (lo + b * BLOCK >= t.n) break;
    const bool full = lo + (b + 1) * BLOCK <= t.n;
    gr[b] = grad4(g, i, t.n, full);
    if (t.master) w[b] = load4(t.master, i, t.n, full);
    else w[b] = load4(static_cast<const float*>(t.p), i, t.n, full);
    if constexpr (BITS == 8) {
      mc[b] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.m) + s);
      vc[b] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.v) + s);
      ms[b] = a.m_scale[blk + b];
      vs[b] = a.v_scale[blk + b];
    } else {
      m[b] = *reinterpret_cast<const F4*>(static_cast<const float*>(a.m) + s);
      v[b] = *reinterpret_cast<const F4*>(static_cast<const float*>(a.v) + s);
    }
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int64_t i = lo + b * BLOCK + lane * 4, s = (blk + b) * BLOCK + lane * 4;
    if (lo + b * BLOCK >= t.n) break;
    const bool full = lo + (b + 1) * BLOCK <= t.n;
    if (t.master) {
      // the parameter is what the user sees and may have written: where it is not the master's rounding, it wins
      const F4 p = load4(static_cast<const uint16_t*>(t.p), i, t.n, full);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[b].e[j] = from_bf16(to_bf16(w[b].e[j])) == p.e[j] ? w[b].e[j] : p.e[j];
    }
    unsigned mmax = 0, vmax = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (BITS == 8) {
        const unsigned mk = (mc[b] >> (8 * j)) & 255, vk = (vc[b] >> (8 * j)) & 255;
        const float x = decode(mk & 127, M_BASE) * ms[b];
        m[b].e[j] = mk & 128 ? -x : x;
        v[b].e[j] = decode(vk, V_BASE) * vs[b];
      }
      float gi;
      {
#pragma clang fp contract(off)
        gi = gr[b].e[j] * factor;
      }
      moments(m[b].e[j], v[b].e[j], gi, c);
      w[b].e[j] = updated(w[b].e[j], m[b].e[j], v[b].e[j], c, fast);
      if constexpr (BITS == 8) {
        // (behind the tensor's end everything is zero and stays zero, unless the block is not finite)
        const unsigned mb = __float_as_uint(m[b].e[j]) & 0x7FFFFFFFu, vb = __float_as_uint(v[b].e[j]) & 0x7FFFFFFFu;
        mmax = mb > mmax ? mb : mmax;
        vmax = vb > vmax ? vb : vmax;
      }
    }
    if (t.master) {
      store4(t.master, i, t.n, full, w[b]);
      store4(static_cast<uint16_t*>(t.p), i, t.n, full, w[b]);
    } else {
      store4(static_cast<float*>(t.p), i, t.n, full, w[b]);
    }
    if constexpr (BITS == 32) {
      *reinterpret_cast<F4*>(static_cast<float*>(a.m) + s) = m[b];
      *reinterpret_cast<F4*>(static_cast<float*>(a.v) + s) = v[b];
    } else {
      const float nm = __uint_as_float(wave_max_u(mmax)), nv = __uint_as_float(wave_max_u(vmax));
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.m) + s) = RANDOM ? encode4_random<true>(m[b].e, nm, s / 4, step) : encode4<true>(m[b].e, nm);
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.v) + s) = RANDOM ? encode4_random<false>(v[b].e, nv, s / 4, step) : encode4<false>(v[b].e, nv);
      if (lane == 0) { a.m_scale[blk + b] = nm; a.v_scale[blk + b] = nv; }
    }
  }
}

// The small form is a step in one launch: each workgroup computes its tensor's constants itself, and the last one to
// arrive, after every other has read its step count, moves the counts and clears the counter for the next launch.
template <int BITS, int NG, bool SMALL, bool RANDOM> __global__ __launch_bounds__(TPB) void adamw_step_kernel(const StepArgs<NG, SMALL> a) {
  update_chunk<BITS, NG, SMALL, RANDOM>(a);
  if constexpr (SMALL) {
    __shared__ int last;
    __syncthreads();                                  // all waves of this workgroup have read their step count
    if (threadIdx.x == 0) {
      last = __hip_atomic_fetch_add(a.small.arrived, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
      if (last) __hip_atomic_store(a.small.arrived, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last) return;
    for (int k = threadIdx.x; k < a.small.ntensors; k += TPB) {
      bool has = true;
      if constexpr (NG != FLAT) has = a.g[k] != nullptr;
      if (has) a.steps[a.t0 + k] += 1;
    }
  }
}

// one wave per block of 256
__global__ __launch_bounds__(TPB) void moments_to8_kernel(const float* m, const float* v, uint8_t* mc, uint8_t* vc, float* ms,
                                                          float* vs, int64_t nblocks) {
  const int64_t blk = (int64_t)blockIdx.x * (TPB / 64) + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (blk >= nblocks) return;
  const int64_t s = blk * BLOCK + lane * 4;
  const f32x4 a = *reinterpret_cast<const f32x4*>(m + s), b = *reinterpret_cast<const f32x4*>(v + s);
  unsigned am = 0, bm = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned x = __float_as_uint(a[j]) & 0x7FFFFFFFu, y = __float_as_uint(b[j]) & 0x7FFFFFFFu;
    am = x > am ? x : am;
    bm = y > bm ? y : bm;
  }
  const float sm = __uint_as_float(wave_max_u(am)), sv = __uint_as_float(wave_max_u(bm));
  const float xm[4] = {a[0], a[1], a[2], a[3]}, xv[4] = {b[0], b[1], b[2], b[3]};
  const uint32_t cm = encode4<true>(xm, sm), cv = encode4<false>(xv, sv);
  *reinterpret_cast<uint32_t*>(mc + s) = cm;
  *reinterpret_cast<uint32_t*>(vc + s) = cv;
  if (lane == 0) { ms[blk] = sm; vs[blk] = sv; }
}

__global__ __launch_bounds__(TPB) void moments_from8_kernel(const uint8_t* mc, const uint8_t* vc, const float* ms, const float* vs,
                                                            float* m, float* v, int64_t nblocks) {
  const int64_t blk = (int64_t)blockIdx.x * (TPB / 64) + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (blk >= nblocks) return;
  const int64_t s = blk * BLOCK + lane * 4;
  const uint32_t cm = *reinterpret_cast<const uint32_t*>(mc + s), cv = *reinterpret_cast<const uint32_t*>(vc + s);
  const float sm = ms[blk], sv = vs[blk];
  f32x4 a, b;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned x = (cm >> (8 * j)) & 255, y = (cv >> (8 * j)) & 255;
    const float z = decode(x & 127, M_BASE) * sm;
    a[j] = x & 128 ? -z : z;
    b[j] = decode(y, V_BASE) * sv;
  }
  *reinterpret_cast<f32x4*>(m + s) = a;
  *reinterpret_cast<f32x4*>(v + s) = b;
}

int check_moments(const char* what, const void* a, const void* b, const void* c, const void* d, const void* e, const void* f,
                  int64_t nblocks) {
  SRX_CHECK_ARG(nblocks >= 0 && nblocks < (1LL << 33), "%s: nblocks %lld out of range", what, (long long)nblocks);
  SRX_CHECK_ARG(nblocks == 0 || (a && b && c && d && e && f), "%s: null pointer", what);
  SRX_CHECK_ARG(((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) % 16 == 0, "%s: moments must be 16-byte aligned", what);
  return SRX_OK;
}

// Addresses as 32-bit distances from the first, in units of what all distances are multiples of (512 bytes for tensors of
// their own): twice as many fit into a launch.
struct Near {
  uint64_t base = ~0ull;
  int shift = 0;
  static bool there(const srx_adamw_desc* d, int i) { return d->grads[i] && d->chunk_start[i + 1] > d->chunk_start[i]; }
  bool fits(const srx_adamw_desc* d) {
    uint64_t last = 0, any = 0;
    for (int i = 0; i < d->ntensors; ++i)
      if (there(d, i)) {
        const uint64_t p = reinterpret_cast<uint64_t>(d->grads[i]);
        base = p < base ? p : base;
        last = p > last ? p : last;
      }
    for (int i = 0; i < d->ntensors; ++i)
      if (there(d, i)) any |= reinterpret_cast<uint64_t>(d->grads[i]) - base;
    if (!any) return true;
    shift = __builtin_ctzll(any);
    return (last - base) >> shift < NO_GRAD;
  }
  uint32_t of(const srx_adamw_desc* d, int i) const {
    return there(d, i) ? (uint32_t)((reinterpret_cast<uint64_t>(d->grads[i]) - base) >> shift) : NO_GRAD;
  }
};

template <int NG, bool SMALL = false> StepArgs<NG, SMALL> step_args(const srx_adamw_desc* d, const Near& near, int t0, int t1) {
  StepArgs<NG, SMALL> a = {};
  a.tensors = d->tensors; a.chunks = d->chunks; a.coef = d->coef; a.partial = d->partial;
  a.m = d->m; a.v = d->v; a.m_scale = d->m_scale; a.v_scale = d->v_scale; a.steps = d->steps;
  a.flat = d->flat_grad; a.flat_dtype = d->flat_dtype; a.chunk0 = d->chunk_start[t0]; a.t0 = t0;
  if (NG == TABLE || (NG > 0 && d->ntensors > NG)) a.table = reinterpret_cast<uint64_t*>(d->coef + 4 + 8 * (int64_t)d->ntensors);
  if constexpr (NG == NEAR_GRADS) { a.near_base = near.base; a.near_shift = near.shift; }
  if constexpr (NG > 0)
    for (int k = 0; k < t1 - t0; ++k) {
      if constexpr (NG == NEAR_GRADS) a.g[k] = near.of(d, t0 + k);
      else a.g[k] = d->grads[t0 + k];
      if (d->grad_dtypes && d->grad_dtypes[t0 + k] == SRX_BF16) a.is_bf16[k >> 6] |= 1ull << (k & 63);
    }
  return a;
}

// One pass over the tensors in launches of at most NG gradients, `fn(args, chunks)` each.
template <int NG, typename F> int each_launch(const srx_adamw_desc* d, const Near& near, F fn) {
  const int per = NG > 0 ? NG : d->ntensors;
  for (int t0 = 0; t0 < d->ntensors; t0 += per) {
    const int t1 = t0 + per < d->ntensors ? t0 + per : d->ntensors;
    const int n = d->chunk_start[t1] - d->chunk_start[t0];
    if (n <= 0) continue;
    if (int rc = fn(step_args<NG>(d, near, t0, t1), n)) return rc;
  }
  return SRX_OK;
}

template <int NG, bool SMALL> int launch_step(const srx_adamw_desc* d, const StepArgs<NG, SMALL>& a, int n, hipStream_t s) {
  if (d->state_bits == 32) hipLaunchKernelGGL((adamw_step_kernel<32, NG, SMALL, false>), dim3(n), dim3(TPB), 0, s, a);
  else if (d->rounding) hipLaunchKernelGGL((adamw_step_kernel<8, NG, SMALL, true>), dim3(n), dim3(TPB), 0, s, a);
  else hipLaunchKernelGGL((adamw_step_kernel<8, NG, SMALL, false>), dim3(n), dim3(TPB), 0, s, a);
  return srx_check_launch("adamw_step");
}

template <int NG> int small_launch(const srx_adamw_desc* d, hipStream_t s) {
  StepArgs<NG, true> a = step_args<NG, true>(d, {}, 0, d->ntensors);
  a.small.arrived = &reinterpret_cast<Ctl*>(d->coef)->arrived;
  a.small.grad_scale = d->grad_scale;
  a.small.ntensors = d->ntensors;
  for (int g = 0; g < d->ngroups; ++g) a.small.groups[g] = d->groups[g];
  return launch_step(d, a, d->chunk_start[d->ntensors], s);
}

template <int NG> int step_launches(const srx_adamw_desc* d, const Near& near, hipStream_t s) {
  const int norm = d->max_norm > 0 || d->skip_nonfinite, chunks = d->chunk_start[d->ntensors];
  if (!norm && chunks > 0 && chunks <= SMALL_CHUNKS) {
    if constexpr (NG == FLAT) return small_launch<FLAT>(d, s);
    else if (NG == MAX_GRADS && d->ntensors <= SMALL_GRADS) return small_launch<SMALL_GRADS>(d, s);
  }
  if (norm) {
    int rc = each_launch<NG>(d, near, [&](const StepArgs<NG>& a, int n) {
      hipLaunchKernelGGL(adamw_norm_kernel<NG>, dim3(n), dim3(TPB), 0, s, a);
      return srx_check_launch("adamw_norm");
    });
    if (rc) return rc;
  }
  for (int t0 = 0; t0 < d->ntensors; t0 += PREP_TENSORS) {
    PrepArgs p = {};
    p.tensors = d->tensors; p.steps = d->steps; p.coef = d->coef; p.partial = d->partial; p.norm = d->norm;
    p.grad_scale = d->grad_scale; p.max_norm = d->max_norm; p.ntensors = d->ntensors; p.t0 = t0;
    p.nchunks = chunks;
    p.norm_mode = !norm ? 0 : t0 ? 2 : 1;
    p.skip_nonfinite = d->skip_nonfinite;
    for (int g = 0; g < d->ngroups; ++g) p.groups[g] = d->groups[g];
    for (int k = 0; k < PREP_TENSORS && t0 + k < d->ntensors; ++k)
      if (NG == FLAT || d->grads[t0 + k]) p.has_grad[k >> 5] |= 1u << (k & 31);
    hipLaunchKernelGGL(adamw_prepare_kernel, dim3(1), dim3(PREP_TPB), 0, s, p);
    if (int rc = srx_check_launch("adamw_prepare")) return rc;
  }
  const auto step = [&](const auto& a, int n) { return launch_step(d, a, n, s); };
  // the norm pass has left the addresses in device memory: the update needs no second launch for them
  if (NG > 0 && norm && d->ntensors > NG) return each_launch<TABLE>(d, near, step);
  return each_launch<NG>(d, near, step);
}

}  // namespace

extern "C" {

int srx_adamw_step(const srx_adamw_desc* d, void* stream) {
  SRX_CHECK_ARG(d != nullptr, "srx_adamw_step: null descriptor");
  SRX_CHECK_ARG(d->state_bits == 32 || d->state_bits == 8, "srx_adamw_step: state_bits must be 32 or 8, got %d", d->state_bits);
  SRX_CHECK_ARG(d->rounding == 0 || (d->rounding == 1 && d->state_bits == 8), "srx_adamw_step: rounding must be 0, or 1 with 8 bits, got %d", d->rounding);
  SRX_CHECK_ARG(d->ntensors > 0, "srx_adamw_step: ntensors must be positive");
  SRX_CHECK_ARG(d->ngroups > 0 && d->ngroups <= SRX_ADAMW_MAX_GROUPS, "srx_adamw_step: %d groups, 1 to %d are supported",
                d->ngroups, SRX_ADAMW_MAX_GROUPS);
  SRX_CHECK_ARG(d->tensors && d->chunks && d->chunk_start && d->groups && d->steps && d->coef, "srx_adamw_step: null table");
  SRX_CHECK_ARG((d->grads != nullptr) != (d->flat_grad != nullptr), "srx_adamw_step: give either grads or flat_grad");
  SRX_CHECK_ARG(!d->flat_grad || d->flat_dtype == SRX_BF16 || d->flat_dtype == SRX_F32, "srx_adamw_step: bad flat_dtype %d", d->flat_dtype);
  SRX_CHECK_ARG((uintptr_t)d->flat_grad % (d->flat_dtype == SRX_BF16 ? 2 : 4) == 0, "srx_adamw_step: flat_grad is not aligned to its type");
  SRX_CHECK_ARG(d->m && d->v && (d->state_bits == 32 || (d->m_scale && d->v_scale)), "srx_adamw_step: null moments");
  SRX_CHECK_ARG(((uintptr_t)d->m | (uintptr_t)d->v) % 16 == 0, "srx_adamw_step: moments must be 16-byte aligned");
  SRX_CHECK_ARG(!(d->max_norm < 0) && d->max_norm == d->max_norm, "srx_adamw_step: max_norm must not be negative or NaN");
  SRX_CHECK_ARG(!(d->max_norm > 0 || d->skip_nonfinite) || (d->partial && d->norm), "srx_adamw_step: the norm needs partial and norm");
  SRX_CHECK_ARG(d->grad_scale - d->grad_scale == 0, "srx_adamw_step: grad_scale must be finite");
  SRX_CHECK_ARG(d->chunk_start[0] == 0, "srx_adamw_step: chunk_start must begin at 0");
  for (int i = 0; i < d->ntensors; ++i) {
    SRX_CHECK_ARG(d->chunk_start[i + 1] >= d->chunk_start[i], "srx_adamw_step: chunk_start must not decrease (tensor %d)", i);
    SRX_CHECK_ARG(!d->grad_dtypes || d->grad_dtypes[i] == SRX_BF16 || d->grad_dtypes[i] == SRX_F32,
                  "srx_adamw_step: bad gradient dtype %d of tensor %d", d->grad_dtypes[i], i);
    if (d->grads)
      SRX_CHECK_ARG((uintptr_t)d->grads[i] % (d->grad_dtypes && d->grad_dtypes[i] == SRX_BF16 ? 2 : 4) == 0,
                    "srx_adamw_step: gradient %d is not aligned to its type", i);
  }
  for (int g = 0; g < d->ngroups; ++g) {
    const srx_adamw_group& q = d->groups[g];
    SRX_CHECK_ARG(q.beta1 >= 0 && q.beta1 < 1 && q.beta2 >= 0 && q.beta2 < 1 && q.eps >= 0 && q.lr >= 0 && q.weight_decay >= 0 &&
                      q.lr - q.lr == 0 && q.weight_decay - q.weight_decay == 0 && q.eps - q.eps == 0,
                  "srx_adamw_step: bad hyper-parameters in group %d (lr %g, betas %g %g, eps %g, weight_decay %g)", g, q.lr,
                  q.beta1, q.beta2, q.eps, q.weight_decay);
  }
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  Near near;
  if (d->flat_grad) return step_launches<FLAT>(d, near, s);
  if (d->ntensors > MAX_GRADS && near.fits(d)) return step_launches<NEAR_GRADS>(d, near, s);
  return step_launches<MAX_GRADS>(d, near, s);
}

int srx_adamw_moments_to8(const float* m, const float* v, void* m_code, void* v_code, float* m_scale, float* v_scale,
                          int64_t nblocks, void* stream) {
  if (int rc = check_moments("srx_adamw_moments_to8", m, v, m_code, v_code, m_scale, v_scale, nblocks)) return rc;
  if (nblocks == 0) return SRX_OK;
  hipLaunchKernelGGL(moments_to8_kernel, dim3((unsigned)((nblocks + 3) / 4)), dim3(TPB), 0, reinterpret_cast<hipStream_t>(stream), m, v,
                     (uint8_t*)m_code, (uint8_t*)v_code, m_scale, v_scale, nblocks);
  return srx_check_launch("moments_to8");
}

int srx_adamw_moments_from8(const void* m_code, const void* v_code, const float* m_scale, const float* v_scale, float* m,
                            float* v, int64_t nblocks, void* stream) {
  if (int rc = check_moments("srx_adamw_moments_from8", m, v, m_code, v_code, m_scale, v_scale, nblocks)) return rc;
  if (nblocks == 0) return SRX_OK;
  hipLaunchKernelGGL(moments_from8_kernel, dim3((unsigned)((nblocks + 3) / 4)), dim3(TPB), 0, reinterpret_cast<hipStream_t>(stream),
                     (const uint8_t*)m_code, (const uint8_t*)v_code, m_scale, v_scale, m, v, nblocks);
  return srx_check_launch("moments_from8");
}

}  // extern "C"
