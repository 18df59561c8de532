// Norms over the channels before and after a residual branch, fused with the branch's gate, the residual scale and the
// residual add (include/srx.h, srx_resnorm_forward / _backward, has the formulas).
//
// One kernel body serves both layouts.  A thread holds K x V elements of each tensor in registers:
//   rows   (channels contiguous): V neighbouring channels, K times, of ONE row; `lanes` threads share a row.
//   planes (pixels contiguous):   V neighbouring pixels of K channels; `lanes` threads of a wave sit side by side
//                                 along the pixels, the others hold other channels of the same pixels.
// Every tensor is read once: statistics, norm and gradients come out of the registers, in fp32.  The backward pass takes
// x and f and forms y again: the same traffic as reading y, and not y's rounding to bf16 (which would put 2^-9 of
// error into every weight gradient).  The sums over the pixels (gradients of weights, biases and gates) stay in registers
// while a workgroup walks its share of the pixels; their partial sums are joined by a second small kernel in a fixed
// order (no atomics: same inputs, same bits).
#include "srx_common.h"

namespace {

constexpr int MAX_Q = 2;          // quantities reduced together
enum { KIND_NONE = 0, KIND_RMS = 1, KIND_LAYER = 2 };
enum { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_IMAGE = 2, GATE_FULL = 3 };

struct Args {
  srx_resnorm_desc d;
  int lanes;            // rows: threads per row (a power of two); planes: lanes along the pixels (64 down to 4)
  int slices;           // shares of an image's pixels
  int64_t len;          // pixels of a share
  int64_t items;        // images * slices
  int64_t P;            // pixels of an "image" (rows without per-image gate: all rows are one image)
  float* part_pre;      // [workgroups][2][C]
  float* part_post;     // [workgroups or items][2][C]
};

// V elements, at any address that is a multiple of the element's size: global memory takes wide accesses there (a row
// of an odd number of channels, a map of an odd number of pixels), so there is no second, narrow form of the kernels.
template <typename T, int V> struct __attribute__((packed, aligned(sizeof(T)))) Vec { T e[V]; };
__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + __expf(-x)); }

template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
// sum over the lanes whose numbers differ in the bits lo, 2 lo, ... hi / 2 (every lane gets it)
__device__ __forceinline__ float lanes_sum(float v, int lo, int hi) {
  if (lo <= 1 && hi > 1) v = dpp_add<0xB1>(v);          // quad_perm 1,0,3,2
  if (lo <= 2 && hi > 2) v = dpp_add<0x4E>(v);          // quad_perm 2,3,0,1
  if (lo <= 4 && hi > 4) v += __shfl_xor(v, 4, 64);
  if (lo <= 8 && hi > 8) v = dpp_add<0x128>(v);         // row_ror 8
  if (lo <= 16 && hi > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (lo <= 32 && hi > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// UNI: all lanes of a wave hold the same channels (planes with 64 lanes along the pixels): weights in scalar registers
template <typename T, bool ROWS, int K, int V, bool UNI> struct Thread {
  static constexpr int E = K * V;                     // elements of each tensor
  static constexpr int NP = ROWS ? 1 : V;             // pixels
  static constexpr int NW = ROWS ? E : K;             // channels
  static __device__ __forceinline__ constexpr int pix(int e) { return ROWS ? 0 : e % V; }
  static __device__ __forceinline__ constexpr int wi(int e) { return ROWS ? e : e / V; }
  typedef Vec<T, V> Raw;

  const Args& a;
  float* lds;
  int round;
  int lane, wave, l, grp;     // rows: l = thread within the row, grp = row of the workgroup; planes: l = lane along the pixels
  int have;                   // elements of a vector that exist: planes, along the pixels; rows: 0 where the row does not exist
  bool full;                  // every element of the wave exists
  int64_t image, base;        // first pixel of the workgroup's tile within the image

  __device__ __forceinline__ Thread(const Args& a_, float* lds_) : a(a_), lds(lds_), round(0) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    l = ROWS ? threadIdx.x & (a.lanes - 1) : lane & (a.lanes - 1);
    grp = UNI ? wave : threadIdx.x / a.lanes;
  }
  __device__ __forceinline__ int chan(int k) const { return ROWS ? (k * a.lanes + l) * V : grp * K + k; }
  // elements of step k that exist
  __device__ __forceinline__ int exist(int k) const {
    const int left = a.d.C - chan(k);
    if (ROWS) return !have || left < 0 ? 0 : left < V ? left : V;
    return left > 0 ? have : 0;
  }
  // whether an element's channel exists (its pixel need not)
  __device__ __forceinline__ bool chan_ok(int e) const { return chan(e / V) + (ROWS ? e % V : 0) < a.d.C; }
  // pixels that a workgroup takes at a time
  __device__ __forceinline__ int tile() const { return ROWS ? (int)blockDim.x / a.lanes : a.lanes * V; }
  __device__ __forceinline__ void at(int64_t img, int64_t base_, int64_t end) {
    image = img;
    base = base_;
    const int64_t left = end - base - (ROWS ? grp : l * V);
    have = left <= 0 ? 0 : ROWS || left >= V ? V : (int)left;
    full = __all(have == V && (ROWS ? chan(K - 1) + V : chan(K - 1) + 1) <= a.d.C);
  }
  // address of step 0, and elements from one step to the next: a uniform part and an offset within the workgroup's tile
  template <typename P> __device__ __forceinline__ P* first(P* p, int64_t stride) const {
    if (ROWS) return p + (image * a.P + base) * stride + ((int64_t)grp * stride + l * V);
    if (UNI) return p + image * stride + (int64_t)(wave * K) * a.P + base;
    return p + image * stride + base + ((int64_t)(grp * K) * a.P + l * V);
  }
  __device__ __forceinline__ int64_t step() const { return ROWS ? a.lanes * V : a.P; }
  __device__ __forceinline__ void read(const void* p, int64_t stride, Raw* z) const {
    const T* q = first(static_cast<const T*>(p), stride);
    const unsigned off = UNI ? l * V : 0;
    if (full) {
#pragma unroll
      for (int k = 0; k < K; ++k) z[k] = *reinterpret_cast<const Raw*>(q + k * step() + off);
      return;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const T* w = q + k * step() + off;
      const int n = exist(k);
      if (n == V) z[k] = *reinterpret_cast<const Raw*>(w);
      else
#pragma unroll
        for (int j = 0; j < V; ++j) z[k].e[j] = j < n ? w[j] : (T)0.f;
    }
  }
  __device__ __forceinline__ void write(void* p, int64_t stride, const float* v) const {
    T* q = first(static_cast<T*>(p), stride);
    const unsigned off = UNI ? l * V : 0;
    if (full) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        Raw z;
#pragma unroll
        for (int j = 0; j < V; ++j) z.e[j] = (T)v[k * V + j];
        *reinterpret_cast<Raw*>(q + k * step() + off) = z;
      }
      return;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      T* w = q + k * step() + off;
      const int n = exist(k);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < n) w[j] = (T)v[k * V + j];
    }
  }
  // per-channel fp32 values (NULL: `missing`); channels that do not exist get 0
  __device__ __forceinline__ float weight(const float* w, float missing, int i) const {
    const int c = ROWS ? chan(i / V) + i % V : chan(i);
    return c >= a.d.C ? 0.f : w ? w[c] : missing;
  }
  static __device__ __forceinline__ float uniform(float v) {
    return UNI ? __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v))) : v;
  }
  // the branch's factor and offset: u = gw n + gb (a full gate multiplies that per element)
  __device__ __forceinline__ void branch(int64_t img, float* gw, float* gb) const {
    const srx_resnorm_desc& d = a.d;
    const float* gate = d.gate_mode == GATE_CHANNEL || d.gate_mode == GATE_IMAGE
                            ? static_cast<const float*>(d.gate) + (d.gate_mode == GATE_IMAGE ? img * d.C : 0) : nullptr;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      float G = weight(gate, 1.f, i);
      if (gate && d.gate_act) G = sigmoid(G);
      G *= d.scale;
      gw[i] = uniform(G * weight(d.w_post, 1.f, i));
      gb[i] = uniform(G * weight(d.b_post, 0.f, i));
    }
  }
  // sums over the channels: of Q quantities, one value for each of the thread's pixels
  template <int Q> __device__ __forceinline__ void reduce(float (&s)[Q][NP]) {
    static_assert(Q <= MAX_Q, "");
    const int lo = ROWS ? 1 : a.lanes, hi = ROWS ? (a.lanes < 64 ? a.lanes : 64) : 64;
    if (!UNI)
#pragma unroll
      for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int j = 0; j < NP; ++j) s[q][j] = lanes_sum(s[q][j], lo, hi);
    const int waves = ROWS ? a.lanes >> 6 : (int)blockDim.x >> 6;      // that share a pixel
    if (waves <= 1) return;
    // two buffers in turn: the barrier of one round keeps the next but one from overwriting what is still being read
    const int per = (ROWS ? 1 : a.lanes) * Q * NP, all = (int)blockDim.x >> 6;
    float* buf = lds + (round & 1) * (all * (ROWS ? 1 : a.lanes) * MAX_Q * NP) + (ROWS ? 0 : l * Q * NP);
    if (ROWS ? lane == 0 : UNI || lane < a.lanes)
#pragma unroll
      for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int j = 0; j < NP; ++j) buf[wave * per + q * NP + j] = s[q][j];
    __syncthreads();
    const int first = ROWS ? wave & ~(waves - 1) : 0;
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
      for (int j = 0; j < NP; ++j) s[q][j] = 0;
    for (int w = first; w < first + waves; ++w)
#pragma unroll
      for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int j = 0; j < NP; ++j) s[q][j] += buf[w * per + q * NP + j];
    ++round;
  }
  // z -> (z - mean) / sqrt(var + eps) or z / sqrt(mean square + eps); returns the factor.  The variance is summed about the
  // mean, in a second round: E[z^2] - mean^2 would lose it for channels that sit far from zero.
  __device__ __forceinline__ void normalise(float* z, int kind, float eps, float* r) {
    const float inv = 1.f / (float)a.d.C;
    float s[1][NP];
    if (kind == KIND_LAYER) {
#pragma unroll
      for (int j = 0; j < NP; ++j) s[0][j] = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) s[0][pix(e)] += z[e];
      reduce<1>(s);
      if (full)
#pragma unroll
        for (int e = 0; e < E; ++e) z[e] -= s[0][pix(e)] * inv;
      else
#pragma unroll
        for (int e = 0; e < E; ++e) z[e] -= chan_ok(e) ? s[0][pix(e)] * inv : 0.f;
    }
#pragma unroll
    for (int j = 0; j < NP; ++j) s[0][j] = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) s[0][pix(e)] += z[e] * z[e];
    reduce<1>(s);
#pragma unroll
    for (int j = 0; j < NP; ++j) r[j] = 1.f / sqrtf(s[0][j] * inv + eps);
#pragma unroll
    for (int e = 0; e < E; ++e) z[e] *= r[pix(e)];
  }
  // dn (gradient of the normalised values n) -> gradient of what was normalised
  __device__ __forceinline__ void normalise_back(float* dn, const float* n, int kind, const float* r) {
    const float inv = 1.f / (float)a.d.C;
    float s[2][NP];
#pragma unroll
    for (int j = 0; j < NP; ++j) s[0][j] = s[1][j] = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) { s[0][pix(e)] += dn[e] * n[e]; s[1][pix(e)] += dn[e]; }
    reduce<2>(s);
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      s[0][j] *= inv;
      s[1][j] = kind == KIND_LAYER ? s[1][j] * inv : 0.f;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) dn[e] = r[pix(e)] * (dn[e] - n[e] * s[0][pix(e)] - s[1][pix(e)]);
  }
  // sum the thread's per-channel values over the workgroup and write them to out[C]
  __device__ __forceinline__ void flush(float* acc, float* out) {
    if (!ROWS) {
#pragma unroll
      for (int i = 0; i < NW; ++i) acc[i] = lanes_sum(acc[i], 1, a.lanes);
      if (l == 0)
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (chan(k) < a.d.C) out[chan(k)] = acc[k];
      return;
    }
#pragma unroll
    for (int i = 0; i < NW; ++i) acc[i] = lanes_sum(acc[i], a.lanes, 64);
    // waves that hold the same channels: every (lanes / 64)-th
    const int per_row = a.lanes > 64 ? a.lanes >> 6 : 1, waves = (int)blockDim.x >> 6;
    const bool first = wave < per_row && lane < a.lanes;
    if (waves > per_row) {
      __syncthreads();                   // the buffer may still be read as a reduction's
      if (lane < a.lanes)
#pragma unroll
        for (int i = 0; i < NW; ++i) lds[(wave * NW + i) * 64 + lane] = acc[i];
      __syncthreads();
      if (first)
        for (int w = wave + per_row; w < waves; w += per_row)
#pragma unroll
          for (int i = 0; i < NW; ++i) acc[i] += lds[(w * NW + i) * 64 + lane];
      __syncthreads();
    }
    if (first)
#pragma unroll
      for (int i = 0; i < NW; ++i)
        if (chan_ok(i)) out[chan(i / V) + i % V] = acc[i];
  }
};

template <typename T, bool ROWS, int K, int V, bool UNI, bool FULL, int THREADS>
__global__ __launch_bounds__(THREADS) void resnorm_fwd_kernel(const Args a) {
  extern __shared__ float lds[];
  typedef Thread<T, ROWS, K, V, UNI> Th;
  Th t(a, lds);
  const srx_resnorm_desc& d = a.d;
  float gw[Th::NW], gb[Th::NW], w1[Th::NW], b1[Th::NW];
  if (d.pre_kind)
#pragma unroll
    for (int i = 0; i < Th::NW; ++i) { w1[i] = Th::uniform(t.weight(d.w_pre, 1.f, i)); b1[i] = Th::uniform(t.weight(d.b_pre, 0.f, i)); }
  if (d.f && d.gate_mode != GATE_IMAGE) t.branch(0, gw, gb);
  for (int64_t item = blockIdx.x; item < a.items; item += gridDim.x) {
    const int64_t img = item / a.slices, lo = item % a.slices * a.len;
    const int64_t hi = lo + a.len < a.P ? lo + a.len : a.P;
    if (d.f && d.gate_mode == GATE_IMAGE) t.branch(img, gw, gb);
    for (int64_t base = lo; base < hi; base += t.tile()) {
      t.at(img, base, hi);
      typename Th::Raw xr[K], fr[K], qr[K];
      t.read(d.x, d.x_stride, xr);
      if (d.f) t.read(d.f, d.f_stride, fr);
      if (FULL) t.read(d.gate, d.gate_stride, qr);
      float y[Th::E], r[Th::NP];
#pragma unroll
      for (int e = 0; e < Th::E; ++e) y[e] = (float)xr[e / V].e[e % V];
      if (d.f) {
        float n[Th::E];
#pragma unroll
        for (int e = 0; e < Th::E; ++e) n[e] = (float)fr[e / V].e[e % V];
        if (d.post_kind) t.normalise(n, d.post_kind, d.post_eps, r);
        if (FULL) {
#pragma unroll
          for (int e = 0; e < Th::E; ++e) {
            const float q = (float)qr[e / V].e[e % V];
            y[e] += (d.gate_act ? sigmoid(q) : q) * (gw[Th::wi(e)] * n[e] + gb[Th::wi(e)]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < Th::E; ++e) y[e] += gw[Th::wi(e)] * n[e] + gb[Th::wi(e)];
        }
        t.write(d.y, d.y_stride, y);
      }
      if (d.pre_kind) {
        t.normalise(y, d.pre_kind, d.pre_eps, r);
#pragma unroll
        for (int e = 0; e < Th::E; ++e) y[e] = y[e] * w1[Th::wi(e)] + b1[Th::wi(e)];
        t.write(d.h, d.h_stride, y);
      }
    }
  }
}

// With D the gradient of y, the branch's per-channel sums are
//   d w_post = s sum G D n,   d b_post = s sum G D,   d G = s sum D (w n + b),
// and where G is the same for all pixels of an image (or is 1) all three follow from sum D n and sum D: two
// accumulators a channel instead of three.  A full gate takes G D in D's place and writes its own gradient.
template <typename T, bool ROWS, int K, int V, bool UNI, bool FULL, int THREADS>
__global__ __launch_bounds__(THREADS) void resnorm_bwd_kernel(const Args a) {
  extern __shared__ float lds[];
  typedef Thread<T, ROWS, K, V, UNI> Th;
  Th t(a, lds);
  const srx_resnorm_desc& d = a.d;
  float gw[Th::NW], gb[Th::NW], w1[Th::NW];
  float s_dhn[Th::NW] = {}, s_dh[Th::NW] = {}, s_dn[Th::NW] = {}, s_d[Th::NW] = {};
  if (d.dh)
#pragma unroll
    for (int i = 0; i < Th::NW; ++i) w1[i] = Th::uniform(t.weight(d.w_pre, 1.f, i));
  if (d.f && d.gate_mode != GATE_IMAGE) t.branch(0, gw, gb);
  for (int64_t item = blockIdx.x; item < a.items; item += gridDim.x) {
    const int64_t img = item / a.slices, lo = item % a.slices * a.len;
    const int64_t hi = lo + a.len < a.P ? lo + a.len : a.P;
    if (d.f && d.gate_mode == GATE_IMAGE) t.branch(img, gw, gb);
    for (int64_t base = lo; base < hi; base += t.tile()) {
      t.at(img, base, hi);
      typename Th::Raw xr[K], fr[K], qr[K], dyr[K], dhr[K];
      if (d.f) t.read(d.f, d.f_stride, fr);
      if (d.dh) t.read(d.x, d.x_stride, xr);
      if (FULL) t.read(d.gate, d.gate_stride, qr);
      if (d.dh) t.read(d.dh, d.dh_stride, dhr);
      if (d.dy) t.read(d.dy, d.dy_stride, dyr);
      float D[Th::E], n[Th::E], r[Th::NP], r2[Th::NP];
      if (d.f) {
#pragma unroll
        for (int e = 0; e < Th::E; ++e) n[e] = (float)fr[e / V].e[e % V];
        if (d.post_kind) t.normalise(n, d.post_kind, d.post_eps, r2);
      }
#pragma unroll
      for (int e = 0; e < Th::E; ++e) D[e] = d.dy ? (float)dyr[e / V].e[e % V] : 0.f;
      if (d.dh) {
        float y[Th::E], dn[Th::E];
#pragma unroll
        for (int e = 0; e < Th::E; ++e) {
          y[e] = (float)xr[e / V].e[e % V];
          if (d.f) {
            float u = gw[Th::wi(e)] * n[e] + gb[Th::wi(e)];
            if (FULL) {
              const float q = (float)qr[e / V].e[e % V];
              u *= d.gate_act ? sigmoid(q) : q;
            }
            y[e] += u;
          }
        }
        t.normalise(y, d.pre_kind, d.pre_eps, r);
#pragma unroll
        for (int e = 0; e < Th::E; ++e) {
          const float g = (float)dhr[e / V].e[e % V];
          s_dhn[Th::wi(e)] += g * y[e];
          s_dh[Th::wi(e)] += g;
          dn[e] = g * w1[Th::wi(e)];
        }
        t.normalise_back(dn, y, d.pre_kind, r);
#pragma unroll
        for (int e = 0; e < Th::E; ++e) D[e] += dn[e];
      }
      if (d.dx) t.write(d.dx, d.dx_stride, D);
      if (d.f) {
        if (FULL) {
          float dq[Th::E];
#pragma unroll
          for (int e = 0; e < Th::E; ++e) {
            const float q = (float)qr[e / V].e[e % V], G = d.gate_act ? sigmoid(q) : q;
            dq[e] = D[e] * (gw[Th::wi(e)] * n[e] + gb[Th::wi(e)]) * (d.gate_act ? G * (1.f - G) : 1.f);
            D[e] *= G;
          }
          if (d.dgate) t.write(d.dgate, d.dgate_stride, dq);
        }
#pragma unroll
        for (int e = 0; e < Th::E; ++e) {
          // pixels that do not exist have D = 0 but for the offset that a mean takes off: they are left out here
          const float De = ROWS || t.have == V || Th::pix(e) < t.have ? D[e] : 0.f;
          s_dn[Th::wi(e)] += De * n[e];
          s_d[Th::wi(e)] += De;
          D[e] *= gw[Th::wi(e)];
        }
        if (d.post_kind) t.normalise_back(D, n, d.post_kind, r2);
        if (d.df) t.write(d.df, d.df_stride, D);
      }
    }
    if (d.f && d.gate_mode == GATE_IMAGE) {
      float* out = a.part_post + item * 2 * d.C;
      t.flush(s_dn, out);
      t.flush(s_d, out + d.C);
#pragma unroll
      for (int i = 0; i < Th::NW; ++i) s_dn[i] = s_d[i] = 0;
    }
  }
  if (d.dh) {
    float* out = a.part_pre + (int64_t)blockIdx.x * 2 * d.C;
    t.flush(s_dhn, out);
    t.flush(s_dh, out + d.C);
  }
  if (d.f && d.gate_mode != GATE_IMAGE) {
    float* out = a.part_post + (int64_t)blockIdx.x * 2 * d.C;
    t.flush(s_dn, out);
    t.flush(s_d, out + d.C);
  }
}

// Joins the partial sums: 16 channels a workgroup, 64 threads a channel that take every 64th partial.
constexpr int JOIN_X = 16, JOIN_Y = 64;
__device__ __forceinline__ float join(float v, float (*lds)[JOIN_X]) {
  __syncthreads();
  lds[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  float s = 0;
#pragma unroll
  for (int i = 0; i < JOIN_Y; ++i) s += lds[i][threadIdx.x];
  return s;
}
__global__ __launch_bounds__(JOIN_X* JOIN_Y) void resnorm_join_kernel(const Args a, int workgroups, int images) {
  __shared__ float lds[JOIN_Y][JOIN_X];
  const srx_resnorm_desc& d = a.d;
  const int c = blockIdx.x * JOIN_X + threadIdx.x;
  const bool ok = c < d.C;
  if (d.dh && (d.dw_pre || d.db_pre)) {
    float sn = 0, s = 0;
    if (ok)
#pragma unroll 4
      for (int i = threadIdx.y; i < workgroups; i += JOIN_Y) {
        sn += a.part_pre[(int64_t)i * 2 * d.C + c];
        s += a.part_pre[((int64_t)i * 2 + 1) * d.C + c];
      }
    sn = join(sn, lds);
    s = join(s, lds);
    if (ok && threadIdx.y == 0) {
      if (d.dw_pre) d.dw_pre[c] = sn;
      if (d.db_pre) d.db_pre[c] = s;
    }
  }
  if (!d.f) return;
  const float w = ok && d.w_post ? d.w_post[c] : 1.f, b = ok && d.b_post ? d.b_post[c] : 0.f;
  const float* gate = d.gate_mode == GATE_CHANNEL || d.gate_mode == GATE_IMAGE ? static_cast<const float*>(d.gate) : nullptr;
  float* dgate = gate ? static_cast<float*>(d.dgate) : nullptr;
  float dw = 0, db = 0;
  if (d.gate_mode == GATE_IMAGE) {
    if (ok)
      for (int i = threadIdx.y; i < images; i += JOIN_Y) {
        float sn = 0, s = 0;
#pragma unroll 4
        for (int k = 0; k < a.slices; ++k) {
          const float* p = a.part_post + ((int64_t)i * a.slices + k) * 2 * d.C + c;
          sn += p[0];
          s += p[d.C];
        }
        const float q = gate[(int64_t)i * d.C + c], G = d.gate_act ? sigmoid(q) : q;
        if (dgate) dgate[(int64_t)i * d.C + c] = d.scale * (w * sn + b * s) * (d.gate_act ? G * (1.f - G) : 1.f);
        dw += d.scale * G * sn;
        db += d.scale * G * s;
      }
    dw = join(dw, lds);
    db = join(db, lds);
  } else {
    if (ok)
#pragma unroll 4
      for (int i = threadIdx.y; i < workgroups; i += JOIN_Y) {
        dw += a.part_post[(int64_t)i * 2 * d.C + c];
        db += a.part_post[((int64_t)i * 2 + 1) * d.C + c];
      }
    dw = join(dw, lds);
    db = join(db, lds);
    const float q = gate && ok ? gate[c] : 1.f, G = gate && d.gate_act ? sigmoid(q) : q;
    if (dgate && ok && threadIdx.y == 0) dgate[c] = d.scale * (w * dw + b * db) * (d.gate_act ? G * (1.f - G) : 1.f);
    dw *= d.scale * G;
    db *= d.scale * G;
  }
  if (ok && threadIdx.y == 0) {
    if (d.dw_post) d.dw_post[c] = dw;
    if (d.db_post) d.db_post[c] = db;
  }
}

// ------------------------------------------------------------------------------------------------ host side
struct Plan {
  Args a;
  int threads, workgroups, images;
  int elems;               // rows: elements a thread holds
  int lds_bytes;
};

constexpr int PLANES_K = 8, PLANES_V = 2;
constexpr int MAX_THREADS = 512;
constexpr int MAX_ROWS_C = 16 * MAX_THREADS, MAX_PLANES_C = 1024;

int pow2_at_least(int64_t n) {
  int p = 1;
  while (p < n) p <<= 1;
  return p;
}

// The decomposition of a call: workspace size and launch use the same one.
void make_plan(const srx_resnorm_desc& d, int backward, Plan& p) {
  const bool rows = d.layout == SRX_RESNORM_ROWS;
  p.a.d = d;
  const bool image_gate = d.f && d.gate_mode == GATE_IMAGE;
  p.images = rows && !image_gate ? 1 : d.B;
  p.a.P = rows && !image_gate ? (int64_t)d.B * d.P : d.P;
  int tile;
  if (rows) {
    p.elems = d.C <= 512 ? 8 : 16;
    p.a.lanes = pow2_at_least((d.C + p.elems - 1) / p.elems);
    p.threads = p.a.lanes > 256 ? p.a.lanes : 256;
    tile = p.threads / p.a.lanes;
  } else {
    const int groups = (d.C + PLANES_K - 1) / PLANES_K;
    p.a.lanes = 64;
    while (groups * p.a.lanes > MAX_THREADS) p.a.lanes /= 2;
    p.threads = 64 * ((groups * p.a.lanes + 63) / 64);
    tile = p.a.lanes * PLANES_V;
  }
  const int64_t tiles = (p.a.P + tile - 1) / tile;
  const int64_t target = backward ? 512 : 4096;
  int64_t s = p.images > 0 ? (target + p.images - 1) / p.images : 1;
  s = s < 1 ? 1 : s > tiles ? tiles : s;
  if (s < 1) s = 1;
  p.a.len = (tiles + s - 1) / s * tile;
  p.a.slices = p.a.len > 0 ? (int)((p.a.P + p.a.len - 1) / p.a.len) : 1;
  if (p.a.slices < 1) p.a.slices = 1;
  p.a.items = p.a.P > 0 ? (int64_t)p.images * p.a.slices : 0;
  p.workgroups = (int)(p.a.items < target ? p.a.items : target);
  const int waves = p.threads / 64;
  int bytes = 2 * waves * MAX_Q * (rows ? 1 : p.a.lanes * PLANES_V) * 4;            // two buffers; at most 32 KB
  if (backward && rows && p.threads == 256 && bytes < waves * p.elems * 64 * 4) bytes = waves * p.elems * 64 * 4;     // flush: 16 KB
  p.lds_bytes = bytes;
}

int check(const char* what, const srx_resnorm_desc* d) {
  SRX_CHECK_ARG(d != nullptr, "%s: null descriptor", what);
  SRX_CHECK_ARG(d->dtype == SRX_BF16 || d->dtype == SRX_F32, "%s: bad dtype %d", what, d->dtype);
  SRX_CHECK_ARG(d->layout == SRX_RESNORM_PLANES || d->layout == SRX_RESNORM_ROWS, "%s: bad layout %d", what, d->layout);
  SRX_CHECK_ARG(d->B >= 0 && d->P >= 0 && d->C > 0, "%s: bad sizes B %d C %d P %d", what, d->B, d->C, d->P);
  const int most = d->layout == SRX_RESNORM_ROWS ? MAX_ROWS_C : MAX_PLANES_C;
  SRX_CHECK_ARG(d->C <= most, "%s: %d channels, at most %d in this layout", what, d->C, most);
  SRX_CHECK_ARG(d->post_kind >= 0 && d->post_kind <= 2 && d->pre_kind >= 0 && d->pre_kind <= 2, "%s: bad norm kind", what);
  SRX_CHECK_ARG(d->gate_mode >= 0 && d->gate_mode <= 3 && (d->gate_act == 0 || d->gate_act == 1), "%s: bad gate mode", what);
  SRX_CHECK_ARG((!d->post_kind || d->post_eps > 0) && (!d->pre_kind || d->pre_eps > 0), "%s: eps must be positive", what);
  SRX_CHECK_ARG(d->f || (!d->post_kind && !d->gate_mode), "%s: a norm after the branch or a gate without a branch", what);
  SRX_CHECK_ARG(d->f || d->pre_kind, "%s: neither a branch nor a norm", what);
  SRX_CHECK_ARG(!d->gate_mode || d->gate, "%s: null gate", what);
  const bool rows = d->layout == SRX_RESNORM_ROWS;
  const void* ptrs[] = {d->x, d->f, d->y, d->h, d->dy, d->dh, d->dx, d->df, d->gate_mode == GATE_FULL ? d->gate : nullptr,
                        d->gate_mode == GATE_FULL ? d->dgate : nullptr};
  const int64_t strides[] = {d->x_stride, d->f_stride, d->y_stride, d->h_stride, d->dy_stride, d->dh_stride, d->dx_stride,
                             d->df_stride, d->gate_stride, d->dgate_stride};
  const int esize = d->dtype == SRX_BF16 ? 2 : 4;
  const int64_t least = rows ? d->C : (int64_t)d->C * d->P;
  for (int i = 0; i < 10; ++i)
    if (ptrs[i]) {
      SRX_CHECK_ARG((uintptr_t)ptrs[i] % esize == 0, "%s: tensor %d is not aligned to its type", what, i);
      SRX_CHECK_ARG(strides[i] >= 0 && (strides[i] >= least || (i < 2 || i == 4 || i == 5 || i == 8)),
                    "%s: tensor %d: stride %lld of an output is under %lld", what, i, (long long)strides[i], (long long)least);
    }
  return SRX_OK;
}

template <typename T, bool ROWS, int K, int V, bool UNI, bool FULL> int launch_with(const Plan& p, int backward, hipStream_t s) {
  if (backward)
    hipLaunchKernelGGL((resnorm_bwd_kernel<T, ROWS, K, V, UNI, FULL, MAX_THREADS>), dim3(p.workgroups), dim3(p.threads), p.lds_bytes, s, p.a);
  else
    hipLaunchKernelGGL((resnorm_fwd_kernel<T, ROWS, K, V, UNI, FULL, MAX_THREADS>), dim3(p.workgroups), dim3(p.threads), p.lds_bytes, s, p.a);
  return srx_check_launch(backward ? "resnorm_bwd" : "resnorm_fwd");
}
template <typename T, bool ROWS, int K, int V, bool UNI> int launch(const Plan& p, int backward, hipStream_t s) {
  return p.a.d.gate_mode == GATE_FULL ? launch_with<T, ROWS, K, V, UNI, true>(p, backward, s) : launch_with<T, ROWS, K, V, UNI, false>(p, backward, s);
}

template <typename T> int dispatch(const Plan& p, int backward, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  if (p.a.d.layout == SRX_RESNORM_ROWS)
    return p.elems == 8 ? launch<T, true, 8 / V, V, false>(p, backward, s) : launch<T, true, 16 / V, V, false>(p, backward, s);
  return p.a.lanes == 64 ? launch<T, false, PLANES_K, PLANES_V, true>(p, backward, s)
                         : launch<T, false, PLANES_K, PLANES_V, false>(p, backward, s);
}

}  // namespace

extern "C" {

int64_t srx_resnorm_ws_floats(const srx_resnorm_desc* d) {
  if (check("srx_resnorm_ws_floats", d)) return -1;
  Plan p = {};
  make_plan(*d, 1, p);
  return 2 * (int64_t)d->C * (p.workgroups + (d->f && d->gate_mode == GATE_IMAGE ? p.a.items : p.workgroups)) + 1;
}

int srx_resnorm_forward(const srx_resnorm_desc* d, void* stream) {
  if (int rc = check("srx_resnorm_forward", d)) return rc;
  if ((int64_t)d->B * d->P == 0) return SRX_OK;
  SRX_CHECK_ARG(d->x && (!d->f || d->y) && (!d->pre_kind || d->h), "srx_resnorm_forward: null tensor");
  Plan p = {};
  make_plan(*d, 0, p);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return d->dtype == SRX_BF16 ? dispatch<bf16>(p, 0, s) : dispatch<float>(p, 0, s);
}

int srx_resnorm_backward(const srx_resnorm_desc* d, void* stream) {
  if (int rc = check("srx_resnorm_backward", d)) return rc;
  const bool empty = (int64_t)d->B * d->P == 0;
  SRX_CHECK_ARG(empty || d->dy || d->dh, "srx_resnorm_backward: neither dy nor dh");
  SRX_CHECK_ARG(!d->dh || (d->pre_kind && (d->x || empty)), "srx_resnorm_backward: dh needs the norm before the next branch, and x");
  SRX_CHECK_ARG(empty || d->ws, "srx_resnorm_backward: null workspace");
  Plan p = {};
  make_plan(*d, 1, p);
  if (empty) p.a.slices = 0;            // the gradients of weights and gates are zeros
  p.a.part_pre = d->ws;
  p.a.part_post = d->ws + 2 * (int64_t)d->C * p.workgroups;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (!empty)
    if (int rc = d->dtype == SRX_BF16 ? dispatch<bf16>(p, 1, s) : dispatch<float>(p, 1, s)) return rc;
  const bool sums = d->dw_pre || d->db_pre || (d->f && (d->dw_post || d->db_post || (d->dgate && d->gate_mode && d->gate_mode != GATE_FULL)));
  if (!sums) return SRX_OK;
  hipLaunchKernelGGL(resnorm_join_kernel, dim3((d->C + JOIN_X - 1) / JOIN_X), dim3(JOIN_X, JOIN_Y), 0, s, p.a, p.workgroups, p.images);
  return srx_check_launch("resnorm_join");
}

}  // extern "C"
