// Norms over the channels before and after a residual branch, fused with the branch's gate, the residual scale and the
// residual add (include/srx.h, srx_resnorm_forward / _backward, has the formulas).
//
// One kernel body serves both layouts.  A thread holds K x V elements of each tensor in registers:
//   rows   (channels contiguous): V neighbouring channels, K times, of ONE row; `lanes` threads share a row.
//   planes (pixels contiguous):   V neighbouring pixels of K channels; `lanes` threads of a wave sit side by side
//                                 along the pixels, the others hold other channels of the same pixels.
// Every tensor is read once: statistics, norm and gradients come out of the registers, in fp32.  The sums over the pixels
// (gradients of weights, biases and gates) stay in registers while a workgroup walks its share of the pixels; their
// partial sums are joined by a second small kernel in a fixed order (no atomics: same inputs, same bits).
#include "srx_common.h"

namespace {

constexpr int MAX_THREADS = 1024;
constexpr int MAX_Q = 2;          // quantities reduced together
enum { KIND_NONE = 0, KIND_RMS = 1, KIND_LAYER = 2 };
enum { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_IMAGE = 2, GATE_FULL = 3 };

struct Args {
  srx_resnorm_desc d;
  int lanes;            // rows: threads per row (a power of two); planes: lanes along the pixels (64, 32 or 16)
  int slices;           // shares of an image's pixels
  int64_t len;          // pixels of a share
  int64_t items;        // images * slices
  int64_t P;            // pixels of an "image" (rows without per-image gate: all rows are one image)
  float* part_pre;      // [workgroups][2][C]
  float* part_post;     // [workgroups or items][2][C]
};

template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T e[V]; };
template <typename T, int V> __device__ __forceinline__ void load(const T* p, float* out) {
  const Vec<T, V> t = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
  for (int j = 0; j < V; ++j) out[j] = (float)t.e[j];
}
template <typename T, int V> __device__ __forceinline__ void store(T* p, const float* v) {
  Vec<T, V> t;
#pragma unroll
  for (int j = 0; j < V; ++j) t.e[j] = (T)v[j];
  *reinterpret_cast<Vec<T, V>*>(p) = t;
}
__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + __expf(-x)); }

template <typename T, bool ROWS, int K, int V> struct Thread {
  static constexpr int E = K * V;                     // elements of each tensor
  static constexpr int NP = ROWS ? 1 : V;             // pixels
  static constexpr int NW = ROWS ? E : K;             // channels
  static __device__ __forceinline__ constexpr int pix(int e) { return ROWS ? 0 : e % V; }
  static __device__ __forceinline__ constexpr int wi(int e) { return ROWS ? e : e / V; }

  const Args& a;
  float* lds;
  int round;
  int lane, wave, l, grp;     // rows: l = thread within the row, grp = row of the workgroup; planes: l = lane along the pixels
  bool chan_ok[K];            // this k's channels exist
  bool ok;                    // the row / the pixels exist
  int64_t pixel;              // first pixel within the image
  int64_t image;

  __device__ __forceinline__ Thread(const Args& a_, float* lds_) : a(a_), lds(lds_), round(0) {
    lane = threadIdx.x & 63;
    wave = threadIdx.x >> 6;
    if (ROWS) { l = threadIdx.x & (a.lanes - 1); grp = threadIdx.x / a.lanes; }
    else { l = lane & (a.lanes - 1); grp = threadIdx.x / a.lanes; }
#pragma unroll
    for (int k = 0; k < K; ++k) chan_ok[k] = chan(k) < a.d.C;
  }
  __device__ __forceinline__ int chan(int k) const { return ROWS ? (k * a.lanes + l) * V : grp * K + k; }
  // pixels that a workgroup takes at a time
  __device__ __forceinline__ int tile() const { return ROWS ? (int)blockDim.x / a.lanes : a.lanes * V; }
  __device__ __forceinline__ void at(int64_t img, int64_t base, int64_t end) {
    image = img;
    pixel = base + (ROWS ? grp : l * V);
    ok = pixel < end;
  }
  // image / row stride -> offset of element 0 of step k
  __device__ __forceinline__ int64_t offset(int64_t stride, int k) const {
    return ROWS ? (image * a.P + pixel) * stride + chan(k) : image * stride + (int64_t)chan(k) * a.P + pixel;
  }
  __device__ __forceinline__ void read(const void* p, int64_t stride, float* z) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (ok && chan_ok[k]) load<T, V>(static_cast<const T*>(p) + offset(stride, k), z + k * V);
      else
#pragma unroll
        for (int j = 0; j < V; ++j) z[k * V + j] = 0.f;
    }
  }
  __device__ __forceinline__ void write(void* p, int64_t stride, const float* z) const {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (ok && chan_ok[k]) store<T, V>(static_cast<T*>(p) + offset(stride, k), z + k * V);
  }
  // per-channel fp32 values (NULL: `missing`); channels that do not exist get 0
  __device__ __forceinline__ void weights(const float* w, float missing, float* out) const {
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const int k = ROWS ? i / V : i, c = chan(k) + (ROWS ? i % V : 0);
      out[i] = !chan_ok[k] ? 0.f : w ? w[c] : missing;
    }
  }
  // sums over the channels: of Q quantities, one value for each of the thread's pixels
  template <int Q> __device__ __forceinline__ void reduce(float (&s)[Q][NP]) {
    static_assert(Q <= MAX_Q, "");
    const int lo = ROWS ? 1 : a.lanes, hi = ROWS ? (a.lanes < 64 ? a.lanes : 64) : 64;
    for (int o = lo; o < hi; o <<= 1)
#pragma unroll
      for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int j = 0; j < NP; ++j) s[q][j] += __shfl_xor(s[q][j], o, 64);
    const int waves = ROWS ? a.lanes >> 6 : (int)blockDim.x >> 6;      // that share a pixel
    if (waves <= 1) return;
    // two buffers in turn: the barrier of one round keeps the next but one from overwriting what is still being read
    const int per = ROWS ? 1 : a.lanes * NP, all = (int)blockDim.x >> 6;
    float* buf = lds + (round & 1) * (all * MAX_Q * per);
    const int slot = ROWS ? 0 : l * NP;
    if (ROWS ? lane == 0 : lane < a.lanes)
#pragma unroll
      for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int j = 0; j < NP; ++j) buf[(wave * Q + q) * per + slot + j] = s[q][j];
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
        for (int j = 0; j < NP; ++j) s[q][j] += buf[(w * Q + q) * per + slot + j];
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
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (chan_ok[e / V]) z[e] -= s[0][pix(e)] * inv;
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
    for (int e = 0; e < E; ++e) {
      const int j = pix(e);
      dn[e] = r[j] * (dn[e] - n[e] * (s[0][j] * inv) - (kind == KIND_LAYER ? s[1][j] * inv : 0.f));
    }
  }
  // sum the thread's per-channel values over the workgroup and write them to out[C]
  __device__ __forceinline__ void flush(float* acc, float* out) {
    if (!ROWS) {
      for (int o = 1; o < a.lanes; o <<= 1)
#pragma unroll
        for (int i = 0; i < NW; ++i) acc[i] += __shfl_xor(acc[i], o, 64);
      if (l == 0)
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (chan_ok[k]) out[chan(k)] = acc[k];
      return;
    }
    for (int o = a.lanes; o < 64; o <<= 1)
#pragma unroll
      for (int i = 0; i < NW; ++i) acc[i] += __shfl_xor(acc[i], o, 64);
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
      for (int k = 0; k < K; ++k)
        if (chan_ok[k])
#pragma unroll
          for (int j = 0; j < V; ++j) out[chan(k) + j] = acc[k * V + j];
  }
};

template <typename T, bool ROWS, int K, int V, int THREADS>
__global__ __launch_bounds__(THREADS) void resnorm_fwd_kernel(const Args a) {
  extern __shared__ float lds[];
  typedef Thread<T, ROWS, K, V> Th;
  Th t(a, lds);
  const srx_resnorm_desc& d = a.d;
  float w2[Th::NW], b2[Th::NW], g[Th::NW], w1[Th::NW], b1[Th::NW];
  if (d.f) { t.weights(d.w_post, 1.f, w2); t.weights(d.b_post, 0.f, b2); }
  if (d.pre_kind) { t.weights(d.w_pre, 1.f, w1); t.weights(d.b_pre, 0.f, b1); }
  for (int64_t item = blockIdx.x; item < a.items; item += gridDim.x) {
    const int64_t img = item / a.slices, lo = item % a.slices * a.len;
    const int64_t hi = lo + a.len < a.P ? lo + a.len : a.P;
    if (d.f && d.gate_mode != GATE_FULL) {
      t.weights(d.gate_mode == GATE_NONE ? nullptr : static_cast<const float*>(d.gate) + (d.gate_mode == GATE_IMAGE ? img * d.C : 0), 1.f, g);
#pragma unroll
      for (int i = 0; i < Th::NW; ++i) g[i] = d.scale * (d.gate_mode && d.gate_act ? sigmoid(g[i]) : g[i]);
    }
    for (int64_t base = lo; base < hi; base += t.tile()) {
      t.at(img, base, hi);
      float y[Th::E], r[Th::NP];
      t.read(d.x, d.x_stride, y);
      if (d.f) {
        float n[Th::E];
        t.read(d.f, d.f_stride, n);
        if (d.post_kind) t.normalise(n, d.post_kind, d.post_eps, r);
        if (d.gate_mode == GATE_FULL) {
          float q[Th::E];
          t.read(d.gate, d.gate_stride, q);
#pragma unroll
          for (int e = 0; e < Th::E; ++e)
            y[e] += d.scale * (d.gate_act ? sigmoid(q[e]) : q[e]) * (n[e] * w2[Th::wi(e)] + b2[Th::wi(e)]);
        } else {
#pragma unroll
          for (int e = 0; e < Th::E; ++e) y[e] += g[Th::wi(e)] * (n[e] * w2[Th::wi(e)] + b2[Th::wi(e)]);
        }
        if (d.y) t.write(d.y, d.y_stride, y);
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
// accumulators a channel instead of three.  A full gate takes s G D in D's place and writes its own gradient.
template <typename T, bool ROWS, int K, int V, int THREADS>
__global__ __launch_bounds__(THREADS) void resnorm_bwd_kernel(const Args a) {
  extern __shared__ float lds[];
  typedef Thread<T, ROWS, K, V> Th;
  Th t(a, lds);
  const srx_resnorm_desc& d = a.d;
  float w2[Th::NW], b2[Th::NW], g[Th::NW], w1[Th::NW];
  float s_dhn[Th::NW] = {}, s_dh[Th::NW] = {}, s_dn[Th::NW] = {}, s_d[Th::NW] = {};
  if (d.f) { t.weights(d.w_post, 1.f, w2); t.weights(d.b_post, 0.f, b2); }
  if (d.dh) t.weights(d.w_pre, 1.f, w1);
  for (int64_t item = blockIdx.x; item < a.items; item += gridDim.x) {
    const int64_t img = item / a.slices, lo = item % a.slices * a.len;
    const int64_t hi = lo + a.len < a.P ? lo + a.len : a.P;
    if (d.f && d.gate_mode != GATE_FULL) {
      t.weights(d.gate_mode == GATE_NONE ? nullptr : static_cast<const float*>(d.gate) + (d.gate_mode == GATE_IMAGE ? img * d.C : 0), 1.f, g);
#pragma unroll
      for (int i = 0; i < Th::NW; ++i) g[i] = d.scale * (d.gate_mode && d.gate_act ? sigmoid(g[i]) : g[i]);
    }
    for (int64_t base = lo; base < hi; base += t.tile()) {
      t.at(img, base, hi);
      float D[Th::E], r[Th::NP];
      if (d.dy) t.read(d.dy, d.dy_stride, D);
      else
#pragma unroll
        for (int e = 0; e < Th::E; ++e) D[e] = 0;
      if (d.dh) {
        float n[Th::E], dn[Th::E];
        t.read(d.y, d.y_stride, n);
        t.read(d.dh, d.dh_stride, dn);
        t.normalise(n, d.pre_kind, d.pre_eps, r);
#pragma unroll
        for (int e = 0; e < Th::E; ++e) {
          s_dhn[Th::wi(e)] += dn[e] * n[e];
          s_dh[Th::wi(e)] += dn[e];
          dn[e] *= w1[Th::wi(e)];
        }
        t.normalise_back(dn, n, d.pre_kind, r);
#pragma unroll
        for (int e = 0; e < Th::E; ++e) D[e] += dn[e];
      }
      if (d.dx) t.write(d.dx, d.dx_stride, D);
      if (d.f) {
        float n[Th::E];
        t.read(d.f, d.f_stride, n);
        if (d.post_kind) t.normalise(n, d.post_kind, d.post_eps, r);
        if (d.gate_mode == GATE_FULL) {
          float q[Th::E];
          t.read(d.gate, d.gate_stride, q);
#pragma unroll
          for (int e = 0; e < Th::E; ++e) {
            const float G = d.gate_act ? sigmoid(q[e]) : q[e];
            q[e] = d.scale * D[e] * (n[e] * w2[Th::wi(e)] + b2[Th::wi(e)]) * (d.gate_act ? G * (1.f - G) : 1.f);
            D[e] *= d.scale * G;
          }
          if (d.dgate) t.write(d.dgate, d.dgate_stride, q);
        }
#pragma unroll
        for (int e = 0; e < Th::E; ++e) {
          s_dn[Th::wi(e)] += D[e] * n[e];
          s_d[Th::wi(e)] += D[e];
          D[e] *= d.gate_mode == GATE_FULL ? w2[Th::wi(e)] : g[Th::wi(e)] * w2[Th::wi(e)];
        }
        if (d.post_kind) t.normalise_back(D, n, d.post_kind, r);
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

// Joins the partial sums: 64 channels a workgroup, 16 threads a channel that take every 16th partial.
constexpr int JOIN_X = 64, JOIN_Y = 16;
__device__ __forceinline__ float join(float v, float (*lds)[JOIN_X]) {
  __syncthreads();
  lds[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  float s = 0;
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
      for (int i = threadIdx.y; i < workgroups; i += JOIN_Y) {
        dw += a.part_post[(int64_t)i * 2 * d.C + c];
        db += a.part_post[((int64_t)i * 2 + 1) * d.C + c];
      }
    dw = join(dw, lds);
    db = join(db, lds);
    if (d.gate_mode != GATE_FULL) {
      const float q = gate && ok ? gate[c] : 1.f, G = gate && d.gate_act ? sigmoid(q) : q;
      if (dgate && ok && threadIdx.y == 0) dgate[c] = d.scale * (w * dw + b * db) * (d.gate_act ? G * (1.f - G) : 1.f);
      dw *= d.scale * G;
      db *= d.scale * G;
    }
  }
  if (ok && threadIdx.y == 0) {
    if (d.dw_post) d.dw_post[c] = dw;
    if (d.db_post) d.db_post[c] = db;
  }
}

// ------------------------------------------------------------------------------------------------ host side
struct Plan {
  Args a;
  int threads, workgroups, v, images;
  int lds_bytes;
};

constexpr int KV = 16;            // elements of a tensor that a thread holds
constexpr int MAX_ROWS_C = KV * MAX_THREADS, MAX_PLANES_C = KV * MAX_THREADS / 16;

int pow2_at_least(int64_t n) {
  int p = 1;
  while (p < n) p <<= 1;
  return p;
}

// The decomposition of a call: workspace size and launch use the same one.
void make_plan(const srx_resnorm_desc& d, int backward, bool vector, Plan& p) {
  const bool rows = d.layout == SRX_RESNORM_ROWS;
  p.a.d = d;
  int tile;
  if (rows) {
    p.v = vector ? (d.dtype == SRX_BF16 ? 8 : 4) : 1;
    p.a.lanes = pow2_at_least((d.C + KV - 1) / KV);
    p.threads = p.a.lanes > 256 ? p.a.lanes : 256;
    tile = p.threads / p.a.lanes;
  } else {
    p.v = vector ? 2 : 1;
    const int k = KV / p.v;
    const int groups = (d.C + k - 1) / k;
    p.a.lanes = groups <= 16 ? 64 : groups <= 32 ? 32 : 16;
    p.threads = 64 * ((groups * p.a.lanes + 63) / 64);
    tile = p.a.lanes * p.v;
  }
  const bool image_gate = d.f && d.gate_mode == GATE_IMAGE;
  p.images = rows && !image_gate ? 1 : d.B;
  p.a.P = rows && !image_gate ? (int64_t)d.B * d.P : d.P;
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
  const int np = rows ? 1 : p.v;
  int bytes = 2 * waves * MAX_Q * (rows ? 1 : p.a.lanes * np) * 4;            // two buffers; at most 32 KB
  if (backward && rows && p.threads == 256 && bytes < waves * KV * 64 * 4) bytes = waves * KV * 64 * 4;     // flush: 16 KB
  p.lds_bytes = bytes;
}

// Vector accesses need every tensor's elements to line up: channels (rows) or pixels (planes) a multiple of the vector, and
// strides and addresses too.
bool can_vector(const srx_resnorm_desc& d) {
  const bool rows = d.layout == SRX_RESNORM_ROWS;
  const int v = rows ? (d.dtype == SRX_BF16 ? 8 : 4) : 2;
  const int esize = d.dtype == SRX_BF16 ? 2 : 4;
  if ((rows ? d.C : d.P) % v || (!rows && d.C > MAX_PLANES_C / v)) return false;
  const void* ptrs[] = {d.x, d.f, d.y, d.h, d.dy, d.dh, d.dx, d.df, d.gate_mode == GATE_FULL ? d.gate : nullptr,
                        d.gate_mode == GATE_FULL ? d.dgate : nullptr};
  const int64_t strides[] = {d.x_stride, d.f_stride, d.y_stride, d.h_stride, d.dy_stride, d.dh_stride, d.dx_stride, d.df_stride,
                             d.gate_stride, d.dgate_stride};
  for (int i = 0; i < 10; ++i)
    if (ptrs[i] && ((uintptr_t)ptrs[i] % (v * esize) || strides[i] % v)) return false;
  return true;
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

template <typename T, bool ROWS, int K, int V, int THREADS> int launch_with(const Plan& p, int backward, hipStream_t s) {
  if (backward)
    hipLaunchKernelGGL((resnorm_bwd_kernel<T, ROWS, K, V, THREADS>), dim3(p.workgroups), dim3(p.threads), p.lds_bytes, s, p.a);
  else
    hipLaunchKernelGGL((resnorm_fwd_kernel<T, ROWS, K, V, THREADS>), dim3(p.workgroups), dim3(p.threads), p.lds_bytes, s, p.a);
  return srx_check_launch(backward ? "resnorm_bwd" : "resnorm_fwd");
}

template <typename T, bool ROWS, int K, int V> int launch(const Plan& p, int backward, hipStream_t s) {
  return p.threads <= 256 ? launch_with<T, ROWS, K, V, 256>(p, backward, s)
         : p.threads <= 512 ? launch_with<T, ROWS, K, V, 512>(p, backward, s) : launch_with<T, ROWS, K, V, 1024>(p, backward, s);
}

template <typename T> int dispatch(const Plan& p, int backward, hipStream_t s) {
  constexpr int VR = sizeof(T) == 2 ? 8 : 4;
  if (p.a.d.layout == SRX_RESNORM_ROWS)
    return p.v == 1 ? launch<T, true, KV, 1>(p, backward, s) : launch<T, true, KV / VR, VR>(p, backward, s);
  return p.v == 1 ? launch<T, false, KV, 1>(p, backward, s) : launch<T, false, KV / 2, 2>(p, backward, s);
}

}  // namespace

extern "C" {

int64_t srx_resnorm_ws_floats(const srx_resnorm_desc* d) {
  if (check("srx_resnorm_ws_floats", d)) return -1;
  Plan p = {}, q = {};
  make_plan(*d, 1, true, p);
  make_plan(*d, 1, false, q);
  const int64_t items = p.a.items > q.a.items ? p.a.items : q.a.items, wgs = p.workgroups > q.workgroups ? p.workgroups : q.workgroups;
  return 2 * (int64_t)d->C * (wgs + (d->f && d->gate_mode == GATE_IMAGE ? items : wgs)) + 1;
}

int srx_resnorm_forward(const srx_resnorm_desc* d, void* stream) {
  if (int rc = check("srx_resnorm_forward", d)) return rc;
  if ((int64_t)d->B * d->P == 0) return SRX_OK;
  SRX_CHECK_ARG(d->x && (!d->f || d->y) && (!d->pre_kind || d->h), "srx_resnorm_forward: null tensor");
  Plan p = {};
  make_plan(*d, 0, can_vector(*d), p);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return d->dtype == SRX_BF16 ? dispatch<bf16>(p, 0, s) : dispatch<float>(p, 0, s);
}

int srx_resnorm_backward(const srx_resnorm_desc* d, void* stream) {
  if (int rc = check("srx_resnorm_backward", d)) return rc;
  const bool empty = (int64_t)d->B * d->P == 0;
  SRX_CHECK_ARG(empty || d->dy || d->dh, "srx_resnorm_backward: neither dy nor dh");
  SRX_CHECK_ARG(!d->dh || (d->pre_kind && (d->y || empty)), "srx_resnorm_backward: dh needs the norm before the next branch, and y");
  SRX_CHECK_ARG(empty || d->ws, "srx_resnorm_backward: null workspace");
  Plan p = {};
  make_plan(*d, 1, can_vector(*d), p);
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
