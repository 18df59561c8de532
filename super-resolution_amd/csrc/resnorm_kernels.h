// Norms over the channels before and after a residual branch, fused with the branch's gate, the residual scale and the
// residual add (include/srx.h, srx_resnorm_forward / _backward, has the formulas): the kernels, included by one translation
// unit per element type.
//
// One kernel body serves both layouts.  A thread holds K x V elements of each tensor in registers:
//   rows   (channels contiguous): V neighbouring channels, K times, of ONE row; `lanes` threads share a row.
//   planes (pixels contiguous):   V neighbouring pixels (1, 2 or 4) of K channels; `lanes` threads of a wave sit side by side
//                                 along the pixels, the others hold other channels of the same pixels.
// Every tensor is read once: statistics, norm and gradients come out of the registers, in fp32.  The backward pass takes
// x and f and forms y again: the same traffic as reading y, and not y's rounding to bf16 (which would put 2^-9 of
// error into every weight gradient).  The sums over the pixels (gradients of weights, biases and gates) stay in registers
// while a workgroup walks its share of the pixels; their partial sums are joined by a second small kernel in a fixed
// order (no atomics: same inputs, same bits).
#pragma once
#include <type_traits>
#include "srx_common.h"

namespace resnorm {

constexpr int MAX_Q = 2;          // quantities reduced together
constexpr int THREADS = 512;      // most threads of a workgroup
constexpr int WAVES = THREADS / 64;
enum { KIND_NONE = 0, KIND_RMS = 1, KIND_LAYER = 2 };
enum { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_IMAGE = 2, GATE_FULL = 3 };

struct Args {
  srx_resnorm_desc d;
  int lanes;            // rows: threads per row (a power of two); planes: lanes along the pixels (64 down to 4)
  int slices;           // shares of an image's tiles: share s takes tiles s, s + slices, ...
  int items;            // images * slices; workgroup w takes items w, w + workgroups, ...
  int64_t P;            // pixels of an "image" (rows without per-image gate: all rows are one image)
  float* part_pre;      // [workgroups][2][C]
  float* part_post;     // [workgroups or items][2][C]
  int jump_images, jump_shares;       // from a workgroup's item to its next: workgroups / slices, workgroups % slices
  __device__ __forceinline__ void next(int& image, int& share) const {
    image += jump_images;
    share += jump_shares;
    if (share >= slices) {
      share -= slices;
      ++image;
    }
  }
};
struct Plan {
  Args a;
  int threads, workgroups, images;
  int elems;               // rows: elements a thread holds; planes: pixels
  int lds_bytes;
};
constexpr int PLANES_K = 8;
int launch_bf16(const Plan& p, int backward, hipStream_t s);
int launch_f32(const Plan& p, int backward, hipStream_t s);

// V elements, at any address that is a multiple of the element's size: global memory takes wide accesses there (a row
// of an odd number of channels, a map of an odd number of pixels), so there is no second, narrow form of the kernels.
// Kept as 32-bit words: the compiler would give every bf16 element a register of its own.
template <typename T, int V> struct __attribute__((packed, aligned(sizeof(T)))) Vec { uint32_t w[V * sizeof(T) / 4]; };
template <> struct Vec<bf16, 1> { uint16_t w; };
template <int V> __device__ __forceinline__ float element(const Vec<float, V>& z, int j) { return __uint_as_float(z.w[j]); }
template <int V> __device__ __forceinline__ float element(const Vec<bf16, V>& z, int j) {
  if constexpr (V == 1) return __uint_as_float((uint32_t)z.w << 16);
  else return __uint_as_float(j & 1 ? z.w[j / 2] & 0xFFFF0000u : z.w[j / 2] << 16);
}
// zeros in place of the first n elements
template <int V> __device__ __forceinline__ void drop(Vec<float, V>& z, int n) {
#pragma unroll
  for (int j = 0; j < V; ++j) z.w[j] = j < n ? 0u : z.w[j];
}
template <int V> __device__ __forceinline__ void drop(Vec<bf16, V>& z, int n) {
  if constexpr (V == 1) z.w = n > 0 ? 0 : z.w;
  else
#pragma unroll
    for (int j = 0; j < V; j += 2) z.w[j / 2] = j + 1 < n ? 0u : j < n ? z.w[j / 2] & 0xFFFF0000u : z.w[j / 2];
}
template <int V> __device__ __forceinline__ Vec<float, V> packed(const float* v, const float*) {
  Vec<float, V> z;
#pragma unroll
  for (int j = 0; j < V; ++j) z.w[j] = __float_as_uint(v[j]);
  return z;
}
template <int V> __device__ __forceinline__ Vec<bf16, V> packed(const float* v, const bf16*) {
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
  Vec<bf16, V> z;
  if constexpr (V == 1) z.w = __builtin_bit_cast(uint16_t, (bf16)v[0]);
  else
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const bf16x2 p = {(bf16)v[j], (bf16)v[j + 1]};
      z.w[j / 2] = __builtin_bit_cast(uint32_t, p);
    }
  return z;
}
// within 2^-22 of the value; eps is a normal number, so the argument is one too
__device__ __forceinline__ float rsqrt_hw(float x) { return __builtin_amdgcn_rsqf(x); }
// within (1.5 |x| + 6) 2^-24 of the value: the hardware's exponential is of base 2, and its argument's two roundings count |x|-fold
__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + __expf(-x)); }

// A barrier for what waves hand each other through LDS, and only that: __syncthreads() would also wait for every global load
// and store in flight, the last tile's results and the next one's inputs among them.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
// sums over the lanes whose numbers differ in the bits lo, 2 lo, ... hi / 2 (every lane gets them)
template <int N> __device__ __forceinline__ void lanes_sum(float* v, int lo, int hi) {
  if (lo <= 1 && hi > 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = dpp_add<0xB1>(v[i]);          // quad_perm 1,0,3,2
  if (lo <= 2 && hi > 2)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = dpp_add<0x4E>(v[i]);          // quad_perm 2,3,0,1
  if (lo <= 4 && hi > 4) {
    if (lo <= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = dpp_add<0x141>(v[i]);       // row_half_mirror: lane ^ 7, and quads are uniform by now
    else
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], 4, 64);
  }
  if (lo <= 8 && hi > 8)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = dpp_add<0x128>(v[i]);         // row_ror 8
  if (lo <= 16 && hi > 16)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i]), false, false);
      v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
  if (lo <= 32 && hi > 32)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i]), false, false);
      v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
}

// Every load is a whole vector that lies inside the tensor, without a branch: one that would pass the end (of a row; of
// a plane; a row or channel that does not exist) starts earlier, and the elements in front of the thread's own, `dup` of
// them, are zeros from then on.  GEN: some norm has a bias (else: no offsets, and no sums for them).
// UNI (planes with 64 lanes along the pixels): a wave's lanes hold the same channels, so that channels, their addresses
// and their weights are scalars.
template <typename T, bool ROWS, bool UNI, int K, int V, bool GEN> struct Thread {
  static constexpr int E = K * V;                     // elements of each tensor
  static constexpr int NP = ROWS ? 1 : V;             // pixels
  static constexpr int NW = ROWS ? E : K;             // channels
  static constexpr int NL = ROWS ? E : 1;             // channels whose weights a thread keeps (planes: they lie in LDS)
  static __device__ __forceinline__ constexpr int pix(int e) { return ROWS ? 0 : e % V; }
  static __device__ __forceinline__ constexpr int wi(int e) { return ROWS ? e : e / V; }
  typedef Vec<T, V> Raw;

  // a tile of the workgroup
  struct Pos {
    int64_t image, base;      // its first pixel within the image
    int64_t row;              // rows: the thread's row
    unsigned off;             // planes: bytes from `base` (and the wave's channel, if it has one) to the lane's first element
    int pdup;                 // planes: pixels that are not the lane's; rows: V where there is no such row
    bool full;                // nothing is dropped in this wave
  };
  const Args& a;
  float* lds;                 // reductions
  float* lw;                  // planes: weights by channel: gw, gb, w1, b1 (GEN) or gw, w1
  int round;
  int lane, wave, l;          // l = thread within the row / lane along the pixels
  int grp;                    // the thread's row of the workgroup / group of K channels
  int cb;                     // planes: first channel that is read: of the last group, like a vector's, such that all K exist
  int rdup[ROWS ? K : 1];     // rows: elements of step k that are not the thread's; planes: channels of the group that are not
  bool cfull;                 // nothing is dropped in this wave because of the channels
  unsigned off0;              // planes: Pos::off within a whole tile
  float gw_[NL], gb_[NL], w1_[NL], b1_[NL];

  __device__ __forceinline__ Thread(const Args& a_, float* lds_) : a(a_), lds(lds_), round(0) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    l = UNI ? lane : threadIdx.x & (a.lanes - 1);
    grp = UNI ? wave : threadIdx.x / a.lanes;
    bool ok = true;
    if (ROWS) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int over = (k * a.lanes + l) * V - (a.d.C - V);
        rdup[k] = over < 0 ? 0 : over < V ? over : V;
        ok = ok && over <= 0;
      }
    } else {
      const int last = a.d.C - K;
      cb = grp * K < last ? grp * K : last;
      rdup[0] = grp * K - cb;
      ok = rdup[0] == 0;
    }
    cfull = __all(ok);
    off0 = ((unsigned)(l * V) + (ROWS || UNI ? 0u : (unsigned)cb * (unsigned)a.P)) * (unsigned)sizeof(T);
    const int floats = 2 * WAVES * MAX_Q * (ROWS ? 1 : lanes() * V);
    lw = lds + floats;
    if (!ROWS && (int)blockDim.x < THREADS) {
      for (int i = threadIdx.x; i < floats; i += blockDim.x) lds[i] = 0;
      lds_barrier();
    }
  }
  __device__ __forceinline__ int lanes() const { return UNI ? 64 : a.lanes; }
  // first channel of step k
  __device__ __forceinline__ int ch(int k) const {
    if (ROWS) {
      const int c = (k * a.lanes + l) * V;
      return c < a.d.C - V ? c : a.d.C - V;
    }
    return cb + k;
  }
  // elements of step k that are not the thread's because of its channels
  __device__ __forceinline__ int cdup(int k) const { return ROWS ? rdup[k % (ROWS ? K : 1)] : k < rdup[0] ? V : 0; }
  __device__ __forceinline__ int dropped(int k, const Pos& o) const { return cdup(k) > o.pdup ? cdup(k) : o.pdup; }
  // whether an element's channel is the thread's (its pixel need not be)
  __device__ __forceinline__ bool chan_ok(int e) const { return ROWS ? e % V >= cdup(e / V) : cdup(e / V) == 0; }
  __device__ __forceinline__ int chan(int e) const { return ch(e / V) + (ROWS ? e % V : 0); }
  // pixels that a workgroup takes at a time
  __device__ __forceinline__ int tile() const { return ROWS ? (int)blockDim.x / a.lanes : lanes() * V; }
  __device__ __forceinline__ Pos at(int64_t img, int64_t base, int64_t end) const {
    Pos o;
    o.image = img;
    o.base = base;
    o.pdup = 0;
    o.full = cfull;
    if (base + tile() <= end) {
      if (ROWS) o.row = img * a.P + base + grp;
      else o.off = off0;
      return o;
    }
    const int64_t want = base + (ROWS ? grp : l * V), last = end - (ROWS ? 1 : V);
    if (ROWS) {
      o.row = img * a.P + (want < last ? want : last);
      o.pdup = want > last ? V : 0;
    } else {
      // where less than a vector is left behind the tile's start, the tile starts earlier
      const int64_t from = want < last ? want : last;
      o.pdup = want - from < V ? (int)(want - from) : V;
      if (base > last) o.base = last;
      o.off = ((unsigned)(from - o.base) + (UNI ? 0u : (unsigned)cb * (unsigned)a.P)) * (unsigned)sizeof(T);
    }
    o.full = cfull && __all(o.pdup == 0);
    return o;
  }
  // planes: a scalar base for each step, and 32 bits of bytes in one register for all of the kernel's accesses
  template <typename P> __device__ __forceinline__ P* first(P* p, int64_t stride, const Pos& o) const {
    return ROWS ? p + o.row * stride : p + (o.image * stride + o.base + (UNI ? cb * a.P : 0));
  }
  template <typename P> __device__ __forceinline__ P* address(P* q, int k, const Pos& o) const {
    if (ROWS) return q + ch(k);
    typedef typename std::conditional<std::is_const<P>::value, const char, char>::type Byte;
    return reinterpret_cast<P*>(reinterpret_cast<Byte*>(q + k * a.P) + o.off);
  }
  __device__ __forceinline__ void read(const void* p, int64_t stride, Raw* z, const Pos& o) const {
    const T* q = first(static_cast<const T*>(p), stride, o);
#pragma unroll
    for (int k = 0; k < K; ++k) z[k] = *reinterpret_cast<const Raw*>(address(q, k, o));
  }
  __device__ __forceinline__ void drop_dups(Raw* z, const Pos& o) const {
#pragma unroll
    for (int k = 0; k < K; ++k) drop<V>(z[k], dropped(k, o));
  }
  __device__ __forceinline__ void write(void* p, int64_t stride, const float* v, const Pos& o) const {
    T* q = first(static_cast<T*>(p), stride, o);
    if (o.full) {
#pragma unroll
      for (int k = 0; k < K; ++k) *reinterpret_cast<Raw*>(address(q, k, o)) = packed<V>(v + k * V, q);
      return;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      T* w = address(q, k, o);
      const int n = dropped(k, o);
      if (n == 0) *reinterpret_cast<Raw*>(w) = packed<V>(v + k * V, q);
      else if (n < V)
#pragma unroll
        for (int j = 1; j < V; ++j)
          if (j >= n) w[j] = (T)v[k * V + j];
    }
  }

  // ---- weights: the branch's factor and offset (u = gw n + gb; a full gate multiplies that per element) and the norm's after it
  template <int N> __device__ __forceinline__ static void weights(const float* w, float missing, int c, float* out) {
    if (w) {
      const Vec<float, N> z = *reinterpret_cast<const Vec<float, N>*>(w + c);
#pragma unroll
      for (int j = 0; j < N; ++j) out[j] = element<N>(z, j);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) out[j] = missing;
    }
  }
  // of N neighbouring channels
  template <int N> __device__ __forceinline__ void branch_weights(int64_t img, int c, float* gw, float* gb) const {
    const srx_resnorm_desc& d = a.d;
    const bool gated = d.gate_mode == GATE_CHANNEL || d.gate_mode == GATE_IMAGE;
    float G[N], w[N], b[N];
    weights<N>(gated ? static_cast<const float*>(d.gate) + (d.gate_mode == GATE_IMAGE ? img * d.C : 0) : nullptr, 1.f, c, G);
    weights<N>(d.w_post, 1.f, c, w);
    if (GEN) weights<N>(d.b_post, 0.f, c, b);
    if (gated && d.gate_act)
#pragma unroll
      for (int j = 0; j < N; ++j) G[j] = sigmoid(G[j]);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      gw[j] = d.scale * G[j] * w[j];
      if (GEN) gb[j] = d.scale * G[j] * b[j];
    }
  }
  // (an element that is not the thread's has n = 0 and dh = 0; its weights count only through offsets)
  __device__ __forceinline__ void branch(int64_t img) {
    if constexpr (ROWS) {
#pragma unroll
      for (int k = 0; k < K; ++k) branch_weights<V>(img, ch(k), gw_ + k * V, gb_ + k * V);
      if (GEN && !cfull)
#pragma unroll
        for (int e = 0; e < E; ++e) gb_[e] = chan_ok(e) ? gb_[e] : 0.f;
    } else {
      lds_barrier();
      for (int c = threadIdx.x; c < a.d.C; c += blockDim.x) {
        float g, b;
        branch_weights<1>(img, c, &g, &b);
        lw[c * (GEN ? 4 : 2)] = g;
        if (GEN) lw[c * 4 + 1] = b;
      }
      lds_barrier();
    }
  }
  __device__ __forceinline__ void norm_weights() {
    const srx_resnorm_desc& d = a.d;
    if constexpr (ROWS) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        weights<V>(d.w_pre, 1.f, ch(k), w1_ + k * V);
        if (GEN) weights<V>(d.b_pre, 0.f, ch(k), b1_ + k * V);
      }
    } else {
      for (int c = threadIdx.x; c < d.C; c += blockDim.x) {
        lw[c * (GEN ? 4 : 2) + (GEN ? 2 : 1)] = d.w_pre ? d.w_pre[c] : 1.f;
        if (GEN) lw[c * 4 + 3] = d.b_pre ? d.b_pre[c] : 0.f;
      }
      lds_barrier();
    }
  }
  __device__ __forceinline__ float gw(int e) const { return ROWS ? gw_[e % NL] : lw[ch(e / V) * (GEN ? 4 : 2)]; }
  __device__ __forceinline__ float gb(int e) const { return !GEN ? 0.f : ROWS ? gb_[e % NL] : cdup(e / V) ? 0.f : lw[ch(e / V) * 4 + 1]; }
  __device__ __forceinline__ float w1(int e) const { return ROWS ? w1_[e % NL] : lw[ch(e / V) * (GEN ? 4 : 2) + (GEN ? 2 : 1)]; }
  __device__ __forceinline__ float b1(int e) const { return !GEN ? 0.f : ROWS ? b1_[e % NL] : lw[ch(e / V) * 4 + 3]; }

  // ---- sums over the channels: of Q quantities, one value for each of the thread's pixels
  template <int Q> __device__ __forceinline__ void reduce(float (&s)[Q][NP]) {
    static_assert(Q <= MAX_Q, "");
    const int lo = ROWS ? 1 : lanes(), hi = ROWS ? (a.lanes < 64 ? a.lanes : 64) : 64;
    if (lo < hi) lanes_sum<Q * NP>(&s[0][0], lo, hi);
    // two buffers in turn: the barrier of one round keeps the next but one from overwriting what is still being read
    const int waves = ROWS ? a.lanes >> 6 : (int)blockDim.x >> 6;      // that share a pixel
    if (waves <= 1) return;
    constexpr int N = Q * NP;
    float* buf = lds + (round & 1) * (WAVES * (ROWS ? 1 : lanes()) * MAX_Q * NP);
    ++round;
    if (ROWS) {
      if (lane == 0)
#pragma unroll
        for (int q = 0; q < Q; ++q) buf[wave * N + q] = s[q][0];
      lds_barrier();
      const int w = (wave & ~(waves - 1)) + (lane & (waves - 1));
#pragma unroll
      for (int q = 0; q < Q; ++q) s[q][0] = buf[w * N + q];
      lanes_sum<N>(&s[0][0], 1, waves);
    } else {
      // slots of waves that the workgroup does not have hold zeros, whatever Q: all eight reads go out together
      const int per = lanes() * MAX_Q * NP;
      if (UNI || lane < lanes())
#pragma unroll
        for (int i = 0; i < N; ++i) buf[wave * per + l * N + i] = s[i / NP][i % NP];
      lds_barrier();
      float v[WAVES][N];
#pragma unroll
      for (int w = 0; w < WAVES; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i) v[w][i] = buf[w * per + l * N + i];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float sum = v[0][i];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) sum += v[w][i];
        s[i / NP][i % NP] = sum;
      }
    }
  }
  __device__ __forceinline__ void centre(float* z, const float* mean) const {
    if (cfull)
#pragma unroll
      for (int e = 0; e < E; ++e) z[e] -= mean[pix(e)];
    else
#pragma unroll
      for (int e = 0; e < E; ++e) z[e] -= chan_ok(e) ? mean[pix(e)] : 0.f;
  }
  // z -> (z - mean) / sqrt(var + eps) or z / sqrt(mean square + eps); returns the factor.  The variance is summed about the
  // mean, in a second round: E[z^2] - mean^2 would lose it for channels that sit far from zero.
  __device__ __forceinline__ void normalise(float* z, int kind, float eps, float* r) {
    const float inv = 1.f / (float)a.d.C;
    float s[1][NP];
    if (GEN && kind == KIND_LAYER) {
#pragma unroll
      for (int j = 0; j < NP; ++j) s[0][j] = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) s[0][pix(e)] += z[e];
      reduce<1>(s);
#pragma unroll
      for (int j = 0; j < NP; ++j) s[0][j] *= inv;
      centre(z, s[0]);
    }
#pragma unroll
    for (int j = 0; j < NP; ++j) s[0][j] = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) s[0][pix(e)] += z[e] * z[e];
    reduce<1>(s);
#pragma unroll
    for (int j = 0; j < NP; ++j) r[j] = rsqrt_hw(s[0][j] * inv + eps);
#pragma unroll
    for (int e = 0; e < E; ++e) z[e] *= r[pix(e)];
  }
  // u of one element; q: the full gate's raw values
  template <bool FULL> __device__ __forceinline__ float branch_value(int e, float n, const Raw* q) const {
    float u = GEN ? gw(e) * n + gb(e) : gw(e) * n;
    if (FULL) {
      const float g = element<V>(q[e / V], e % V);
      u *= a.d.gate_act ? sigmoid(g) : g;
    }
    return u;
  }
  // sum the thread's per-channel values over the workgroup and write them to out[C] (GEN: and a second set behind it)
  __device__ __forceinline__ void flush(float* first_set, float* second_set, float* out) {
    constexpr int Q = GEN ? 2 : 1;
    float* const sets[2] = {first_set, second_set};
    if (!ROWS) {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        lanes_sum<NW>(sets[q], 1, lanes());
        if (l == 0)
#pragma unroll
          for (int k = 0; k < K; ++k)
            if (cdup(k) == 0) out[q * a.d.C + ch(k)] = sets[q][k];
      }
      return;
    }
    if (a.lanes < 64)
#pragma unroll
      for (int q = 0; q < Q; ++q) lanes_sum<NW>(sets[q], a.lanes, 64);
    // waves that hold the same channels: every (lanes / 64)-th
    const int per_row = a.lanes > 64 ? a.lanes >> 6 : 1, waves = (int)blockDim.x >> 6;
    const bool first = wave < per_row && lane < a.lanes;
    if (waves > per_row) {
      lds_barrier();                     // the buffer may still be read as a reduction's
      if (lane < a.lanes)
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
          for (int i = 0; i < NW; ++i) lds[((wave * Q + q) * NW + i) * 64 + lane] = sets[q][i];
      lds_barrier();
      if (first)
        for (int w = wave + per_row; w < waves; w += per_row)
#pragma unroll
          for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int i = 0; i < NW; ++i) sets[q][i] += lds[((w * Q + q) * NW + i) * 64 + lane];
      lds_barrier();
    }
    if (first)
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        float* const to = out + q * a.d.C;
        if (cfull) {
#pragma unroll
          for (int k = 0; k < K; ++k) *reinterpret_cast<Vec<float, V>*>(to + ch(k)) = packed<V>(sets[q] + k * V, to);
        } else {
#pragma unroll
          for (int i = 0; i < NW; ++i)
            if (chan_ok(i)) to[chan(i)] = sets[q][i];
        }
      }
  }
};

// When the weights are fetched: once, and again where the gate is another image's.  Maps do it after their first tile's loads
// are on their way (16 x 64 x 64 x 64 bf16: forward 8.8 -> 8.5 us, backward 24.4 -> 22.2), rows in front of them: their
// weights are registers, which a branch in the loop would tie up (4096 x 1024 bf16: forward 8.6 against 9.3 us).
template <typename Th, bool ROWS> struct WeightsOf {
  Th& t;
  const bool has_branch, has_norm;
  int image = -1;
  __device__ __forceinline__ WeightsOf(Th& t_, bool f, bool n) : t(t_), has_branch(f), has_norm(n) {
    if (!ROWS) return;
    if (has_norm) t.norm_weights();
    if (has_branch && t.a.d.gate_mode != GATE_IMAGE) t.branch(0);
  }
  __device__ __forceinline__ void item(int img) {
    if (ROWS && has_branch && t.a.d.gate_mode == GATE_IMAGE) t.branch(img);
  }
  __device__ __forceinline__ void tile(int img) {
    if (ROWS) return;
    if (image < 0 && has_norm) t.norm_weights();
    if (has_branch && (image < 0 || (t.a.d.gate_mode == GATE_IMAGE && image != img))) t.branch(img);
    image = img;
  }
};

// The workgroup's first item.  Workgroups go to the eight dies in turn.  In maps each die takes 16 neighbouring tiles, which
// share cache lines where a tile has few pixels (many channels) or starts within a line (odd sizes): forward / backward,
// bf16, 8 x 1024 x 32 x 32 26 / 47 us against 65 / 115 in plain order, 64 x 64 x 127 x 129 112 / 229 against 153 / 253, 64 x 64
// x 128 x 128 102 / 175 against 102 / 173.  (One run for each die: 128 us forward there, eight places in memory at a time.)
constexpr int RUN = 16;
template <bool ROWS> __device__ __forceinline__ int first_item() {
  const int b = blockIdx.x;
  if (ROWS) return b;
  int run = (int)gridDim.x >> 3;
  run = run < RUN ? run : RUN;
  const int group = 8 * run, whole = run ? (int)gridDim.x / group * group : 0;
  if (b >= whole) return b;
  const int at = b / group * group, in = b - at;
  return at + (in & 7) * run + (in >> 3);
}

template <typename T, bool ROWS, bool UNI, int K, int V, bool FULL, bool GEN>
__global__ __launch_bounds__(THREADS) void resnorm_fwd_kernel(const Args a) {
  extern __shared__ float lds[];
  typedef Thread<T, ROWS, UNI, K, V, GEN> Th;
  Th t(a, lds);
  const srx_resnorm_desc& d = a.d;
  const int64_t step = (int64_t)a.slices * t.tile();
  const int start = first_item<ROWS>();
  int img = start / a.slices, share = start - img * a.slices;
  WeightsOf<Th, ROWS> w(t, d.f, d.pre_kind);
  for (int item = start; item < a.items; item += gridDim.x, a.next(img, share)) {
    w.item(img);
    const int64_t first = (int64_t)share * t.tile();
    for (int64_t base = first; base < a.P; base += step) {
      const typename Th::Pos o = t.at(img, base, a.P);
      typename Th::Raw xr[K], fr[K], qr[K];
      float y[Th::E], r[Th::NP];
      if (d.f) {
        t.read(d.f, d.f_stride, fr, o);
        t.read(d.x, d.x_stride, xr, o);
        if (FULL) t.read(d.gate, d.gate_stride, qr, o);
        w.tile(img);
        if (!o.full) {
          t.drop_dups(fr, o);
          t.drop_dups(xr, o);
          if (FULL) t.drop_dups(qr, o);
        }
        float n[Th::E];
#pragma unroll
        for (int e = 0; e < Th::E; ++e) n[e] = element<V>(fr[e / V], e % V);
        if (d.post_kind) t.normalise(n, d.post_kind, d.post_eps, r);
#pragma unroll
        for (int e = 0; e < Th::E; ++e) y[e] = element<V>(xr[e / V], e % V) + t.template branch_value<FULL>(e, n[e], qr);
        t.write(d.y, d.y_stride, y, o);
      } else {
        t.read(d.x, d.x_stride, xr, o);
        w.tile(img);
        if (!o.full) t.drop_dups(xr, o);
#pragma unroll
        for (int e = 0; e < Th::E; ++e) y[e] = element<V>(xr[e / V], e % V);
      }
      if (d.pre_kind) {
        t.normalise(y, d.pre_kind, d.pre_eps, r);
#pragma unroll
        for (int e = 0; e < Th::E; ++e) y[e] = GEN ? y[e] * t.w1(e) + t.b1(e) : y[e] * t.w1(e);
        t.write(d.h, d.h_stride, y, o);
      }
    }
  }
}

// With n the normalised y and g = dh w:  D = dy + r (g - n mean(g n) - [mean g]); as n = (y - mu) r, sum g n comes out of the
// same round of reductions as the variance.
// The branch's per-channel sums are
//   d w_post = s sum G D n,   d b_post = s sum G D,   d G = s sum D (w n + b),
// and where G is the same for all pixels of an image (or is 1) all three follow from sum D n and sum D: two
// accumulators a channel instead of three.  A full gate takes G D in D's place and writes its own gradient.
//
// ALL: every tensor is there (the pass between two branches), which the compiler has to know to wait for one tensor's loads
// and not for all that may have been issued.  (Reading the next tile while one is computed gained nothing: 177.7 us with and
// without it for 64 maps of 64 x 128 x 128 in bf16.)
template <typename T, bool ROWS, bool UNI, int K, int V, bool FULL, bool GEN, bool ALL>
__global__ __launch_bounds__(THREADS) void resnorm_bwd_kernel(const Args a) {
  extern __shared__ float lds[];
  typedef Thread<T, ROWS, UNI, K, V, GEN> Th;
  Th t(a, lds);
  const srx_resnorm_desc& d = a.d;
  const bool has_f = ALL || d.f, has_dh = ALL || d.dh, has_dy = ALL || d.dy;
  const float inv = 1.f / (float)d.C;
  float s_dhn[Th::NW] = {}, s_dh[Th::NW] = {}, s_dn[Th::NW] = {}, s_d[Th::NW] = {};
  const int64_t step = (int64_t)a.slices * t.tile();
  const int start = first_item<ROWS>();
  int img = start / a.slices, share = start - img * a.slices;
  WeightsOf<Th, ROWS> w(t, has_f, has_dh);
  for (int item = start; item < a.items; item += gridDim.x, a.next(img, share)) {
    w.item(img);
    for (int64_t base = (int64_t)share * t.tile(); base < a.P; base += step) {
      const typename Th::Pos o = t.at(img, base, a.P);
      typename Th::Raw xr[K], fr[K], qr[K], dyr[K], dhr[K];
      if (has_f) t.read(d.f, d.f_stride, fr, o);
      if (has_dh) t.read(d.x, d.x_stride, xr, o);
      if (FULL) t.read(d.gate, d.gate_stride, qr, o);
      if (has_dh) t.read(d.dh, d.dh_stride, dhr, o);
      if (has_dy) t.read(d.dy, d.dy_stride, dyr, o);
      w.tile(img);
      if (!o.full) {
        t.drop_dups(fr, o);
        t.drop_dups(xr, o);
        if (FULL) t.drop_dups(qr, o);
        t.drop_dups(dhr, o);
        t.drop_dups(dyr, o);
      }
      float D[Th::E], n[Th::E], r[Th::NP], r2[Th::NP];
      float s[2][Th::NP];
      if (has_f) {
#pragma unroll
        for (int e = 0; e < Th::E; ++e) n[e] = element<V>(fr[e / V], e % V);
        if (d.post_kind) t.normalise(n, d.post_kind, d.post_eps, r2);
      }
      if (has_dh) {
        float mean_g[Th::NP] = {};
        // y, in D's place for now
        if (has_f)
#pragma unroll
          for (int e = 0; e < Th::E; ++e) D[e] = element<V>(xr[e / V], e % V) + t.template branch_value<FULL>(e, n[e], qr);
        else
#pragma unroll
          for (int e = 0; e < Th::E; ++e) D[e] = element<V>(xr[e / V], e % V);
        if (GEN && d.pre_kind == KIND_LAYER) {
#pragma unroll
          for (int j = 0; j < Th::NP; ++j) s[0][j] = s[1][j] = 0;
#pragma unroll
          for (int e = 0; e < Th::E; ++e) { s[0][Th::pix(e)] += D[e]; s[1][Th::pix(e)] += element<V>(dhr[e / V], e % V) * t.w1(e); }
          t.template reduce<2>(s);
#pragma unroll
          for (int j = 0; j < Th::NP; ++j) { s[0][j] *= inv; mean_g[j] = s[1][j] * inv; }
          t.centre(D, s[0]);
        }
#pragma unroll
        for (int j = 0; j < Th::NP; ++j) s[0][j] = s[1][j] = 0;
#pragma unroll
        for (int e = 0; e < Th::E; ++e) {
          s[0][Th::pix(e)] += D[e] * D[e];
          s[1][Th::pix(e)] += element<V>(dhr[e / V], e % V) * t.w1(e) * D[e];
        }
        t.template reduce<2>(s);
#pragma unroll
        for (int j = 0; j < Th::NP; ++j) {
          r[j] = rsqrt_hw(s[0][j] * inv + d.pre_eps);
          s[1][j] *= inv * r[j];
        }
#pragma unroll
        for (int e = 0; e < Th::E; ++e) {
          const float g = element<V>(dhr[e / V], e % V), ny = D[e] * r[Th::pix(e)];
          s_dhn[Th::wi(e)] += g * ny;
          if (GEN) s_dh[Th::wi(e)] += g;
          D[e] = r[Th::pix(e)] * (GEN ? g * t.w1(e) - ny * s[1][Th::pix(e)] - mean_g[Th::pix(e)] : g * t.w1(e) - ny * s[1][Th::pix(e)]);
        }
        if (GEN && !o.full)           // what a mean's offset leaves where there is nothing
#pragma unroll
          for (int e = 0; e < Th::E; ++e) D[e] = e % V < t.dropped(e / V, o) ? 0.f : D[e];
        if (has_dy)
#pragma unroll
          for (int e = 0; e < Th::E; ++e) D[e] += element<V>(dyr[e / V], e % V);
      } else {
#pragma unroll
        for (int e = 0; e < Th::E; ++e) D[e] = element<V>(dyr[e / V], e % V);
      }
      if (ALL || d.dx) t.write(d.dx, d.dx_stride, D, o);
      if (has_f) {
        if (FULL) {
          float dq[Th::E];
#pragma unroll
          for (int e = 0; e < Th::E; ++e) {
            const float q = element<V>(qr[e / V], e % V), G = d.gate_act ? sigmoid(q) : q;
            dq[e] = D[e] * (GEN ? t.gw(e) * n[e] + t.gb(e) : t.gw(e) * n[e]) * (d.gate_act ? G * (1.f - G) : 1.f);
            D[e] *= G;
          }
          if (d.dgate) t.write(d.dgate, d.dgate_stride, dq, o);
        }
#pragma unroll
        for (int e = 0; e < Th::E; ++e) {
          s_dn[Th::wi(e)] += D[e] * n[e];
          if (GEN) s_d[Th::wi(e)] += D[e];
          D[e] *= t.gw(e);
        }
        if (ALL || d.df) {
          if (d.post_kind) {
#pragma unroll
            for (int j = 0; j < Th::NP; ++j) s[0][j] = s[1][j] = 0;
#pragma unroll
            for (int e = 0; e < Th::E; ++e) {
              s[0][Th::pix(e)] += D[e] * n[e];
              if (GEN) s[1][Th::pix(e)] += D[e];
            }
            if (GEN) t.template reduce<2>(s);
            else t.template reduce<1>(*reinterpret_cast<float(*)[1][Th::NP]>(&s));
#pragma unroll
            for (int j = 0; j < Th::NP; ++j) {
              s[0][j] *= inv;
              if (GEN) s[1][j] = d.post_kind == KIND_LAYER ? s[1][j] * inv : 0.f;
            }
#pragma unroll
            for (int e = 0; e < Th::E; ++e)
              D[e] = r2[Th::pix(e)] * (GEN ? D[e] - n[e] * s[0][Th::pix(e)] - s[1][Th::pix(e)] : D[e] - n[e] * s[0][Th::pix(e)]);
          }
          t.write(d.df, d.df_stride, D, o);
        }
      }
    }
    if (has_f && d.gate_mode == GATE_IMAGE) {
      t.flush(s_dn, s_d, a.part_post + (int64_t)item * 2 * d.C);
#pragma unroll
      for (int i = 0; i < Th::NW; ++i) s_dn[i] = s_d[i] = 0;
    }
  }
  if (has_dh) t.flush(s_dhn, s_dh, a.part_pre + (int64_t)blockIdx.x * 2 * d.C);
  if (has_f && d.gate_mode != GATE_IMAGE) t.flush(s_dn, s_d, a.part_post + (int64_t)blockIdx.x * 2 * d.C);
}

template <typename T, bool ROWS, bool UNI, int K, int V, bool FULL, bool GEN> int launch_with(const Plan& p, int backward, hipStream_t s) {
  const srx_resnorm_desc& d = p.a.d;
  if (backward && d.f && d.dh && d.dy && d.dx && d.df)
    hipLaunchKernelGGL((resnorm_bwd_kernel<T, ROWS, UNI, K, V, FULL, GEN, true>), dim3(p.workgroups), dim3(p.threads), p.lds_bytes, s, p.a);
  else if (backward)
    hipLaunchKernelGGL((resnorm_bwd_kernel<T, ROWS, UNI, K, V, FULL, GEN, false>), dim3(p.workgroups), dim3(p.threads), p.lds_bytes, s, p.a);
  else
    hipLaunchKernelGGL((resnorm_fwd_kernel<T, ROWS, UNI, K, V, FULL, GEN>), dim3(p.workgroups), dim3(p.threads), p.lds_bytes, s, p.a);
  return srx_check_launch(backward ? "resnorm_bwd" : "resnorm_fwd");
}
// whether there are means or offsets, or sums for them are wanted
inline bool general(const srx_resnorm_desc& d) {
  return d.post_kind == KIND_LAYER || d.pre_kind == KIND_LAYER || d.b_post || d.b_pre || d.db_post || d.db_pre;
}
template <typename T, bool ROWS, bool UNI, int K, int V> int launch_for(const Plan& p, int backward, hipStream_t s) {
  const bool gen = general(p.a.d);
  if (p.a.d.gate_mode == GATE_FULL)
    return gen ? launch_with<T, ROWS, UNI, K, V, true, true>(p, backward, s) : launch_with<T, ROWS, UNI, K, V, true, false>(p, backward, s);
  return gen ? launch_with<T, ROWS, UNI, K, V, false, true>(p, backward, s) : launch_with<T, ROWS, UNI, K, V, false, false>(p, backward, s);
}
template <typename T> int launch(const Plan& p, int backward, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  if (p.a.d.layout == SRX_RESNORM_PLANES) {
    const bool uni = p.a.lanes == 64;
    if (p.a.d.C < PLANES_K) return launch_for<T, false, true, 1, 2>(p, backward, s);
    if (p.elems == 4) return launch_with<T, false, false, PLANES_K, 4, false, false>(p, backward, s);
    if (p.elems == 1) return uni ? launch_for<T, false, true, PLANES_K, 1>(p, backward, s) : launch_for<T, false, false, PLANES_K, 1>(p, backward, s);
    return uni ? launch_for<T, false, true, PLANES_K, 2>(p, backward, s) : launch_for<T, false, false, PLANES_K, 2>(p, backward, s);
  }
  if (p.a.d.C < V) return launch_for<T, true, false, V, 1>(p, backward, s);           // rows shorter than a vector: one thread a row
  return p.elems == 8 ? launch_for<T, true, false, 8 / V, V>(p, backward, s) : launch_for<T, true, false, 16 / V, V>(p, backward, s);
}

}  // namespace resnorm
