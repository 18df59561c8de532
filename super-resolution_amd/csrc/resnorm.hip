// Norms around a gated residual branch: argument checks, decomposition, and the join of the sums over pixels.  The kernels
// are in resnorm_kernels.h.
#include <float.h>
#include "resnorm_kernels.h"

using namespace resnorm;

namespace {

// Joins the partial sums: 16 channels a workgroup, 64 threads a channel that take every 64th partial, in a fixed order.
constexpr int JOIN_X = 16, JOIN_Y = 64, JOIN_WAVES = JOIN_X * JOIN_Y / 64;
// Images whose gates one workgroup joins; with more, a launch of its own goes before the join.  A backward pass with it,
// without it (bf16): 8192 images of 16 x 256 rows 144 us, 737; 4096 of 64 x 8 x 8 127 us, 438; 256 of 512 x 256 rows 104 us, 117.
constexpr int JOIN_IMAGES = 64;
__host__ __device__ constexpr int join_groups(int images) { return images / JOIN_IMAGES + (images % JOIN_IMAGES > 0); }
// sums of p[i step] and, where second > 0, of p[i step + second] over i = y, y + EVERY, ... < n: eight loads of each in flight
// (a partial sum was written on another die: a load takes the better part of a microsecond)
template <int EVERY> __device__ __forceinline__ void join_sum(const float* p, int y, int n, int step, int second, float& s0, float& s1) {
  for (int i0 = y; i0 < n; i0 += 8 * EVERY) {
    float v[8], u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = i0 + j * EVERY;
      v[j] = i < n ? p[(int64_t)i * step] : 0.f;
      u[j] = second && i < n ? p[(int64_t)i * step + second] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) { s0 += v[j]; s1 += u[j]; }
  }
}
// Gates of images i0 <= i < i1: writes their gradients; s0, s1 += the images' sums of D n and D, times s G.  A wave takes an
// image: its four threads a channel share the image's partial sums, and the first of them holds the results.
__device__ __forceinline__ void join_images(const Args& a, int i0, int i1, int c, float w, float b, bool bias, float& s0, float& s1) {
  const srx_resnorm_desc& d = a.d;
  constexpr int YS = 64 / JOIN_X;
  const bool ok = c < d.C;
  const int y = threadIdx.x / JOIN_X & (YS - 1);
  const float* gate = static_cast<const float*>(d.gate);
  float* dgate = static_cast<float*>(d.dgate);
  for (int i = i0 + (threadIdx.x >> 6); i < i1; i += JOIN_WAVES) {
    float t[2] = {};
    if (ok) join_sum<YS>(a.part_post + (int64_t)i * a.slices * 2 * d.C + c, y, a.slices, 2 * d.C, bias ? d.C : 0, t[0], t[1]);
    lanes_sum<2>(t, JOIN_X, 64);
    if (!ok || y) continue;
    const float q = gate[(int64_t)i * d.C + c], G = d.gate_act ? sigmoid(q) : q;
    if (dgate) dgate[(int64_t)i * d.C + c] = d.scale * (w * t[0] + b * t[1]) * (d.gate_act ? G * (1.f - G) : 1.f);
    s0 += d.scale * G * t[0];
    s1 += d.scale * G * t[1];
  }
}
// the workgroup's sums over its threads of a channel, in a fixed order; for threads below 16, channels
template <int N> __device__ __forceinline__ void join_threads(float (&s)[N], float (*lds)[JOIN_WAVES][JOIN_X]) {
  const int x = threadIdx.x & (JOIN_X - 1);
  lanes_sum<N>(s, JOIN_X, 64);
  if ((threadIdx.x & 63) < JOIN_X)
#pragma unroll
    for (int i = 0; i < N; ++i) lds[i][threadIdx.x >> 6][x] = s[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s[i] = 0;
#pragma unroll
    for (int k = 0; k < JOIN_WAVES; ++k) s[i] += lds[i][k][x];
  }
}
// Many images: workgroup (., k) takes JOIN_IMAGES of them and leaves the sums of their gates at part_gate[k].
__global__ __launch_bounds__(JOIN_X* JOIN_Y) void resnorm_join_images_kernel(const Args a, float* part_gate, int images, bool bias) {
  __shared__ float lds[2][JOIN_WAVES][JOIN_X];
  const srx_resnorm_desc& d = a.d;
  const int c = blockIdx.y * JOIN_X + (threadIdx.x & (JOIN_X - 1)), i0 = blockIdx.x * JOIN_IMAGES;
  const bool ok = c < d.C;
  const float w = ok && d.w_post ? d.w_post[c] : 1.f, b = ok && d.b_post ? d.b_post[c] : 0.f;
  float s[2] = {};
  join_images(a, i0, images - i0 < JOIN_IMAGES ? images : i0 + JOIN_IMAGES, c, w, b, bias, s[0], s[1]);
  join_threads<2>(s, lds);
  if (threadIdx.x >= JOIN_X || !ok) return;
  part_gate[(int64_t)blockIdx.x * 2 * d.C + c] = s[0];
  part_gate[(int64_t)blockIdx.x * 2 * d.C + d.C + c] = s[1];
}
__global__ __launch_bounds__(JOIN_X* JOIN_Y) void resnorm_join_kernel(const Args a, const float* part_gate, int workgroups, int images, bool bias) {
  __shared__ float lds[4][JOIN_WAVES][JOIN_X];
  const srx_resnorm_desc& d = a.d;
  const int y = threadIdx.x / JOIN_X, c = blockIdx.x * JOIN_X + (threadIdx.x & (JOIN_X - 1));
  const bool ok = c < d.C, pre = d.dh && (d.dw_pre || d.db_pre);
  const float* gate = d.gate_mode == GATE_CHANNEL ? static_cast<const float*>(d.gate) : nullptr;
  float* dgate = gate ? static_cast<float*>(d.dgate) : nullptr;
  const float w = ok && d.w_post ? d.w_post[c] : 1.f, b = ok && d.b_post ? d.b_post[c] : 0.f;
  const float q = ok && gate ? gate[c] : 1.f;
  float s[4] = {};                       // sum dh n, sum dh, sum D n (image gates: times s G), sum D
  if (ok && pre) join_sum<JOIN_Y>(a.part_pre + c, y, workgroups, 2 * d.C, bias ? d.C : 0, s[0], s[1]);
  if (d.f && d.gate_mode == GATE_IMAGE) {
    if (part_gate) {
      if (ok) join_sum<JOIN_Y>(part_gate + c, y, join_groups(images), 2 * d.C, bias ? d.C : 0, s[2], s[3]);
    } else {
      join_images(a, 0, images, c, w, b, bias, s[2], s[3]);
    }
  } else if (ok && d.f) {
    join_sum<JOIN_Y>(a.part_post + c, y, workgroups, 2 * d.C, bias ? d.C : 0, s[2], s[3]);
  }
  join_threads<4>(s, lds);
  if (y > 0 || !ok) return;
  if (pre && d.dw_pre) d.dw_pre[c] = s[0];
  if (pre && d.db_pre) d.db_pre[c] = s[1];
  if (!d.f) return;
  if (d.gate_mode != GATE_IMAGE) {
    const float G = gate && d.gate_act ? sigmoid(q) : q;
    if (dgate) dgate[c] = d.scale * (w * s[2] + b * s[3]) * (gate && d.gate_act ? G * (1.f - G) : 1.f);
    s[2] *= d.scale * G;
    s[3] *= d.scale * G;
  }
  if (d.dw_post) d.dw_post[c] = s[2];
  if (d.db_post) d.db_post[c] = s[3];
}

// ------------------------------------------------------------------------------------------------ host side
constexpr int MAX_ROWS_C = SRX_RESNORM_MAX_ROWS_C, MAX_PLANES_C = SRX_RESNORM_MAX_PLANES_C;
static_assert(MAX_ROWS_C == 16 * THREADS, "");

int pow2_at_least(int64_t n) {
  int p = 1;
  while (p < n) p <<= 1;
  return p;
}

// The decomposition of a call; gen: whether it takes the general form.  Workspace size and launch use the same one.
void make_plan(const srx_resnorm_desc& d, int backward, bool gen, Plan& p) {
  p.a.d = d;
  if (d.P == 1) p.a.d.layout = SRX_RESNORM_ROWS;          // one pixel an image: its channels are contiguous
  const bool rows = p.a.d.layout == SRX_RESNORM_ROWS;
  const bool image_gate = d.f && d.gate_mode == GATE_IMAGE;
  p.images = rows && !image_gate ? 1 : d.B;
  p.a.P = rows && !image_gate ? (int64_t)d.B * d.P : d.P;
  // Backward: as many workgroups as run at once, since each pays for its start, its sums over the lanes and its partial sums
  // (about 9 us).
  int64_t most = backward ? 256 : 4096;
  int tile;
  if (rows) {
    // 16 elements a thread: where 8 would need more threads than there are, and where a wave then holds a row by itself and needs
    // no barrier: forward in bf16, 4096 rows of 1024 7.5 us against 8.2, 32768 of 520 27.3 against 30.3, with means 4096 of 1024
    // 10.3 against 11.3; not for few rows (100 of 768 3.9 against 3.5, 1000 4.3 against 4.2), a full gate beside (1531 of 1000 7.1
    // against 6.6), in fp32 (8192 of 777 25.1 against 20.9) or backward (registers).
    const bool row_in_wave = !backward && d.dtype == SRX_BF16 && d.gate_mode != GATE_FULL && d.C > 512 && d.C <= 1024 && p.a.P * p.images > 2048;
    p.elems = d.C <= 8 * THREADS && !row_in_wave ? 8 : 16;
    p.a.lanes = pow2_at_least((d.C + p.elems - 1) / p.elems);
    p.threads = backward || p.a.lanes > 256 ? THREADS : 256;
    // Registers (113 in lean rows, 132 with a full gate, 147 general, 175 both) leave a compute unit two workgroups of eight
    // waves, or one, or three and two of four waves.  The small ones need rows for their starts: from eight tiles each on.
    // One of eight waves against several of four: 32768 rows of 520 in bf16 full 122 -> 92 us, general 135 -> 104, both 164 -> 158,
    // fp32 general 185 -> 132; 4096 rows of 1024 29.7 -> 30.9, 1531 of 1000 24 -> 29.7 (not taken).
    const bool lean = !gen, full = d.gate_mode == GATE_FULL;
    if (backward && p.elems == 8 && lean && !full && d.C * (d.dtype == SRX_BF16 ? 2 : 4) >= 16) {
      most = 512;
    } else if (backward && p.elems == 8 && p.a.lanes <= 256) {
      const int64_t many = !lean && full ? 512 : 768;
      if (p.a.P * p.images / (256 / p.a.lanes) >= 8 * many) {
        p.threads = 256;
        most = many;
      }
    }
    tile = p.threads / p.a.lanes;
  } else {
    const int groups = d.C < PLANES_K ? d.C : (d.C + PLANES_K - 1) / PLANES_K;        // few channels: one a wave
    p.a.lanes = 64;
    while (groups * p.a.lanes > THREADS) p.a.lanes /= 2;
    p.threads = 64 * ((groups * p.a.lanes + 63) / 64);
    // Whole workgroups that fit by their registers (140 lean: 12 waves a compute unit; 160 to 224: 8): with a few more, the chip
    // runs twice for them (16 x 99 x 128 x 128 in bf16 178 us with 292, 112 with 256).  A channel a wave (60): more would fit than
    // pay (three channels of 16 x 128 x 128 17 us, 20 with 24 waves; seven 34 us with one workgroup, 24 with two).
    const bool light = p.a.lanes == 64 && !gen && d.gate_mode != GATE_FULL;
    const int resident = d.C < PLANES_K ? 14 : light ? 12 : 8, waves = p.threads / 64;
    if (backward) most *= waves < resident ? resident / waves : 1;
    // Pixels a thread: two; one where that leaves no more than half the compute units a workgroup (forward / backward, bf16: 1 x
    // 64 x 64 x 64 3.9 / 12.2 us against 4.9 / 12.7 with two, means 5.2 / 16.8 against 6.6 / 18.9; but 16 x 64 x 64 x 64 9.5 against
    // 8.7); four where few lanes lie along the pixels (16 x 512 x 64 x 64 50 / 136 against 54 / 167, 16 x 1024 x 64 x 64
    // 153 / 263 against 245 / 366; but 16 x 256 x 16 x 16 7.0 / 17.6 against 5.4 / 13.8) and nothing else needs the registers
    // (means: 8 x 1024 x 32 x 32 34 / 84 against 34 / 63).
    const auto tiles = [&](int v) { return (p.a.P + p.a.lanes * v - 1) / (p.a.lanes * v) * p.images; };
    p.elems = 2;
    if (d.C >= PLANES_K && tiles(2) <= 128) p.elems = 1;
    if (d.C > 256 && p.a.P >= 4 && tiles(4) >= 256 && !gen && d.gate_mode != GATE_FULL) p.elems = 4;
    tile = p.a.lanes * p.elems;
  }
  // Workgroups walk the tiles side by side, neighbours in time being neighbours in memory.  With a gate for each image an item
  // stays within its image, so that its sums are the image's.
  const int64_t tiles = (p.a.P + tile - 1) / tile;
  int64_t s = tiles;
  if (image_gate && p.images > 0) {
    // the shares of an image: as few rounds of workgroups as short as they can be (a share's own sums cost about two tiles); bf16
    // 20 x 64 x 64 x 64 backward 27.6 us against 34.8 with the least number that keeps all compute units busy, 300 images 229 against 303
    const int64_t base = most / p.images > 1 ? most / p.images : 1;
    int64_t best = 0;
    for (int64_t n = base; n <= base + 8 && n <= tiles; ++n) {
      const int64_t cost = (p.images * n + most - 1) / most * ((tiles + n - 1) / n + 2);
      if (!best || cost < best) { best = cost; s = n; }
    }
  }
  if (p.images > 0 && s > (1LL << 30) / p.images) s = (1LL << 30) / p.images;
  p.a.slices = s < 1 ? 1 : (int)s;
  p.a.items = p.a.P > 0 ? p.images * p.a.slices : 0;
  p.workgroups = (int)(p.a.items < most ? p.a.items : most);
  p.a.jump_images = p.workgroups / p.a.slices;
  p.a.jump_shares = p.workgroups % p.a.slices;
  const int waves = p.threads / 64;
  int bytes = 2 * WAVES * MAX_Q * (rows ? 1 : p.a.lanes * p.elems) * 4;            // two buffers of a reduction: at most 16 KB
  if (!rows) bytes += p.threads / p.a.lanes * PLANES_K * 16;                        // weights: at most 16 KB
  if (backward && rows && p.a.lanes < p.threads && bytes < waves * p.elems * 128 * 4) bytes = waves * p.elems * 128 * 4;   // flush: at most 64 KB
  p.lds_bytes = bytes;
}

// what a call computes: types, sizes, kinds
int check_form(const char* what, const srx_resnorm_desc* d) {
  SRX_CHECK_ARG(d != nullptr, "%s: null descriptor", what);
  SRX_CHECK_ARG(d->dtype == SRX_BF16 || d->dtype == SRX_F32, "%s: bad dtype %d", what, d->dtype);
  SRX_CHECK_ARG(d->layout == SRX_RESNORM_PLANES || d->layout == SRX_RESNORM_ROWS, "%s: bad layout %d", what, d->layout);
  SRX_CHECK_ARG(d->B >= 0 && d->P >= 0 && d->C > 0, "%s: bad sizes B %d C %d P %d", what, d->B, d->C, d->P);
  const bool by_image = (d->layout == SRX_RESNORM_PLANES && d->P > 1) || d->gate_mode == GATE_IMAGE;
  SRX_CHECK_ARG(!by_image || d->B <= (1 << 30), "%s: %d images, at most 2^30", what, d->B);
  const int most = d->layout == SRX_RESNORM_ROWS ? MAX_ROWS_C : MAX_PLANES_C;
  SRX_CHECK_ARG(d->C <= most, "%s: %d channels, at most %d in this layout", what, d->C, most);
  SRX_CHECK_ARG(d->post_kind >= 0 && d->post_kind <= 2 && d->pre_kind >= 0 && d->pre_kind <= 2, "%s: bad norm kind", what);
  SRX_CHECK_ARG(d->gate_mode >= 0 && d->gate_mode <= 3 && (d->gate_act == 0 || d->gate_act == 1), "%s: bad gate mode", what);
  SRX_CHECK_ARG((!d->post_kind || d->post_eps >= FLT_MIN) && (!d->pre_kind || d->pre_eps >= FLT_MIN), "%s: eps must be positive (a normal number)", what);
  // beyond 64 channels a workgroup's lanes address their channels with 32 bits
  SRX_CHECK_ARG(d->layout == SRX_RESNORM_ROWS || d->C <= 64 || (int64_t)d->C * d->P * (d->dtype == SRX_BF16 ? 2 : 4) < (1LL << 32),
                "%s: an image of more than 64 channels must stay under 4 GB", what);
  return SRX_OK;
}
// and what it computes on
int check(const char* what, const srx_resnorm_desc* d) {
  if (int rc = check_form(what, d)) return rc;
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

}  // namespace

extern "C" {

int64_t srx_resnorm_ws_floats(const srx_resnorm_desc* d) {
  if (check_form("srx_resnorm_ws_floats", d)) return -1;
  // enough for either form: addresses decide between them, and may not be there yet
  srx_resnorm_desc asked = *d;
  if (d->gate_mode) asked.f = &asked;                     // a gate is on a branch
  const bool image_gate = d->gate_mode == GATE_IMAGE;
  int64_t floats = 1;
  for (const bool gen : {false, true}) {
    Plan p = {};
    make_plan(asked, 1, gen, p);
    const int64_t need = 2 * (int64_t)d->C * (p.workgroups + (image_gate ? p.a.items + join_groups(p.images) : p.workgroups)) + 1;
    if (need > floats) floats = need;
  }
  return floats;
}

int srx_resnorm_forward(const srx_resnorm_desc* d, void* stream) {
  if (int rc = check("srx_resnorm_forward", d)) return rc;
  if ((int64_t)d->B * d->P == 0) return SRX_OK;
  SRX_CHECK_ARG(d->x && (!d->f || d->y) && (!d->pre_kind || d->h), "srx_resnorm_forward: null tensor");
  Plan p = {};
  make_plan(*d, 0, general(*d), p);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return d->dtype == SRX_BF16 ? launch_bf16(p, 0, s) : launch_f32(p, 0, s);
}

int srx_resnorm_backward(const srx_resnorm_desc* d, void* stream) {
  if (int rc = check("srx_resnorm_backward", d)) return rc;
  const bool empty = (int64_t)d->B * d->P == 0;
  SRX_CHECK_ARG(empty || d->dy || d->dh, "srx_resnorm_backward: neither dy nor dh");
  SRX_CHECK_ARG(!d->dh || (d->pre_kind && (d->x || empty)), "srx_resnorm_backward: dh needs the norm before the next branch, and x");
  SRX_CHECK_ARG(empty || d->ws, "srx_resnorm_backward: null workspace");
  Plan p = {};
  make_plan(*d, 1, general(*d), p);
  if (empty) p.a.slices = 0;            // the gradients of weights and gates are zeros
  p.a.part_pre = d->ws;
  p.a.part_post = d->ws + 2 * (int64_t)d->C * p.workgroups;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (!empty)
    if (int rc = d->dtype == SRX_BF16 ? launch_bf16(p, 1, s) : launch_f32(p, 1, s)) return rc;
  const bool sums = d->dw_pre || d->db_pre || (d->f && (d->dw_post || d->db_post || (d->dgate && d->gate_mode && d->gate_mode != GATE_FULL)));
  if (!sums) return SRX_OK;
  const unsigned channels = (d->C + JOIN_X - 1) / JOIN_X;
  float* part_gate = nullptr;
  if (d->f && d->gate_mode == GATE_IMAGE && p.images > JOIN_IMAGES && d->ws) {
    part_gate = p.a.part_post + 2 * (int64_t)d->C * p.a.items;
    hipLaunchKernelGGL(resnorm_join_images_kernel, dim3(join_groups(p.images), channels), dim3(JOIN_X * JOIN_Y), 0, s, p.a, part_gate, p.images, general(*d));
    if (int rc = srx_check_launch("resnorm_join_images")) return rc;
  }
  hipLaunchKernelGGL(resnorm_join_kernel, dim3(channels), dim3(JOIN_X * JOIN_Y), 0, s, p.a, part_gate, p.workgroups, p.images, general(*d));
  return srx_check_launch("resnorm_join");
}

}  // extern "C"
