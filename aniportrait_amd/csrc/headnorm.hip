// RMS norm of query and key heads with the position rotation, forward and backward (gfx950).
//   y = R(pos) (x rstd w),  rstd = (mean x^2 + eps)^-1/2,  R turns the channel pairs of the first `rot` channels by the table's
//   angles; pairs are (i, i + rot / 2) or (2 i, 2 i + 1).
//   backward: u = R^T dy, dw = sum u x rstd, dx = rstd (u w - x^ mean(u w x^)), x^ = x rstd.
// Bound by memory: one read and one write per element (backward two reads, one write), 7 - 18 operations between them.  A head is
// held by L = 4 .. 32 lanes, 8 channels each, chosen so that both halves of a lane's four pairs are its own: no value changes lanes
// but the sums.  A group of lanes walks over `hc` heads of one token, whose cos / sin it loads once.
#include "mapattn.h"

using namespace mapattn;

namespace {

struct HeadNormArgs {
  const void* x[2];
  int64_t x_sb[2], x_st[2], x_sh[2];
  void* y[2];
  int64_t y_sb[2], y_st[2], y_sh[2];
  const void* dy[2];
  int64_t dy_sb[2], dy_st[2], dy_sh[2];
  const float* w[2];
  const float* rope;
  const int* positions;
  int64_t M;
  int T, H[2], d, rot, hc, rope_rows, inter;
  float eps, inv_d, alpha;
  float* part;  // [block][2][d]
  float* dw[2];
  int nblk;
};

template <typename T>
__device__ __forceinline__ void widen(float (&x)[8], u32x2 u, u32x2 v) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x[2 * i] = Num<T>::lo(u[i]);
    x[2 * i + 1] = Num<T>::hi(u[i]);
    x[4 + 2 * i] = Num<T>::lo(v[i]);
    x[5 + 2 * i] = Num<T>::hi(v[i]);
  }
}
template <typename T>
__device__ __forceinline__ void load8(float (&x)[8], const char* row, int a, int b) {
  widen<T>(x, *(const u32x2*)(row + 2 * a), *(const u32x2*)(row + 2 * b));
}
template <typename T>
__device__ __forceinline__ void store8(char* row, int a, int b, const float (&x)[8]) {
  *(u32x2*)(row + 2 * a) = u32x2{Num<T>::pack(x[0], x[1]), Num<T>::pack(x[2], x[3])};
  *(u32x2*)(row + 2 * b) = u32x2{Num<T>::pack(x[4], x[5]), Num<T>::pack(x[6], x[7])};
}
template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// the lane's four pairs turned by the angles of cs = (cos, sin) x 4; sgn = -1 turns back
__device__ __forceinline__ void turn(float (&x)[8], const float (&cs)[8], bool inter, float sgn) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float c = cs[2 * i], s = sgn * cs[2 * i + 1];
    const float a = inter ? x[2 * i] : x[i], b = inter ? x[2 * i + 1] : x[4 + i];
    const float p = fmaf(a, c, -(b * s)), q = fmaf(a, s, b * c);
    if (inter) {
      x[2 * i] = p;
      x[2 * i + 1] = q;
    } else {
      x[i] = p;
      x[4 + i] = q;
    }
  }
}

// where a lane's channels lie, and its angles
struct Lane {
  int a, b;
  bool on, rot;
  __device__ __forceinline__ Lane(const HeadNormArgs& p, int j) {
    on = 8 * j < p.d;
    rot = 8 * j < p.rot;
    const bool half = rot && !p.inter;
    a = half ? 4 * j : 8 * j;
    b = half ? p.rot / 2 + 4 * j : 8 * j + 4;
  }
};
__device__ __forceinline__ void load_cs(float (&cs)[8], const HeadNormArgs& p, const Lane& ln, int64_t m, int t, int j) {
#pragma unroll
  for (int i = 0; i < 8; ++i) cs[i] = (i & 1) ? 0.f : 1.f;
  if (!ln.rot) return;
  int pos = p.positions ? p.positions[m] : t;
  pos = pos < 0 ? 0 : (pos >= p.rope_rows ? p.rope_rows - 1 : pos);
  const f32x4* src = (const f32x4*)(p.rope + (int64_t)pos * p.rot + 8 * j);
  const f32x4 u = src[0], v = src[1];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    cs[i] = u[i];
    cs[4 + i] = v[i];
  }
}

}  // namespace

template <typename T, int L>
__global__ __launch_bounds__(256) void head_norm_kernel(const HeadNormArgs p) {
  const int j = threadIdx.x % L;
  const int heads = p.H[0] + p.H[1], chunks = (heads + p.hc - 1) / p.hc;
  const int64_t item = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (item >= p.M * chunks) return;
  const int64_t m = item / chunks;
  const int h0 = (int)(item - m * chunks) * p.hc, h1 = min(h0 + p.hc, heads);
  const int64_t b = m / p.T;
  const int t = (int)(m - b * p.T);
  const Lane ln(p, j);
  float cs[8];
  load_cs(cs, p, ln, m, t, j);
  constexpr int U = 4;  // heads whose loads are in flight together
  for (int h2 = h0; h2 < h1; h2 += U) {
    float x[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int hh = h2 + u, w = hh >= p.H[0], h = w ? hh - p.H[0] : hh;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[u][i] = 0.f;
      if (ln.on && hh < h1) load8<T>(x[u], (const char*)p.x[w] + 2 * (b * p.x_sb[w] + t * p.x_st[w] + h * p.x_sh[w]), ln.a, ln.b);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int hh = h2 + u, w = hh >= p.H[0], h = w ? hh - p.H[0] : hh;
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x[u][i], x[u][i], ss);
      ss = group_sum<L>(ss);
      if (!ln.on || hh >= h1) continue;
      const float rstd = __builtin_amdgcn_rsqf(fmaf(ss, p.inv_d, p.eps));
      const f32x4 wa = *(const f32x4*)(p.w[w] + ln.a), wb = *(const f32x4*)(p.w[w] + ln.b);
      const float f = w ? rstd : rstd * p.alpha;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[u][i] *= f * wa[i];
        x[u][4 + i] *= f * wb[i];
      }
      if (ln.rot) turn(x[u], cs, p.inter, 1.f);
      store8<T>((char*)p.y[w] + 2 * (b * p.y_sb[w] + t * p.y_st[w] + h * p.y_sh[w]), ln.a, ln.b, x[u]);
    }
  }
}

template <typename T, int L>
__global__ __launch_bounds__(256) void head_norm_bwd_kernel(const HeadNormArgs p) {
  __shared__ float red[2][256 * 8];
  const int j = threadIdx.x % L, grp = threadIdx.x / L;
  const int heads = p.H[0] + p.H[1], chunks = (heads + p.hc - 1) / p.hc;
  const int64_t items = p.M * chunks;
  const Lane ln(p, j);
  float dw[2][8], wt[2][8];
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      dw[w][i] = 0.f;
      wt[w][i] = ln.on && p.w[w] ? p.w[w][(i < 4 ? ln.a : ln.b) + (i & 3)] : 0.f;
    }
  for (int64_t item = (int64_t)blockIdx.x * (256 / L) + grp; item < items; item += (int64_t)gridDim.x * (256 / L)) {
    const int64_t m = item / chunks;
    const int h0 = (int)(item - m * chunks) * p.hc, h1 = min(h0 + p.hc, heads);
    const int64_t b = m / p.T;
    const int t = (int)(m - b * p.T);
    float cs[8];
    load_cs(cs, p, ln, m, t, j);
    constexpr int U = 4;  // heads whose loads are in flight together
    for (int h2 = h0; h2 < h1; h2 += U) {
      u32x2 xa[U], xb[U], ga[U], gb[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int hh = h2 + k, w = hh >= p.H[0], h = w ? hh - p.H[0] : hh;
        xa[k] = xb[k] = ga[k] = gb[k] = u32x2{0u, 0u};
        if (ln.on && hh < h1) {
          const char* xr = (const char*)p.x[w] + 2 * (b * p.x_sb[w] + t * p.x_st[w] + h * p.x_sh[w]);
          const char* gr = (const char*)p.dy[w] + 2 * (b * p.dy_sb[w] + t * p.dy_st[w] + h * p.dy_sh[w]);
          xa[k] = *(const u32x2*)(xr + 2 * ln.a);
          xb[k] = *(const u32x2*)(xr + 2 * ln.b);
          ga[k] = *(const u32x2*)(gr + 2 * ln.a);
          gb[k] = *(const u32x2*)(gr + 2 * ln.b);
        }
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int hh = h2 + k, w = hh >= p.H[0], h = w ? hh - p.H[0] : hh;
        float x[8], u[8];
        widen<T>(x, xa[k], xb[k]);
        widen<T>(u, ga[k], gb[k]);
        if (ln.rot) turn(u, cs, p.inter, -1.f);
        float ss = 0.f, dot = 0.f;
        const float al = w ? 1.f : p.alpha;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ss = fmaf(x[i], x[i], ss);
          u[i] *= al;
          dot = fmaf(u[i] * (w ? wt[1][i] : wt[0][i]), x[i], dot);
        }
        ss = group_sum<L>(ss);
        dot = group_sum<L>(dot);
        const float rstd = __builtin_amdgcn_rsqf(fmaf(ss, p.inv_d, p.eps));
        const float c = dot * p.inv_d * rstd * rstd;  // mean(u w x^) rstd
        const float f0 = w ? 0.f : rstd, f1 = w ? rstd : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float g = u[i] * x[i];
          dw[0][i] = fmaf(g, f0, dw[0][i]);
          dw[1][i] = fmaf(g, f1, dw[1][i]);
          x[i] = rstd * fmaf(u[i], w ? wt[1][i] : wt[0][i], -(x[i] * c));
        }
        if (ln.on && hh < h1) store8<T>((char*)p.y[w] + 2 * (b * p.y_sb[w] + t * p.y_st[w] + h * p.y_sh[w]), ln.a, ln.b, x);
      }
    }
  }
  // ---- the workgroup's part of dw: groups added in their order --------------------------------------------------------------
  if (p.part == nullptr) return;
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (ln.on) red[w][grp * (8 * L) + (i < 4 ? ln.a : ln.b) + (i & 3)] = dw[w][i];
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * p.d; c += 256) {
    const int w = c >= p.d, ch = w ? c - p.d : c;
    float t = 0.f;
    for (int g = 0; g < 256 / L; ++g) t += red[w][g * (8 * L) + ch];
    p.part[((int64_t)blockIdx.x * 2 + w) * p.d + ch] = t;
  }
}

// dw[w][c] = sum of the blocks' parts: 64 channels x 16 slices of blocks per workgroup
__global__ __launch_bounds__(1024) void head_norm_dw_kernel(const HeadNormArgs p) {
  __shared__ float red[16][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), sl = threadIdx.x >> 6;
  float t = 0.f;
  if (c < 2 * p.d)
#pragma unroll 8
    for (int i = sl; i < p.nblk; i += 16) t += p.part[(int64_t)i * 2 * p.d + c];
  red[sl][threadIdx.x & 63] = t;
  __syncthreads();
  if (sl == 0 && c < 2 * p.d) {
    t = 0.f;
    for (int i = 0; i < 16; ++i) t += red[i][threadIdx.x];
    float* dst = c >= p.d ? p.dw[1] : p.dw[0];
    if (dst) dst[c >= p.d ? c - p.d : c] = t;
  }
}

namespace {

int check_side(const char* what, const char* side, const void* x, int64_t sb, int64_t st, int64_t sh) {
  ANIP_REQUIRE(x != nullptr, "%s: %s is NULL", what, side);
  ANIP_REQUIRE(((uintptr_t)x & 15) == 0 && sb % 8 == 0 && st % 8 == 0 && sh % 8 == 0, "%s: %s must be 16-byte aligned with strides that are multiples of 8 elements", what, side);
  return 0;
}

int fill(const char* what, const anip_qk_norm_params* p, bool backward, HeadNormArgs& a) {
  ANIP_REQUIRE(p != nullptr, "%s: NULL parameters", what);
  ANIP_REQUIRE(p->dtype == 0 || p->dtype == 1, "%s: dtype must be 0 (fp16) or 1 (bf16)", what);
  ANIP_REQUIRE(p->B >= 1 && p->T >= 1 && p->Hq >= 1 && p->Hkv >= 0, "%s: B, T, Hq >= 1 and Hkv >= 0 are wanted", what);
  ANIP_REQUIRE(p->d >= 8 && p->d <= 256 && p->d % 8 == 0, "%s: head width %d: a multiple of 8 up to 256 is wanted", what, p->d);
  ANIP_REQUIRE(p->rot >= 0 && p->rot <= p->d && p->rot % 8 == 0, "%s: rot %d: a multiple of 8 up to the head width is wanted", what, p->rot);
  ANIP_REQUIRE(p->rot == 0 || (p->rope != nullptr && p->rope_rows >= 1 && ((uintptr_t)p->rope & 15) == 0), "%s: the rotation needs its table, 16-byte aligned", what);
  ANIP_REQUIRE(p->rot == 0 || p->positions != nullptr || p->rope_rows >= p->T, "%s: the rotation table has %d rows for %d tokens", what, p->rope_rows, p->T);
  ANIP_REQUIRE(p->q_weight != nullptr && ((uintptr_t)p->q_weight & 15) == 0, "%s: q_weight is wanted, 16-byte aligned", what);
  ANIP_REQUIRE(p->Hkv == 0 || (p->k_weight != nullptr && ((uintptr_t)p->k_weight & 15) == 0), "%s: k_weight is wanted, 16-byte aligned", what);
  ANIP_REQUIRE((int64_t)p->B * p->T * (p->Hq + p->Hkv) < (1ll << 33), "%s: too many heads in all", what);
  a = HeadNormArgs{};
  a.M = (int64_t)p->B * p->T;
  a.T = p->T;
  a.H[0] = p->Hq;
  a.H[1] = p->Hkv;
  a.d = p->d;
  a.rot = p->rot;
  a.inter = p->interleaved != 0;
  a.eps = p->eps;
  a.inv_d = 1.0f / p->d;
  a.alpha = p->q_alpha;
  a.w[0] = p->q_weight;
  a.w[1] = p->k_weight;
  a.rope = p->rope;
  a.rope_rows = p->rope_rows;
  a.positions = p->positions;
  const void* x[2] = {p->q, p->k};
  const int64_t* xs[2] = {p->q_stride, p->k_stride};
  void* y[2] = {p->q_out, p->k_out};
  const int64_t* ys[2] = {p->q_out_stride, p->k_out_stride};
  const void* g[2] = {p->dq_out, p->dk_out};
  const int64_t* gs[2] = {p->dq_out_stride, p->dk_out_stride};
  for (int w = 0; w < (p->Hkv ? 2 : 1); ++w) {
    if (check_side(what, w ? "k" : "q", x[w], xs[w][0], xs[w][1], xs[w][2])) return -1;
    if (check_side(what, w ? "the output for k" : "the output for q", y[w], ys[w][0], ys[w][1], ys[w][2])) return -1;
    if (backward && check_side(what, w ? "dk_out" : "dq_out", g[w], gs[w][0], gs[w][1], gs[w][2])) return -1;
    a.x[w] = x[w], a.x_sb[w] = xs[w][0], a.x_st[w] = xs[w][1], a.x_sh[w] = xs[w][2];
    a.y[w] = y[w], a.y_sb[w] = ys[w][0], a.y_st[w] = ys[w][1], a.y_sh[w] = ys[w][2];
    a.dy[w] = g[w], a.dy_sb[w] = gs[w][0], a.dy_st[w] = gs[w][1], a.dy_sh[w] = gs[w][2];
  }
  return 0;
}

int lanes_of(int d) { return d <= 32 ? 4 : d <= 64 ? 8 : d <= 128 ? 16 : 32; }
// heads per group of lanes: as many as leave 4 waves for every SIMD, 8 at most
int heads_per_group(int64_t M, int heads, int L) {
  for (int hc = 8; hc > 1; hc /= 2)
    if (M * ((heads + hc - 1) / hc) * L / 64 >= 4096) return hc;
  return 1;
}

template <typename T>
int run_fwd(const HeadNormArgs& a, int L, hipStream_t s) {
  const int64_t items = a.M * ((a.H[0] + a.H[1] + a.hc - 1) / a.hc);
  const dim3 grid((unsigned)cdiv64(items, 256 / L));
  switch (L) {
    case 4: hipLaunchKernelGGL((head_norm_kernel<T, 4>), grid, dim3(256), 0, s, a); break;
    case 8: hipLaunchKernelGGL((head_norm_kernel<T, 8>), grid, dim3(256), 0, s, a); break;
    case 16: hipLaunchKernelGGL((head_norm_kernel<T, 16>), grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL((head_norm_kernel<T, 32>), grid, dim3(256), 0, s, a);
  }
  ANIP_LAUNCH_CHECK("head_norm_kernel");
  return 0;
}
template <typename T>
int run_bwd(const HeadNormArgs& a, int L, hipStream_t s) {
  const dim3 grid((unsigned)a.nblk);
  switch (L) {
    case 4: hipLaunchKernelGGL((head_norm_bwd_kernel<T, 4>), grid, dim3(256), 0, s, a); break;
    case 8: hipLaunchKernelGGL((head_norm_bwd_kernel<T, 8>), grid, dim3(256), 0, s, a); break;
    case 16: hipLaunchKernelGGL((head_norm_bwd_kernel<T, 16>), grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL((head_norm_bwd_kernel<T, 32>), grid, dim3(256), 0, s, a);
  }
  ANIP_LAUNCH_CHECK("head_norm_bwd_kernel");
  hipLaunchKernelGGL(head_norm_dw_kernel, dim3((unsigned)((2 * a.d + 63) / 64)), dim3(1024), 0, s, a);
  ANIP_LAUNCH_CHECK("head_norm_dw_kernel");
  return 0;
}

int bwd_blocks(int64_t M, int heads, int hc, int L) {
  const int64_t want = cdiv64(M * ((heads + hc - 1) / hc), 256 / L);
  return (int)(want < 1024 ? want : 1024);
}

}  // namespace

extern "C" int anip_qk_norm_rope(const anip_qk_norm_params* p, void* stream) {
  HeadNormArgs a;
  const int rc = fill("anip_qk_norm_rope", p, false, a);
  if (rc) return rc;
  const int L = lanes_of(a.d);
  a.hc = heads_per_group(a.M, a.H[0] + a.H[1], L);
  AnipProfScope prof_(ANIP_K_QK_NORM, stream);
  return p->dtype ? run_fwd<bf16_t>(a, L, (hipStream_t)stream) : run_fwd<f16>(a, L, (hipStream_t)stream);
}

extern "C" int64_t anip_qk_norm_rope_backward_ws_floats(int64_t M, int heads, int d) {
  if (M < 1 || heads < 1 || d < 8 || d > 256) return 0;
  const int L = lanes_of(d);
  return (int64_t)bwd_blocks(M, heads, heads_per_group(M, heads, L), L) * 2 * d;
}

extern "C" int anip_qk_norm_rope_backward(const anip_qk_norm_params* p, void* stream) {
  HeadNormArgs a;
  const int rc = fill("anip_qk_norm_rope_backward", p, true, a);
  if (rc) return rc;
  ANIP_REQUIRE(p->ws != nullptr && p->dq_weight != nullptr && (p->Hkv == 0 || p->dk_weight != nullptr), "anip_qk_norm_rope_backward: ws and the weights' gradients are wanted");
  const int L = lanes_of(a.d), heads = a.H[0] + a.H[1];
  a.hc = heads_per_group(a.M, heads, L);
  a.nblk = bwd_blocks(a.M, heads, a.hc, L);
  ANIP_REQUIRE(p->ws_floats >= (int64_t)a.nblk * 2 * a.d, "anip_qk_norm_rope_backward: ws holds %lld floats, %lld are wanted", (long long)p->ws_floats, (long long)a.nblk * 2 * a.d);
  a.part = p->ws;
  a.dw[0] = p->dq_weight;
  a.dw[1] = p->Hkv ? p->dk_weight : nullptr;
  AnipProfScope prof_(ANIP_K_QK_NORM, stream);
  return p->dtype ? run_bwd<bf16_t>(a, L, (hipStream_t)stream) : run_bwd<f16>(a, L, (hipStream_t)stream);
}
