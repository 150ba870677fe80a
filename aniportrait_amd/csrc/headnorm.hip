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
  uint32_t items;
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
__device__ __forceinline__ void store8(char* row, int a, int b, const float (&x)[8]) {
  *(u32x2*)(row + 2 * a) = u32x2{Num<T>::pack(x[0], x[1]), Num<T>::pack(x[2], x[3])};
  *(u32x2*)(row + 2 * b) = u32x2{Num<T>::pack(x[4], x[5]), Num<T>::pack(x[6], x[7])};
}
// sum over groups of L lanes, in the vector ALU: quads, then mirrored halves and rows of 16, then the row 16 lanes on
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), CTRL, 0xF, 0xF, true));
}
template <int L>
__device__ __forceinline__ float group_sum(float v) {
  v = dpp_add<0xB1>(v);                // quad_perm [1, 0, 3, 2]
  v = dpp_add<0x4E>(v);                // quad_perm [2, 3, 0, 1]
  if (L >= 8) v = dpp_add<0x141>(v);   // row_half_mirror
  if (L >= 16) v = dpp_add<0x140>(v);  // row_mirror
  if (L == 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}
// the lane's four pairs turned by the angles of cs = (cos, sin) x 4; sgn = -1 turns back
template <bool INTER>
__device__ __forceinline__ void turn(float (&x)[8], const float (&cs)[8], float sgn) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float c = cs[2 * i], s = sgn * cs[2 * i + 1];
    float& a = x[INTER ? 2 * i : i];
    float& b = x[INTER ? 2 * i + 1 : 4 + i];
    const float p = fmaf(a, c, -(b * s)), q = fmaf(a, s, b * c);
    a = p;
    b = q;
  }
}

// where a lane's channels lie, and its angles
struct Lane {
  int a, b;
  bool on, rot;
  __device__ __forceinline__ Lane(const HeadNormArgs& p, int j, bool inter) {
    on = 8 * j < p.d;
    rot = 8 * j < p.rot;
    const bool half = rot && !inter;
    a = half ? 4 * j : 8 * j;
    b = half ? p.rot / 2 + 4 * j : 8 * j + 4;
  }
};
__device__ __forceinline__ void load_cs(float (&cs)[8], const HeadNormArgs& p, const Lane& ln, uint32_t m, int t, int j) {
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

// a group of lanes' share of the work: up to hc heads of one token, all of them query heads (w = 0) or key heads (w = 1)
struct Item {
  uint32_t m, b, t;  // token, its sequence and place there (fewer than 2^31 items: 32-bit divisions, 20 instructions instead of 140)
  int w, h0, n;
  __device__ __forceinline__ Item(const HeadNormArgs& p, uint32_t item) {
    const uint32_t cq = (p.H[0] + p.hc - 1) / p.hc, ck = (p.H[1] + p.hc - 1) / p.hc;
    m = item / (cq + ck);
    uint32_t c = item - m * (cq + ck);
    b = m / (uint32_t)p.T;
    t = m - b * p.T;
    w = c >= cq;
    if (w) c -= cq;
    h0 = (int)c * p.hc;
    n = min(p.hc, (w ? p.H[1] : p.H[0]) - h0);
  }
};

template <typename T, int L, bool INTER>
__global__ __launch_bounds__(256) void head_norm_kernel(const HeadNormArgs p) {
  constexpr int U = 4;  // heads whose loads are in flight together
  const int j = threadIdx.x % L;
  const uint32_t item = blockIdx.x * (256 / L) + threadIdx.x / L;
  if (item >= p.items) return;
  const Item it(p, item);
  const int w = it.w;
  const int64_t b = it.b, t = it.t;
  const Lane ln(p, j, INTER);
  const char* src = (const char*)p.x[w] + 2 * (b * p.x_sb[w] + t * p.x_st[w] + it.h0 * p.x_sh[w]);
  char* dst = (char*)p.y[w] + 2 * (b * p.y_sb[w] + t * p.y_st[w] + it.h0 * p.y_sh[w]);
  const int64_t sh = p.x_sh[w] * 2, dh = p.y_sh[w] * 2;
  u32x2 xa[U], xb[U];
  auto load = [&](int h) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      xa[u] = xb[u] = u32x2{0u, 0u};
      if (ln.on && h + u < it.n) {
        xa[u] = *(const u32x2*)(src + u * sh + 2 * ln.a);
        xb[u] = *(const u32x2*)(src + u * sh + 2 * ln.b);
      }
    }
    src += U * sh;
  };
  load(0);
  float cs[8], wt[8];
  load_cs(cs, p, ln, it.m, it.t, j);
  const float f0 = w ? 1.f : p.alpha;
#pragma unroll
  for (int i = 0; i < 8; ++i) wt[i] = ln.on ? f0 * p.w[w][(i < 4 ? ln.a : ln.b) + (i & 3)] : 0.f;
  for (int h = 0;;) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[8];
      widen<T>(x, xa[u], xb[u]);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
      const float rstd = __builtin_amdgcn_rsqf(fmaf(group_sum<L>(ss), p.inv_d, p.eps));
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * rstd * wt[i];
      if (ln.rot) turn<INTER>(x, cs, 1.f);
      if (ln.on && h + u < it.n) store8<T>(dst + u * dh, ln.a, ln.b, x);
    }
    h += U;
    dst += U * dh;
    if (h >= it.n) break;
    load(h);
  }
}

template <typename T, int L, bool INTER>
__global__ __launch_bounds__(256) void head_norm_bwd_kernel(const HeadNormArgs p) {
  constexpr int U = 2;  // (4: 162 registers, three waves per SIMD, 87 us against 70 at 524 672 heads of 80)
  __shared__ float red[2][256 * 8];
  const int j = threadIdx.x % L, grp = threadIdx.x / L;
  const Lane ln(p, j, INTER);
  float dw[2][8];
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[w][i] = 0.f;
  for (uint32_t item = blockIdx.x * (256 / L) + grp; item < p.items; item += gridDim.x * (256 / L)) {
    const Item it(p, item);
    const int w = it.w;
    const int64_t b = it.b, t = it.t;
    const char* xr = (const char*)p.x[w] + 2 * (b * p.x_sb[w] + t * p.x_st[w] + it.h0 * p.x_sh[w]);
    const char* gr = (const char*)p.dy[w] + 2 * (b * p.dy_sb[w] + t * p.dy_st[w] + it.h0 * p.dy_sh[w]);
    char* yr = (char*)p.y[w] + 2 * (b * p.y_sb[w] + t * p.y_st[w] + it.h0 * p.y_sh[w]);
    const int64_t xh = p.x_sh[w] * 2, gh = p.dy_sh[w] * 2, yh = p.y_sh[w] * 2;
    u32x2 xa[U], xb[U], ga[U], gb[U];
    auto load = [&](int h) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        xa[u] = xb[u] = ga[u] = gb[u] = u32x2{0u, 0u};
        if (ln.on && h + u < it.n) {
          xa[u] = *(const u32x2*)(xr + u * xh + 2 * ln.a);
          xb[u] = *(const u32x2*)(xr + u * xh + 2 * ln.b);
          ga[u] = *(const u32x2*)(gr + u * gh + 2 * ln.a);
          gb[u] = *(const u32x2*)(gr + u * gh + 2 * ln.b);
        }
      }
      xr += U * xh;
      gr += U * gh;
    };
    load(0);
    float cs[8], wt[8], acc[8];
    load_cs(cs, p, ln, it.m, it.t, j);
    const float al = w ? 1.f : p.alpha;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      wt[i] = ln.on ? al * p.w[w][(i < 4 ? ln.a : ln.b) + (i & 3)] : 0.f;
      acc[i] = 0.f;
    }
    for (int h = 0;;) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        float x[8], u[8];
        widen<T>(x, xa[k], xb[k]);
        widen<T>(u, ga[k], gb[k]);
        if (ln.rot) turn<INTER>(u, cs, -1.f);
        float ss = 0.f, dot = 0.f, g[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ss = fmaf(x[i], x[i], ss);
          g[i] = u[i] * x[i];
          dot = fmaf(g[i], wt[i], dot);
        }
        // (a head behind the last is zeros: it adds nothing, also with eps = 0)
        const float rstd = h + k < it.n ? __builtin_amdgcn_rsqf(fmaf(group_sum<L>(ss), p.inv_d, p.eps)) : 0.f;
        const float c = -group_sum<L>(dot) * p.inv_d * rstd * rstd * rstd;  // -mean(u w x^) rstd^2: meets x
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc[i] = fmaf(g[i], rstd, acc[i]);
          x[i] = fmaf(u[i] * wt[i], rstd, x[i] * c);
        }
        if (ln.on && h + k < it.n) store8<T>(yr + k * yh, ln.a, ln.b, x);
      }
      h += U;
      yr += U * yh;
      if (h >= it.n) break;
      load(h);
    }
    const float aq = w ? 0.f : al, ak = w ? 1.f : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      dw[0][i] = fmaf(acc[i], aq, dw[0][i]);
      dw[1][i] = fmaf(acc[i], ak, dw[1][i]);
    }
  }
  // ---- the workgroup's part of dw: groups added in their order --------------------------------------------------------------
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
  ANIP_REQUIRE(p->eps >= 0.f && p->eps < 1e30f, "%s: eps must not be negative", what);
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
int64_t items_of(int64_t M, int Hq, int Hkv, int hc) { return M * ((Hq + hc - 1) / hc + (Hkv + hc - 1) / hc); }
// heads per group of lanes: as many, up to 8, as leave 4 waves for every SIMD
int heads_per_group(int64_t M, int Hq, int Hkv, int L) {
  for (int hc = 8; hc > 1; hc /= 2)
    if (items_of(M, Hq, Hkv, hc) * L / 64 >= 4096) return hc;
  return 1;
}
int set_items(HeadNormArgs& a) {
  const int64_t n = items_of(a.M, a.H[0], a.H[1], a.hc);
  ANIP_REQUIRE(n < (1ll << 31), "anip_qk_norm_rope: %lld groups of heads are too many for one launch", (long long)n);
  a.items = (uint32_t)n;
  return 0;
}
int bwd_blocks(int64_t items, int L) {
  const int64_t want = cdiv64(items, 256 / L);
  return (int)(want < 1024 ? want : 1024);
}

template <typename T, bool INTER>
int run_fwd(const HeadNormArgs& a, int L, hipStream_t s) {
  const unsigned n = mapattn_grid("head_norm_kernel", cdiv64(a.items, 256 / L), 256);
  if (!n) return -1;
  const dim3 grid(n);
  switch (L) {
    case 4: hipLaunchKernelGGL((head_norm_kernel<T, 4, INTER>), grid, dim3(256), 0, s, a); break;
    case 8: hipLaunchKernelGGL((head_norm_kernel<T, 8, INTER>), grid, dim3(256), 0, s, a); break;
    case 16: hipLaunchKernelGGL((head_norm_kernel<T, 16, INTER>), grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL((head_norm_kernel<T, 32, INTER>), grid, dim3(256), 0, s, a);
  }
  ANIP_LAUNCH_CHECK("head_norm_kernel");
  return 0;
}
template <typename T, bool INTER>
int run_bwd(const HeadNormArgs& a, int L, hipStream_t s) {
  const dim3 grid((unsigned)a.nblk);
  switch (L) {
    case 4: hipLaunchKernelGGL((head_norm_bwd_kernel<T, 4, INTER>), grid, dim3(256), 0, s, a); break;
    case 8: hipLaunchKernelGGL((head_norm_bwd_kernel<T, 8, INTER>), grid, dim3(256), 0, s, a); break;
    case 16: hipLaunchKernelGGL((head_norm_bwd_kernel<T, 16, INTER>), grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL((head_norm_bwd_kernel<T, 32, INTER>), grid, dim3(256), 0, s, a);
  }
  ANIP_LAUNCH_CHECK("head_norm_bwd_kernel");
  hipLaunchKernelGGL(head_norm_dw_kernel, dim3((unsigned)((2 * a.d + 63) / 64)), dim3(1024), 0, s, a);
  ANIP_LAUNCH_CHECK("head_norm_dw_kernel");
  return 0;
}

}  // namespace

extern "C" int anip_qk_norm_rope(const anip_qk_norm_params* p, void* stream) {
  HeadNormArgs a;
  const int rc = fill("anip_qk_norm_rope", p, false, a);
  if (rc) return rc;
  const int L = lanes_of(a.d);
  a.hc = heads_per_group(a.M, a.H[0], a.H[1], L);
  if (set_items(a) != 0) return -1;
  hipStream_t s = (hipStream_t)stream;
  AnipProfScope prof_(ANIP_K_QK_NORM, stream);
  if (p->dtype) return a.inter ? run_fwd<bf16_t, true>(a, L, s) : run_fwd<bf16_t, false>(a, L, s);
  return a.inter ? run_fwd<f16, true>(a, L, s) : run_fwd<f16, false>(a, L, s);
}

extern "C" int64_t anip_qk_norm_rope_backward_ws_floats(int64_t M, int Hq, int Hkv, int d) {
  if (M < 1 || Hq < 1 || Hkv < 0 || d < 8 || d > 256) return 0;
  const int L = lanes_of(d);
  return (int64_t)bwd_blocks(items_of(M, Hq, Hkv, heads_per_group(M, Hq, Hkv, L)), L) * 2 * d;
}

extern "C" int anip_qk_norm_rope_backward(const anip_qk_norm_params* p, void* stream) {
  HeadNormArgs a;
  const int rc = fill("anip_qk_norm_rope_backward", p, true, a);
  if (rc) return rc;
  ANIP_REQUIRE(p->ws != nullptr && p->dq_weight != nullptr && (p->Hkv == 0 || p->dk_weight != nullptr), "anip_qk_norm_rope_backward: ws and the weights' gradients are wanted");
  const int L = lanes_of(a.d);
  a.hc = heads_per_group(a.M, a.H[0], a.H[1], L);
  if (set_items(a) != 0) return -1;
  a.nblk = bwd_blocks(a.items, L);
  ANIP_REQUIRE(p->ws_floats >= (int64_t)a.nblk * 2 * a.d, "anip_qk_norm_rope_backward: ws holds %lld floats, %lld are wanted", (long long)p->ws_floats, (long long)a.nblk * 2 * a.d);
  a.part = p->ws;
  a.dw[0] = p->dq_weight;
  a.dw[1] = p->Hkv ? p->dk_weight : nullptr;
  hipStream_t s = (hipStream_t)stream;
  AnipProfScope prof_(ANIP_K_QK_NORM, stream);
  if (p->dtype) return a.inter ? run_bwd<bf16_t, true>(a, L, s) : run_bwd<bf16_t, false>(a, L, s);
  return a.inter ? run_bwd<f16, true>(a, L, s) : run_bwd<f16, false>(a, L, s);
}
