// Attention over one or two softmax maps (gfx950): what the forward, single-token and backward kernels share.
//   MAPS = 1: o_i = softmax_j(scale q_i.k_j + table[h][bucket(j - p_i)]) v_j          (learned bias by relative position)
//   MAPS = 2: o_i = (softmax_j(scale q1_i.k1_j) - lam_h softmax_j(scale q2_i.k2_j)) v_j   (differential attention, dv = 2 d)
// p_i = q_start[b] + i is the position of query i; key j is seen if j < kv_lens[b] and, when causal, j <= p_i.
//
// Matrix products run on v_mfma_f32_32x32x16 with the operands arranged so that no value changes lanes between two of them:
// lane (l & 31, h = l >> 5) of an accumulator holds column l & 31 and rows 8 (r / 4) + 4 h + r % 4, r = 0 .. 15, of a 32 x 32
// tile.  Its registers 8 s .. 8 s + 7 are, as they lie, the B operand of the next product over the 16 rows 16 s ..: contraction
// slot (h, i) then stands for row 16 s + 8 (i / 4) + 4 h + i % 4, and the A operand is read in the same order.  A operands that
// need the transposed tile (V^T, K^T, Q^T, dO^T) are read from the row-major tile with ds_read_b64_tr_b16: 16 lanes fetch a
// 4 x 16 block, lane i receives its column i.
#pragma once
#include "common.h"

struct MapAttnArgs {
  const void *q, *k, *v;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;  // elements
  int B, Tq, Tk, H, Hkv, G, d, dv, causal;
  float scale, scale_log2;
  const int *kv_lens, *q_start;
  int start0;  // position of the first query where q_start is NULL
  const void* table;
  const int* buckets;
  int NB, R;
  const float* lam;
  void *out, *out2;
  float* lse;
  // forward, keys split over workgroups: partial results
  int splits;
  float *part_o, *part_l;  // [split][(b Tq + t) H + h][MAPS][dv], [split][..][MAPS] (base 2)
  // single-token kernel
  int kw, teams;  // teams (a wave per map) that share a problem: 1 or all of the workgroup's
  // backward
  const void* dout;
  int64_t do_sb, do_st, do_sh;
  void *dq, *dk, *dvo, *dtable;
  float* dlam;
  int Tp;             // padded rows of rows_lse / rows_d
  float* rows3;       // (split) [h][b][split][3][32 QW]: sum of dS, sums of P beyond -R and beyond R, of a row's part; two maps: [..][2][32 QW], sums of P W
  float *rows_lse, *rows_d;  // [(b H + h) MAPS + m][Tp]: -lse in base 2 (-inf for rows without keys), -D (two maps: 2^-PSH D)
  f32x2* sizes;       // (fp16) [m][b H + h][QW]: the largest |dO| and |D| of 32 rows, times the map's weight
  int QW, ND, DR;     // 32-query groups per head; floats per group in diag; relative positions -DR .. DR that they hold (and DIAG_PAD beyond)
  float* diag;        // [h][b][group][ND + 2]: sums of dS along diagonals (+ below -R, above R)
  float* dlam_part;   // [h][b][group]
  float* diag_part;   // [h][parts][ND + 2]
  int parts;
  // ahead of the keys' kernel, in its launch: workgroups that add the parts of dtable / dlam, and those of a split dQ
  int qsplits;        // parts of the queries' kernel
  float* part_q;
  int sum_blocks, join_blocks;
};

namespace mapattn {

typedef __bf16 bf16_t;
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x2v __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int DIAG_PAD = 96;  // a step of 64 keys x 32 queries that touches (-R, R) reaches less than that beyond

template <typename T>
struct Num;
template <>
struct Num<f16> {
  // P is written 2^PSH times larger where it is summed over queries: fp16 keeps full precision down to 2^-14 only, and the
  // weights of long rows are smaller
  static constexpr int PSH = 8;
  // dS, which is as large as the gradient that comes in, takes a power of two that follows the data
  static constexpr bool SCALED = true;
  __device__ static __forceinline__ uint32_t pack(float a, float b) {
    f32x2 t = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(t, f16x2v));  // v_cvt_pk_f16_f32: to nearest even
  }
  __device__ static __forceinline__ float lo(uint32_t u) { return (float)__builtin_bit_cast(f16x2v, u)[0]; }
  __device__ static __forceinline__ float hi(uint32_t u) { return (float)__builtin_bit_cast(f16x2v, u)[1]; }
  __device__ static __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Num<bf16_t> {
  static constexpr int PSH = 0;
  static constexpr bool SCALED = false;
  __device__ static __forceinline__ uint32_t pack(float a, float b) {
    f32x2 t = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(t, bf16x2));
  }
  __device__ static __forceinline__ float lo(uint32_t u) { return __uint_as_float(u << 16); }
  __device__ static __forceinline__ float hi(uint32_t u) { return __uint_as_float(u & 0xFFFF0000u); }
  __device__ static __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};

// ---- tiles in LDS --------------------------------------------------------------------------------------------------------
// A tile of ROWS rows of CH 16-byte chunks (CH % 4 == 0) lies row by row, its chunks permuted inside the row so that both reads
// meet 64 different banks: 16 lanes on 16 rows of one chunk column, and 32 lanes on 4 rows x 4 chunks.
template <int CH>
__device__ __forceinline__ constexpr int swz(int row) {
  return (CH % 16 == 0) ? (((row & 3) << 2) | ((row >> 2) & 3)) : (CH % 16 == 8) ? ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)) : ((row >> 2) & 3);
}
template <int CH>
__device__ __forceinline__ constexpr int chunk_at(int row, int c) {
  return (row * CH + (c ^ swz<CH>(row))) * 16;
}

__device__ __forceinline__ u32x4 lds16(const char* p) { return *(const u32x4*)p; }
__device__ __forceinline__ u32x2 lds_tr(const char* p) {
  typedef __attribute__((address_space(3))) s16x4* lp;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(__attribute__((address_space(3))) void*)p));
}
__device__ __forceinline__ u32x4 join(u32x2 a, u32x2 b) { return u32x4{a[0], a[1], b[0], b[1]}; }

// Both reads keep one offset per lane and derive the others: a chunk 32 or 64 bytes on is an exclusive or where the swizzle
// reaches those bits (CH a multiple of 8), an immediate otherwise.  The compiler holds the derived offsets in registers across
// the tiles; opaque() makes it derive them anew, where the accumulators need the registers.
__device__ __forceinline__ void opaque(int& x) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+v"(x));
#endif
}
// row-major reads: lane (l & 31, h) takes row l & 31, chunk 2 (STEP kk + m) + h (STEP = 2: a pair of waves, m = 0, 1, shares the row)
template <int CH, int STEP = 1>
struct RowRead {
  int base;
  __device__ __forceinline__ void init(int lane, int m = 0) { base = chunk_at<CH>(lane & 31, 2 * m + (lane >> 5)); }
  __device__ __forceinline__ u32x4 get(const char* tile, int sub, int kk) const {
    // where the swizzle stays below chunk bit 2 an odd step flips bit 1 and the rest adds
    const int off = CH % 8 == 0 ? base ^ (32 * STEP * kk) : STEP == 2 ? base + 64 * kk : (kk & 1 ? base ^ 32 : base) + 64 * (kk >> 1);
    return lds16(tile + off + sub * (32 * CH * 16));
  }
};
// transposed reads: the A operand with rows = channels 32 (nt0 + nt) .. + 31 and contraction over tile rows 16 kb .. + 15
template <int CH>
struct TrRead {
  int base;
  __device__ __forceinline__ void init(int lane, int nt0 = 0) {
    const int j = lane & 15, g = (lane >> 4) & 1, h = lane >> 5;
    base = chunk_at<CH>(4 * h + (j >> 2), 4 * nt0 + 2 * g + ((j & 3) >> 1)) + (j & 1) * 8;
  }
  __device__ __forceinline__ u32x4 get(const char* tile, int kb, int nt) const {
    const int off = CH % 8 == 0 ? base ^ (64 * nt) : base + 64 * nt;
    const char* p = tile + kb * (16 * CH * 16);
    return join(lds_tr(p + off), lds_tr(p + (off ^ 32) + 8 * CH * 16));  // rows 8 on: chunk bit 1 flips
  }
};

// one LDS-DMA instruction: 64 lanes x 16 B from base + voff[lane] to lds + 16 lane; lanes at or behind `bytes` write zeros
__device__ __forceinline__ void dma16(const void* base, uint32_t bytes, char* lds, uint32_t voff) {
  auto rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 16, voff, 0, 0, 0);
}
__device__ __forceinline__ void dma4(const void* base, uint32_t bytes, char* lds, uint32_t voff) {
  auto rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 4, voff, 0, 0, 0);
}
#define MAPATTN_WAIT_DMA() asm volatile("s_waitcnt vmcnt(0)" ::: "memory")

// a barrier for values that cross in LDS: waits for this wave's LDS operations alone.  (__syncthreads also waits for the global
// operations, and with them for the next tile's DMA.)
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// a tile's way into LDS: piece p (1 KiB = 64 chunks) is fetched by wave p % NW; rows behind the last one and channels behind d
// arrive as zeros (the buffer descriptor's bound), whatever lies there in memory
template <int CH, int ROWS, int NW>
struct TileDma {
  static constexpr int P = ROWS * CH / 64, NPW = (P + NW - 1) / NW;
  uint32_t off[NPW];
  uint32_t stride, width;
  __device__ __forceinline__ void init(int wave, int lane, int64_t stride_elems, int d) {
    stride = (uint32_t)(stride_elems * 2);
    width = (uint32_t)(d * 2);
#pragma unroll
    for (int i = 0; i < NPW; ++i) {
      const int s = 64 * (wave + NW * i) + lane;
      const int row = s / CH, c = (s - row * CH) ^ swz<CH>(row);
      off[i] = (c * 8 < d) ? (uint32_t)row * stride + (uint32_t)c * 16u : 0x80000000u;
    }
  }
  // rows [0, valid) of the tile exist (valid may be <= 0 or exceed ROWS); base and valid are wave-uniform
  __device__ __forceinline__ void issue(const void* base, int valid, char* lds, int wave) const {
    const int n = valid > ROWS ? ROWS : valid;
    const uint32_t bytes = n > 0 ? (uint32_t)(n - 1) * stride + width : 0u;
#pragma unroll
    for (int i = 0; i < NPW; ++i)
      if (P % NW == 0 || wave + NW * i < P) dma16(base, bytes, lds + (wave + NW * i) * 1024, off[i]);
  }
};

// B operand fragments of a row held in registers: chunk 2 (STEP kk + m) + h of the row, zeros where it does not exist
template <int KS, int STEP = 1>
__device__ __forceinline__ void load_row(u32x4 (&f)[KS], const void* row, bool exists, int h, int d, int m = 0) {
#pragma unroll
  for (int kk = 0; kk < KS; ++kk) {
    const int c = 2 * (STEP * kk + m) + h;
    f[kk] = u32x4{0u, 0u, 0u, 0u};
    if (exists && c * 8 < d) f[kk] = *(const u32x4*)((const char*)row + c * 16);
  }
}

__device__ __forceinline__ float xor32_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor32_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}
// row of register r in the lower half-wave; the upper one holds 4 rows on
__device__ __forceinline__ constexpr int acc_row(int r) { return 8 * (r >> 2) + (r & 3); }

__device__ __forceinline__ int seq_start(const MapAttnArgs& a, int b) {
  if (a.q_start == nullptr) return a.start0;
  const int n = a.q_start[b];
  return n < -(1 << 29) ? -(1 << 29) : (n > (1 << 29) ? (1 << 29) : n);
}
// keys that a query of the sequence may see; causal: none behind the last query (a cache's rows that nothing was written to yet)
__device__ __forceinline__ int seq_len(const MapAttnArgs& a, int b) {
  int n = a.kv_lens == nullptr ? a.Tk : min(a.kv_lens[b], a.Tk);
  if (a.causal) n = min(n, seq_start(a, b) + a.Tq);
  return max(n, 0);
}

template <typename T>
__device__ __forceinline__ float bias_at(const MapAttnArgs& a, int h, int rel) {
  const int x = rel < -a.R ? 0 : (rel > a.R ? 2 * a.R : rel + a.R);
  int n = a.buckets[x];
  n = n < 0 ? 0 : (n >= a.NB ? a.NB - 1 : n);
  return (float)((const T*)a.table)[(int64_t)h * a.NB + n] * LOG2E;
}
// near[x] = bias (base 2) of relative position x - R - E, x = 0 .. 2 (R + E): the saturated ends repeat over E entries, so that a
// tile that touches (-R, R) reads without clamping
template <typename T>
__device__ __forceinline__ void fill_near(const MapAttnArgs& a, int h, int E, float* near, int tid, int n) {
  for (int x = tid; x < 2 * (a.R + E) + 1; x += n) near[x] = bias_at<T>(a, h, x - a.R - E);
}

// the power of two that brings x into [2^(t - 1), 2^t); 0 where there is nothing to scale
__device__ __forceinline__ int power_to(float x, int t) {
  const int e = t - __builtin_amdgcn_frexp_expf(x);
  return x > 0.f && x < INFINITY ? (e < -100 ? -100 : (e > 100 ? 100 : e)) : 0;
}
__device__ __forceinline__ float power(int e) { return __builtin_amdgcn_ldexpf(1.0f, e); }

// block -> (slot among `slots` tiles, (batch, head) among nbh): all tiles of a (batch, head) on one XCD where the heads can be
// spread evenly over the 8 of them, so that K and V are fetched into one L2 only.  `falling`: the work falls with the slot
// (causal).  Then all heads' heaviest tiles come first, and where a CU holds two workgroups (TWO) and gets no more, the second ones
// in the opposite order: a heavy one beside a light one (2 x 2048, 16 heads of 64: forward 48 -> 40 us, dQ 72 -> 60).
template <bool TWO>
__device__ __forceinline__ void place(int lin, int slots, int nbh, bool falling, int& slot, int& bh) {
  const bool even = (nbh & 7) == 0;
  const int x = even ? lin & 7 : 0, step = even ? 8 : 1, nb = even ? nbh >> 3 : nbh;
  int y = even ? lin >> 3 : lin;
  if (falling) {
    const int n = slots * nb, cus = even ? 32 : 256;
    if (TWO && n > cus && n <= 2 * cus && y >= cus) y = n - 1 - (y - cus);
    slot = y / nb;
    bh = (y - slot * nb) * step + x;
  } else {
    bh = y / slots;
    slot = y - bh * slots;
    bh = bh * step + x;
  }
}

// (contraction steps over d, 32-channel tiles of V) of the instances; d, dv round up to the next one
#define MAPATTN_GEOS_1(X) X(2, 1) X(3, 2) X(4, 2) X(5, 3) X(8, 4) X(10, 5)
#define MAPATTN_GEOS_2(X) X(2, 2) X(3, 3) X(4, 4) X(5, 5) X(8, 8)

}  // namespace mapattn

// a launch's workgroups, checked against what one launch takes (2^31 of them, 2^32 threads); 0 and the error set otherwise
static inline unsigned mapattn_grid(const char* name, int64_t blocks, int threads) {
  if (blocks >= 1 && blocks < (1ll << 31) && blocks * threads < (1ll << 32)) return (unsigned)blocks;
  anip_set_error("%s: %lld workgroups of %d threads are too many for one launch", name, (long long)blocks, threads);
  return 0;
}

int mapattn_forward(const MapAttnArgs& a, int maps, int bf16, hipStream_t s);
int mapattn_token(const MapAttnArgs& a, int maps, int bf16, hipStream_t s);
int mapattn_combine(const MapAttnArgs& a, int maps, int bf16, hipStream_t s);
int mapattn_dq(const MapAttnArgs& a, int maps, int bf16, int nw, hipStream_t s);
int mapattn_dkv(const MapAttnArgs& a, int maps, int bf16, int nw, hipStream_t s);
