// Backward of the attention of mapattn.h.  With P_m the softmax maps, W = dO V^T (shared by both maps), D_m = rowsum(P_m W) =
// dO . o_m and w_1 = 1, w_2 = -lam:
//   dS_m = w_m P_m (W - D_m)   dQ_m = scale dS_m K_m   dK_m = scale dS_m^T Q_m   dV = (P_1 - lam P_2)^T dO
//   dlam = -sum P_2 W          dtable[bucket] = sum of dS over the pairs of the bucket
// Two kernels, one that owns queries (dQ, dlam, dtable's partial sums) and one that owns keys (dK, dV): each recomputes P and W
// (7 products instead of 5 at one map) and needs no atomics, so equal inputs give equal gradients.  P is recomputed from the row
// statistics of the forward; D from dO and the stored outputs for dQ, or from P and W where a row's keys all lie in one step, and from P
// and W of all its keys for dK.  dS and P are rounded to the inputs' type as operands of the
// matrix products (off by 2^-8 or 2^-11 of a term at most, averaged over a row); all sums are 32-bit.  In fp16 both are rounded as a
// power of two times themselves that follows the data, so that gradients of any size keep that precision.
#include "mapattn.h"

using namespace mapattn;

// Differential attention gives each map a wave of its own (both maps' accumulators would take all registers of one from d = 64
// on).  The pair shares W: each wave sums it over half of the channels and they exchange the halves through LDS; for dV they
// exchange P as well and each takes half of the channels' tiles.  Both values cross in 32 bits, with one barrier per tile of 32.

__device__ __forceinline__ void put16(float* x, const f32x16& v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) *(f32x4*)(x + i * 256) = f32x4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
}
__device__ __forceinline__ f32x16 get16(const float* x) {
  f32x16 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x4 t = *(const f32x4*)(x + i * 256);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[4 * i + e] = t[e];
  }
  return v;
}

// fragments of a wave's Q rows in LDS instead of registers, so that nothing goes to scratch: one map of 160 channels, and lone waves of 128
constexpr int dq_held(int maps, int ks, int ng) { return maps == 1 ? (ng == 4 ? (ks == 10 ? 6 : 0) : (ks == 8 ? 4 : 0)) : 0; }

// t + the squares of eight values
template <typename T>
__device__ __forceinline__ float squares(const u32x4& x, float t) {
#pragma unroll
  for (int i = 0; i < 4; ++i) t = fmaf(Num<T>::lo(x[i]), Num<T>::lo(x[i]), fmaf(Num<T>::hi(x[i]), Num<T>::hi(x[i]), t));
  return t;
}
// the largest of a wave's values (none below 0) in all lanes, in the vector ALU: quads, mirrored halves and rows of 16, then rows
template <int CTRL>
__device__ __forceinline__ float dpp_most(float v) {
  return fmaxf(v, __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), CTRL, 0xF, 0xF, true)));
}
__device__ __forceinline__ float wave_most(float v) {
  v = dpp_most<0x140>(dpp_most<0x141>(dpp_most<0x4E>(dpp_most<0xB1>(v))));
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return xor32_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

// ---- dQ: 32 queries per wave (pair), tiles of KT keys -----------------------------------------------------------------------
template <typename T, int MAPS, int KS, int NT, int KT, int NG, int NS>
__global__ __launch_bounds__(64 * NG * MAPS, (NG == 4 || (MAPS == 1 && KS <= 8) ? 2 : 1)) void mapattn_dq_kernel(const MapAttnArgs a) {
  constexpr bool BIAS = MAPS == 1, SCALED = Num<T>::SCALED;
  constexpr int NW = NG * MAPS, BQ = 32 * NG, DT = (KS + 1) / 2, KSV = MAPS == 1 ? KS : NT;  // KSV: steps over this wave's share of dv
  constexpr int KCH = 4 * DT, VCH = 4 * NT;
  constexpr int K_BYTES = KT * KCH * 16, V_BYTES = KT * VCH * 16, STAGE = MAPS * K_BYTES + V_BYTES;
  constexpr int E = BQ + KT;
  static_assert(MAPS == 1 || KT == 32, "the pair's exchange has one slot per tile");
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  constexpr int QL = dq_held(MAPS, KS, NG);
  float* near = (float*)(smem + 2 * STAGE + NW * QL * 1024);  // (one map)

  const int tid = threadIdx.x, lane = tid & 63, ql = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave / MAPS, m = wave % MAPS;
  float* mine = (float*)(smem + 2 * STAGE) + wave * 1024 + lane * 4;         // (two maps) 16 values of each lane
  float* theirs = (float*)(smem + 2 * STAGE) + (wave ^ 1) * 1024 + lane * 4;
  const int nqb = a.Tp / BQ;
  int qb, bh;
  place<MAPS == 1>(blockIdx.x, nqb * a.splits, a.B * a.H, a.causal, qb, bh);
  const int split = qb % a.splits;
  qb = nqb - 1 - qb / a.splits;
  const int b = bh / a.H, head = bh - b * a.H, kvh = head / a.G;
  const int len = seq_len(a, b), start = seq_start(a, b);
  const int q0 = qb * BQ + grp * 32, qi = q0 + ql, pw = start + q0;
  const bool valid = qi < a.Tq;
  const int lim = a.causal ? min(len - 1, start + qi) : len - 1;
  int kend = len;
  if (a.causal) kend = min(kend, start + min(qb * BQ + BQ, a.Tq));
  if (qb * BQ >= a.Tq) kend = 0;  // padding rows: only their row statistics are written
  const int nt_keys = kend > 0 ? (kend + KT - 1) / KT : 0;
  const int nt0 = (int)((int64_t)nt_keys * split / a.splits), nt_all = (int)((int64_t)nt_keys * (split + 1) / a.splits);

  const float lam = MAPS == 2 ? a.lam[head] : 0.f;
  u32x4 qf[KS], df[KSV];
  const char* drow = (const char*)a.dout + 2 * (b * a.do_sb + (int64_t)qi * a.do_st + (int64_t)head * a.do_sh);
  load_row<KS>(qf, (const char*)a.q + 2 * (b * a.q_sb + (int64_t)qi * a.q_st + (int64_t)(head * MAPS + m) * a.q_sh), valid, h, a.d);
  load_row<KSV, MAPS>(df, drow, valid, h, a.dv, m);
  char* qlds = smem + 2 * STAGE + wave * (QL * 1024) + lane * 16;  // the last QL fragments of the Q rows
#pragma unroll
  for (int i = 0; i < QL; ++i) *(u32x4*)(qlds + i * 1024) = qf[KS - QL + i];

  // the split that has the first keys (the first one where there are none) leaves the rows' statistics for the keys' kernel
  const bool first = nt_keys > 0 ? nt0 == 0 && nt_all > 0 : split == 0;
  const int64_t rows_at = ((int64_t)bh * MAPS + m) * a.Tp + qi;

  // ---- row statistics: D_m = dO . o_m (o_1 = o + lam o_2), -lse in base 2 -------------------------------------------------
  float nl, D, n2 = 0.f;  // (n2: |dO|^2)
  {
    const int64_t orow = (((int64_t)b * a.Tq + qi) * a.H + head) * a.dv * 2;
    auto dot = [&](const void* o) {
      float t = 0.f;
      n2 = 0.f;
#pragma unroll 4
      for (int c = h; c < a.dv / 8; c += 2) {
        u32x4 x = {0u, 0u, 0u, 0u}, y = x;
        if (valid) {
          x = *(const u32x4*)(drow + c * 16);
          y = *(const u32x4*)((const char*)o + orow + c * 16);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) t = fmaf(Num<T>::lo(x[i]), Num<T>::lo(y[i]), fmaf(Num<T>::hi(x[i]), Num<T>::hi(y[i]), t));
        if (SCALED) n2 = squares<T>(x, n2);
      }
      return xor32_sum(t);
    };
    if (MAPS == 1) {
      D = dot(a.out);
    } else {
      D = dot(a.out2);
      if (m == 0) D = fmaf(lam, D, dot(a.out));
    }
    const float l = valid ? a.lse[((int64_t)bh * MAPS + m) * a.Tq + qi] * LOG2E : -INFINITY;
    nl = l == -INFINITY ? -INFINITY : -l;  // rows without keys: P = 2^-inf = 0
    if (h == 0 && first) a.rows_lse[rows_at] = nl + Num<T>::PSH;
  }

  // dS = wf P W + wd P, in fp16 2^fe times that.  dS is as large as P |dO| |V|, and fp16 keeps its precision from 2^-14 to 2^16: 2^fe
  // brings the largest |dO| of the wave's rows to 2^8.  That is room for weights of 2^-20 beside values of about 1, and for values of up
  // to about 50.  If larger ones overflow it, the walk is done again with room for 128 times larger ones, and for any (a maximum of dS in
  // every step instead: dQ at 2 x 2048, 16 / 4 heads of 64, 70 us against 65).
  const float w0 = MAPS == 2 && m == 1 ? -lam : 1.f;
  int fe = 0, again = 0;
  bool finite = true;  // (rows of NaN or infinities keep them to themselves)
  if (SCALED) {
    n2 = xor32_sum(n2);
    finite = fabsf(n2) < INFINITY && fabsf(D) < INFINITY && nl == nl;
    const float most = __builtin_amdgcn_sqrtf(wave_most(finite ? n2 : 0.f)) * fabsf(w0), mostD = wave_most(finite ? fabsf(D) : 0.f) * fabsf(w0);
    fe = __builtin_amdgcn_readfirstlane(power_to(most, 8));
    if (first && lane == 0 && q0 < a.Tq) a.sizes[((int64_t)m * a.B * a.H + bh) * a.QW + q0 / 32] = f32x2{most, mostD};
  }

  float* diag = nullptr;
  if (BIAS && q0 < a.Tq) {
    diag = a.diag + ((((int64_t)head * a.B + b) * a.QW + q0 / 32) * a.splits + split) * (a.ND + 2);
    for (int x = lane; x < a.ND + 2; x += 64) diag[x] = 0.f;  // (complete before the first tile's wait; later stores are this wave's own)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }

  const char* kb[MAPS];
#pragma unroll
  for (int i = 0; i < MAPS; ++i) kb[i] = (const char*)a.k + 2 * (b * a.k_sb + (int64_t)(kvh * MAPS + i) * a.k_sh);
  const char* vb = (const char*)a.v + 2 * (b * a.v_sb + (int64_t)kvh * a.v_sh);
  TileDma<KCH, KT, NW> kd;
  TileDma<VCH, KT, NW> vd;
  kd.init(wave, lane, a.k_st, a.d);
  vd.init(wave, lane, a.v_st, a.dv);
  auto issue = [&](int t) {
    char* st = smem + (t & 1) * STAGE;
    const int64_t row = (int64_t)t * KT;
    const int n = len - t * KT;
#pragma unroll
    for (int i = 0; i < MAPS; ++i) kd.issue(kb[i] + row * a.k_st * 2, n, st + i * K_BYTES, wave);
    vd.issue(vb + row * a.v_st * 2, n, st + MAPS * K_BYTES, wave);
  };
  RowRead<KCH> kr;
  RowRead<VCH, MAPS> vr;
  TrRead<KCH> kt;
  kr.init(lane);
  vr.init(lane, MAPS == 2 ? m : 0);
  kt.init(lane);

  f32x16 dq[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) dq[dt] = zero16();
  float far_lo = 0.f, far_hi = 0.f, sum_lo = 0.f, sum_hi = 0.f, p_lo = 0.f, p_hi = 0.f, sum_near = 0.f, pw_sum = 0.f;
  float dpos = 0.f, dneg = 0.f;  // diagonals rel = base + ql and base - 32 + ql of the current 32 keys, base = k0 - pw
  int next_base = 0;
  bool open = false;
  if (BIAS) {
    fill_near<T>(a, head, E, near, tid, 64 * NW);
    far_lo = bias_at<T>(a, head, -a.R);
    far_hi = bias_at<T>(a, head, a.R);
  }
  // All keys of these rows in one step: D from P and W themselves.  Rounded outputs leave W - D of rows with few keys nothing but
  // their rounding (one key: dS is 0; a sequence of one key in a padded batch gave its 898 rows a dQ of 5e-3 of the other one's)
  const int whole = (a.causal ? min(len, start + q0 + 32) : len) <= 32 * NS ? 0 : -1;

  float wf = power(fe) * w0, wd = -wf * D;
  if (nt0 < nt_all) issue(nt0);
  for (int t = nt0;; ++t) {
    if (t >= nt_all) {
      if (!SCALED || again == 2 || nt0 >= nt_all) break;
      // an infinity among the rounded dS leaves one, or NaN, in dQ
      float bad[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) bad[r & 3] = fmaf(dq[dt][r], 0.f, bad[r & 3]);
      int* over = (int*)smem;
      const int mine_over = __any(finite && (bad[0] + bad[1]) + (bad[2] + bad[3]) != 0.f);
      lds_barrier();  // all tiles read
      if (lane == 0) over[wave] = mine_over;
      lds_barrier();
      int any = 0;
#pragma unroll
      for (int i = 0; i < NW; ++i) any |= over[i];
      if (!__builtin_amdgcn_readfirstlane(any)) break;
      lds_barrier();  // all flags read
      ++again;
      if (mine_over) fe -= 7;  // |W| and |D| are at most |dO| 2^16 sqrt(256): with |dO| at 2^-6, the second time, dS stays below 2^15
      wf = power(fe) * w0, wd = -wf * D;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) dq[dt] = zero16();
      sum_lo = sum_hi = p_lo = p_hi = sum_near = pw_sum = dpos = dneg = 0.f;
      open = false;
      t = nt0;
      issue(t);
    }
    MAPATTN_WAIT_DMA();
    __syncthreads();
    if (t + 1 < nt_all) issue(t + 1);
    const char* st = smem + (t & 1) * STAGE;
    const int kt0 = t * KT;
    const bool skip = a.causal && kt0 > pw + 31;
    if (MAPS == 1 && skip) continue;
#pragma unroll
    for (int sub = 0; sub < KT / 32; sub += NS) {
      const int k0 = kt0 + 32 * sub;
      f32x16 s[NS], w[NS];
#pragma unroll
      for (int i = 0; i < NS; ++i) s[i] = w[i] = zero16();
      if (MAPS == 1 || !skip) {
#pragma unroll
        for (int kk = 0; kk < KSV; ++kk)
#pragma unroll
          for (int i = 0; i < NS; ++i) w[i] = Num<T>::mfma(vr.get(st + MAPS * K_BYTES, sub + i, kk), df[kk], w[i]);
        if (MAPS == 2) put16(mine, w[0]);
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
#pragma unroll
          for (int i = 0; i < NS; ++i)
            s[i] = Num<T>::mfma(kr.get(st + m * K_BYTES, sub + i, kk), kk < KS - QL ? qf[kk] : lds16(qlds + (kk - (KS - QL)) * 1024), s[i]);
      }
      float mul = a.scale_log2, add = 0.f;
      int zone = 0;  // -1, 1: all of these pairs beyond the bias's reach
      if (BIAS) {
        if (k0 + 32 * NS - 1 - pw <= -a.R) { add = far_lo; zone = -1; }
        else if (k0 - (pw + 31) >= a.R) { add = far_hi; zone = 1; }
        else {
          const float* nb = near + (k0 + 4 * h - (pw + ql) + a.R + E);
#pragma unroll
          for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[i][r] = fmaf(s[i][r], mul, nb[32 * i + acc_row(r)]);
          mul = 1.f;
        }
      }
      if (k0 + 32 * NS - 1 >= len || (a.causal && k0 + 32 * NS - 1 > pw)) {
        const int dl = lim - k0 - 4 * h;
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[i][r] = 32 * i + acc_row(r) > dl ? -INFINITY : s[i][r];
      }
      const float c = add + nl;
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[i][r] = __builtin_amdgcn_exp2f(fmaf(s[i][r], mul, c));
      if (MAPS == 2) {
        lds_barrier();  // the other half of W is there (the next tile's comes behind its own first barrier)
        if (skip) continue;
        const f32x16 w2 = get16(theirs);
#pragma unroll
        for (int r = 0; r < 16; ++r) w[0][r] += w2[r];
#pragma unroll
        for (int r = 0; r < 16; ++r) pw_sum = fmaf(s[0][r], w[0][r], pw_sum);
      }
      if (k0 == whole) {
        float pw1 = 0.f, p1 = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            pw1 = fmaf(s[i][r], w[i][r], pw1);
            p1 += s[i][r];
          }
        pw1 = xor32_sum(pw1), p1 = xor32_sum(p1);
        D = p1 > 0.f ? pw1 / p1 : 0.f;
        wd = -wf * D;
      }
      auto total = [&] {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) t += s[i][r];
        return t;
      };
      if (BIAS) {
        if (zone != 0) {
          const float t = total();
          if (zone < 0) p_lo += t;
          else p_hi += t;
        } else {  // those of the pairs that are beyond reach
          const int rel = k0 + 4 * h - (pw + ql), lo = -a.R - rel, hi = (a.R > 0 ? a.R : 1) - rel;
          if (k0 - (pw + 31) <= -a.R)
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
              for (int r = 0; r < 16; ++r) p_lo += 32 * i + acc_row(r) <= lo ? s[i][r] : 0.f;
          if (k0 + 32 * NS - 1 - pw >= a.R)
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
              for (int r = 0; r < 16; ++r) p_hi += 32 * i + acc_row(r) >= hi ? s[i][r] : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[i][r] *= MAPS == 1 && !SCALED ? w[i][r] - D : fmaf(w[i][r], wf, wd);
      if (BIAS) {
        const float t = total();
        if (zone != 0) {
          if (zone < 0) sum_lo += t;
          else sum_hi += t;
        } else {
          sum_near += t;
          // value of (key k0 + ko, query ql) belongs to diagonal ko - ql: lane x takes it from lane (ko - x) mod 32 of its half
          open = true;
          next_base = k0 + 32 * NS - pw;
#pragma unroll
          for (int i = 0; i < NS; ++i) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int ko = acc_row(r) + 4 * h;
              const float v = __uint_as_float(__builtin_amdgcn_ds_bpermute((((ko - ql) & 31) | (lane & 32)) << 2, __float_as_uint(s[i][r])));
              dpos += ql <= ko ? v : 0.f;
              dneg += ql <= ko ? 0.f : v;
            }
            const float done = xor32_sum(dneg);  // no later key reaches these 32 diagonals
            if (diag && h == 0) diag[k0 + 32 * i - pw - 32 + ql + a.DR + DIAG_PAD] = __builtin_amdgcn_ldexpf(done, -fe);
            dneg = dpos;
            dpos = 0.f;
          }
        }
      }
#pragma unroll
      for (int kb2 = 0; kb2 < 2 * NS; ++kb2) {
        const f32x16& x = s[kb2 >> 1];
        u32x4 p;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = Num<T>::pack(x[8 * (kb2 & 1) + 2 * i], x[8 * (kb2 & 1) + 2 * i + 1]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) dq[dt] = Num<T>::mfma(kt.get(st + m * K_BYTES, 2 * sub + kb2, dt), p, dq[dt]);
      }
    }
  }

  // D for the keys' kernel from P and W themselves, in all rows: what D was off by is left over in the row's dS, whose sum is 0; two maps
  // add P W.  Where few keys hold a row's weight W - D is small, and mostly what the rounding of the outputs made of D (bf16, queries of
  // 8 times 1: dk 4.5e-3 off with D from the outputs, 2.4e-3 with this, whatever the queries' size; dQ, whose walk it ends, keeps 4.9e-3).
  // Costs nothing where the walk is whole, and a launch of 3 us where it is split.
  const float fi = power(-fe);
  sum_lo *= fi, sum_hi *= fi, sum_near *= fi;
  const float left = xor32_sum(MAPS == 1 ? sum_lo + sum_hi + sum_near : pw_sum);
  if (h == 0) {
    if (a.splits == 1) a.rows_d[rows_at] = MAPS == 1 ? -(D + left) : left * (1.0f / (1 << Num<T>::PSH));
    else if (first) a.rows_d[rows_at] = MAPS == 1 ? -D : 0.f;
  }
  // parts of rows: what is left over and the sums of P beyond -R and beyond R; two maps: the sums of P W
  float* part = a.rows3 + ((((int64_t)head * a.B + b) * a.splits + split) * (MAPS == 1 ? 3 : 2) + m) * a.QW * 32 + q0 + ql;
  if (a.splits > 1 && h == 0 && q0 < a.Tq) part[0] = left;
  if (BIAS && diag) {
    const float done = xor32_sum(dneg) * fi;
    if (open && h == 0) diag[next_base - 32 + ql + a.DR + DIAG_PAD] = done;
    // What D is off by (the rounded outputs, the forward's rounded P) is what a row's dS leave over from their sum of 0.  It meets
    // a bucket with the row's P in it: with most of it, beyond the bias's reach, where it is taken out; with a few keys' up to
    // there, where it is small beside the roundings.  dtable in bf16, 2 heads, 2 x 3954: 2e-2 off with it, less than 4e-3 without;
    // its two sums over P and dS cost 3 to 4 % of the backward (2 x 2048, 16 / 4 heads of 64, bf16: 120 us without, 126 with).
    if (a.splits == 1) {
      sum_lo = fmaf(-left, p_lo, sum_lo);
      sum_hi = fmaf(-left, p_hi, sum_hi);
    } else {  // (sum_table knows the whole row)
      const float pl = xor32_sum(p_lo), ph = xor32_sum(p_hi);
      if (h == 0) {
        part[a.QW * 32] = pl;
        part[a.QW * 64] = ph;
      }
    }
    const float lo = wave_sum(sum_lo), hi = wave_sum(sum_hi);
    if (lane == 0) {
      diag[a.ND] = lo;
      diag[a.ND + 1] = hi;
    }
  }
  if (MAPS == 2 && m == 1 && q0 < a.Tq) {
    const float t = wave_sum(pw_sum);
    if (lane == 0) a.dlam_part[(((int64_t)head * a.B + b) * a.QW + q0 / 32) * a.splits + split] = -t;
  }
  if (!valid) return;
  const float scale = a.scale * fi;
  if (a.splits > 1) {
    float* pp = a.part_q + (((int64_t)split * a.B * a.Tq + (int64_t)b * a.Tq + qi) * a.H * MAPS + head * MAPS + m) * a.d;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        const int c0 = dt * 32 + rq * 8 + h * 4;
        const f32x16& x = dq[dt];
        if (c0 < a.d) *(f32x4*)(pp + c0) = f32x4{x[4 * rq] * scale, x[4 * rq + 1] * scale, x[4 * rq + 2] * scale, x[4 * rq + 3] * scale};
      }
    return;
  }
  char* op = (char*)a.dq + ((((int64_t)b * a.Tq + qi) * a.H + head) * MAPS + m) * a.d * 2;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      const int c0 = dt * 32 + rq * 8 + h * 4;
      const f32x16& x = dq[dt];
      if (c0 < a.d)
        *(u32x2*)(op + c0 * 2) = u32x2{Num<T>::pack(x[4 * rq] * scale, x[4 * rq + 1] * scale), Num<T>::pack(x[4 * rq + 2] * scale, x[4 * rq + 3] * scale)};
    }
}

// ---- sums of parts, in a fixed order ----------------------------------------------------------------------------------------
// The queries' kernel leaves sums for each 32 queries (dtable's diagonals, dlam) and, split, dQ in parts.  They are added by the
// first workgroups of the keys' launch, beside its own work; dtable of many groups by kernels of its own.

// four channels of a gradient from the 32-bit parts of a split walk, `n` values apart
__device__ __forceinline__ f32x4 add_parts(const float* p, int parts, int64_t n) {
  f32x4 t = *(const f32x4*)p;
#pragma unroll 4
  for (int s = 1; s < parts; ++s) t += *(const f32x4*)(p + s * n);
  return t;
}
template <typename T>
__device__ __forceinline__ void join_dq(const MapAttnArgs& a, int block) {
  const int64_t n = (int64_t)a.B * a.Tq * a.H * a.dv, i = ((int64_t)block * blockDim.x + threadIdx.x) * 4;
  if (i >= n) return;
  const f32x4 t = add_parts(a.part_q + i, a.qsplits, n);
  *(u32x2*)((char*)a.dq + i * 2) = u32x2{Num<T>::pack(t[0], t[1]), Num<T>::pack(t[2], t[3])};
}
// a head's bucket sums from `parts` rows of diagonals: each lane adds the rows of a slot, then lane c takes the 64 slots of the wave
// that belong to bucket c, one after the other, from the other lanes' registers.  Bound by the loads' latency in short launches: the
// rows of 16 parts, and the next slots' first 16, are on their way at once (2 heads, 3 x 19: 12 us of the keys' launch,
// 43 with a wave for each bucket that walks over the slots in LDS)
template <typename T>
__device__ __forceinline__ void sum_table(const MapAttnArgs& a, int head, const float* rows, int parts, float* sums) {
  const int n = a.ND + 2, lane = threadIdx.x & 63;
  const float* p = rows + (int64_t)head * parts * n;
  auto load = [&](int x, int i0, float (&t)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) t[i] = i0 + i < parts && x < n ? p[(int64_t)(i0 + i) * n + x] : 0.f;
  };
  // slot x < ND: relative position x - DR - DIAG_PAD, beyond +-R as +-R; the last two: all pairs beyond -R, and beyond R
  auto bucket = [&](int x) {
    int r = x - DIAG_PAD + a.R - a.DR;
    r = x == a.ND || r < 0 ? 0 : (x > a.ND || r > 2 * a.R ? 2 * a.R : r);
    const int bx = x < n ? a.buckets[r] : -1;
    return x >= n ? -1 : (bx < 0 ? 0 : (bx >= a.NB ? a.NB - 1 : bx));
  };
  // split rows: what the far sums have to lose (see the queries' kernel)
  float off[2] = {0.f, 0.f};
  if (a.qsplits > 1) {
    const int per = a.QW * 32;
    for (int i = threadIdx.x; i < a.B * per; i += blockDim.x) {
      const int b = i / per;
      const float* r3 = a.rows3 + ((int64_t)head * a.B + b) * a.qsplits * 3 * per + (i - b * per);
      float e = 0.f, lo = 0.f, hi = 0.f;
#pragma unroll 4
      for (int s = 0; s < a.qsplits; ++s, r3 += 3 * per) {
        e += r3[0];
        lo += r3[per];
        hi += r3[2 * per];
      }
      off[0] = fmaf(e, lo, off[0]);
      off[1] = fmaf(e, hi, off[1]);
    }
  }
  for (int c0 = 0; c0 < a.NB; c0 += 64) {
    float acc = 0.f, t[16];
    int x = threadIdx.x, bx = bucket(x);
    load(x, 0, t);
    while (x - lane < n) {
      const int xn = x + blockDim.x, bn = bucket(xn);
      float tn[16], v = 0.f;
      load(xn, 0, tn);
#pragma unroll
      for (int i = 0; i < 16; ++i) v += t[i];
      for (int i0 = 16; i0 < parts; i0 += 16) {
        load(x, i0, t);
#pragma unroll
        for (int i = 0; i < 16; ++i) v += t[i];
      }
#pragma unroll
      for (int i = 0; i < 64; ++i) {
        const float vi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), i));
        acc += __builtin_amdgcn_readlane(bx, i) == c0 + lane ? vi : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) t[i] = tn[i];
      x = xn, bx = bn;
    }
    if (a.qsplits > 1) {
      const int ends[2] = {bucket(a.ND), bucket(a.ND + 1)};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float t = wave_sum(off[i]);
        if (ends[i] == c0 + lane) acc -= t;
      }
    }
    __syncthreads();
    sums[threadIdx.x] = acc;
    __syncthreads();
    if ((int)threadIdx.x < min(64, a.NB - c0)) {
      float s = 0.f;
      for (int w = 0; w < (int)blockDim.x; w += 64) s += sums[w + lane];
      ((T*)a.dtable)[(int64_t)head * a.NB + c0 + lane] = (T)s;
    }
  }
}
__device__ __forceinline__ void sum_lam(const MapAttnArgs& a, int head, float* sums) {
  const int64_t rows = (int64_t)a.B * a.QW * a.qsplits;
  const float* p = a.dlam_part + head * rows;
  float t = 0.f;
  for (int64_t r = threadIdx.x; r < rows; r += blockDim.x) t += p[r];
  t = wave_sum(t);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    t = 0.f;
    for (int w = 0; w < (int)blockDim.x >> 6; ++w) t += sums[w];
    a.dlam[head] = t;
  }
}

// fragments of a wave's K rows in LDS instead of registers.  Two maps, the widest heads: 477 us against 503 at 2 x 4096 causal, 8
// heads of 128 + 128, where 18 registers went to scratch.  One map of up to 128 channels: with 7 of 8 there (and 32 queries a step)
// two waves share a SIMD where there was one: 168 -> 139 us with 6 at 2 x 2048 causal, 16 heads of 128, 86 -> 46 at 16 x 500 (4 of 8: 12
// registers in scratch, 170 us; all 8: 147; in fp16 6 leave 36 bytes there, 7 none, at the same time).
constexpr int dkv_held(int maps, int ks, int ng) { return maps == 2 ? (ks >= 8 ? 3 : 0) : (ks == 8 && ng == 4 ? 7 : 0); }
// two waves of the kernel on a SIMD
constexpr bool dkv_two(int maps, int ks, int ng) { return (maps == 1 && ks <= 5) || (ng == 4 && (maps == 2 || ks <= 8)); }

// ---- dK, dV: 32 keys per wave (pair; K and V rows in registers), tiles of QT queries of every head that shares them ------------
template <typename T, int MAPS, int KS, int NT, int QT, int NG, int NS>
__global__ __launch_bounds__(64 * NG * MAPS, dkv_two(MAPS, KS, NG) ? 2 : 1) void mapattn_dkv_kernel(const MapAttnArgs a) {
  constexpr bool BIAS = MAPS == 1, SCALED = Num<T>::SCALED;
  constexpr int NW = NG * MAPS, BK = 32 * NG, DT = (KS + 1) / 2;
  constexpr int KSV = MAPS == 1 ? KS : NT;               // steps over this wave's share of dv in W
  constexpr int VT = MAPS == 1 ? NT : (NT + 1) / 2;      // 32-channel tiles of this wave's share of dV
  constexpr int QCH = 4 * DT, OCH = 4 * NT;
  constexpr int Q_BYTES = QT * QCH * 16, O_BYTES = QT * OCH * 16, R_BYTES = 256;
  constexpr int STAGE = MAPS * Q_BYTES + O_BYTES + 2 * MAPS * R_BYTES;
  constexpr int E = BK + QT;
  static_assert(MAPS == 1 || QT == 32, "the pair's exchange has one slot per tile");
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  float* near = (float*)(smem + 2 * STAGE + NW * dkv_held(MAPS, KS, NG) * 1024);  // (one map)

  const int tid = threadIdx.x, lane = tid & 63, kl = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave / MAPS, m = wave % MAPS;
  float* mine = (float*)(smem + 2 * STAGE) + wave * 2048 + lane * 4;         // (two maps) 16 values of W, 16 of P of each lane
  float* theirs = (float*)(smem + 2 * STAGE) + (wave ^ 1) * 2048 + lane * 4;
  const int nkb = (a.Tk + BK - 1) / BK;
  int lin = blockIdx.x;
  if (lin < a.sum_blocks) {
    if (MAPS == 1) sum_table<T>(a, lin, a.diag, a.B * a.QW * a.qsplits, (float*)smem);
    else sum_lam(a, lin, (float*)smem);
    return;
  }
  lin -= a.sum_blocks;
  if (lin < a.join_blocks) return join_dq<T>(a, lin);
  lin -= a.join_blocks;
  int kblk, bk;
  // causal: the first keys meet the most queries (128 channels, the second half reversed: 53 us against 46 at 16 x 500, 143 against 139)
  place<MAPS == 1 && (KS <= 5)>(lin, nkb * a.splits, a.B * a.Hkv, a.causal, kblk, bk);
  const int split = kblk % a.splits;
  kblk /= a.splits;
  const int b = bk / a.Hkv, kvh = bk - b * a.Hkv;
  const int len = seq_len(a, b), start = seq_start(a, b);
  const int kw0 = kblk * BK + grp * 32, key = kw0 + kl;
  const bool valid = key < len;

  // the last KL fragments of the K rows wait in LDS where registers are short; in scratch, their loads would wait for the DMA
  constexpr int KL = dkv_held(MAPS, KS, NG);
  char* klds = smem + 2 * STAGE + (MAPS == 2 ? NW * 8192 : 0) + wave * (KL * 1024) + lane * 16;
  u32x4 kf[KS], vf[KSV];
  load_row<KS>(kf, (const char*)a.k + 2 * (b * a.k_sb + (int64_t)key * a.k_st + (int64_t)(kvh * MAPS + m) * a.k_sh), valid, h, a.d);
  load_row<KSV, MAPS>(vf, (const char*)a.v + 2 * (b * a.v_sb + (int64_t)key * a.v_st + (int64_t)kvh * a.v_sh), valid, h, a.dv, m);

#pragma unroll
  for (int i = 0; i < KL; ++i) *(u32x4*)(klds + i * 1024) = kf[KS - KL + i];

  // ---- query tiles that meet these keys -----------------------------------------------------------------------------------
  const int nqt = (a.Tq + QT - 1) / QT;
  int tq0 = 0;
  if (a.causal) {
    const int first = kblk * BK - start;  // first query that sees the workgroup's first key
    tq0 = first <= 0 ? 0 : min(first / QT, nqt);
  }
  const int per = kblk * BK < len ? nqt - tq0 : 0, all = per * a.G;
  const int it0 = (int)((int64_t)all * split / a.splits), total = (int)((int64_t)all * (split + 1) / a.splits);

  TileDma<QCH, QT, NW> qd;
  TileDma<OCH, QT, NW> od;
  qd.init(wave, lane, a.q_st, a.d);
  od.init(wave, lane, a.do_st, a.dv);
  auto issue = [&](int it) {
    const int g = it / per, t = tq0 + it - g * per, head = kvh * a.G + g;
    char* st = smem + (it & 1) * STAGE;
    const int64_t row = (int64_t)t * QT;
    const int n = a.Tq - t * QT;
#pragma unroll
    for (int i = 0; i < MAPS; ++i)
      qd.issue((const char*)a.q + 2 * (b * a.q_sb + row * a.q_st + (int64_t)(head * MAPS + i) * a.q_sh), n, st + i * Q_BYTES, wave);
    od.issue((const char*)a.dout + 2 * (b * a.do_sb + row * a.do_st + (int64_t)head * a.do_sh), n, st + MAPS * Q_BYTES, wave);
    char* rt = st + MAPS * Q_BYTES + O_BYTES;
#pragma unroll
    for (int i = 0; i < 2 * MAPS; ++i)
      if (i % NW == wave) {
        const float* src = (i < MAPS ? a.rows_lse : a.rows_d) + ((int64_t)(b * a.H + head) * MAPS + i % MAPS) * a.Tp + row;
        dma4(src, QT * 4, rt + i * R_BYTES, lane * 4);
      }
  };
  RowRead<QCH> qr;
  RowRead<OCH, MAPS> orr;
  TrRead<QCH> qt;
  TrRead<OCH> ot;
  qr.init(lane);
  orr.init(lane, MAPS == 2 ? m : 0);
  qt.init(lane);
  ot.init(lane, m * VT);

  f32x16 dk[DT], dv[VT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) dk[dt] = zero16();
#pragma unroll
  for (int nt = 0; nt < VT; ++nt) dv[nt] = zero16();
  float far_lo = 0.f, far_hi = 0.f, lam = 0.f;
  constexpr float PF = 1.0f / (1 << Num<T>::PSH);
  if (it0 < total) issue(it0);
  // (fp16) dS is rounded as 2^fe of itself: below 2^14 for all queries and the wave's keys, since |W| <= |dO| |V|, and as large as that allows
  f32x2 most = {0.f, 0.f};
  if (SCALED) {
    const f32x2* z = a.sizes + ((int64_t)m * a.B * a.H + (int64_t)b * a.H + kvh * a.G) * a.QW;
    for (int i = lane; i < a.G * a.QW; i += 64) {
      const f32x2 x = z[i];
      most[0] = fmaxf(most[0], x[0]), most[1] = fmaxf(most[1], x[1]);
    }
  }
  int fe = 0;
  if (SCALED) {
    float v2 = 0.f;
#pragma unroll
    for (int kk = 0; kk < KSV; ++kk) v2 = squares<T>(vf[kk], v2);
    if (MAPS == 2) {  // the other half of the channels
      mine[0] = v2;
      lds_barrier();
      v2 += theirs[0];
    }
    fe = __builtin_amdgcn_readfirstlane(power_to(fmaf(wave_most(most[0]), __builtin_amdgcn_sqrtf(wave_most(xor32_sum(v2))), wave_most(most[1])), 14));
  }
  const float fs = power(fe);
  // (fp16, two maps) what meets dO in dV is up to 2^PSH (1 + |lam|) large: from |lam| = 127 on it is rounded as a part of itself
  int pe = 0;
  if (SCALED && MAPS == 2) {
    float l = 0.f;
    for (int g = 0; g < a.G; ++g) l = fmaxf(l, fabsf(a.lam[kvh * a.G + g]));
    pe = min(0, __builtin_amdgcn_readfirstlane(power_to(1.0f + l, 15 - Num<T>::PSH)));
  }
  const float ps = power(pe);

  for (int it = it0; it < total; ++it) {
    const int g = it / per, t = tq0 + it - g * per;
    if (it == it0 || it - g * per == 0) {  // the next head: its bias, its lam
      const int head = kvh * a.G + g;
      if (BIAS) {
        if (it > it0) __syncthreads();  // the head before is read to the end
        fill_near<T>(a, head, E, near, tid, 64 * NW);
        far_lo = bias_at<T>(a, head, -a.R);
        far_hi = bias_at<T>(a, head, a.R);
      } else {
        lam = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(a.lam[head])));
      }
    }
    MAPATTN_WAIT_DMA();
    __syncthreads();
    if (it + 1 < total) issue(it + 1);
    if (MAPS * NT >= 16) {
      opaque(qr.base);
      opaque(orr.base);
      opaque(qt.base);
      opaque(ot.base);
    }
    const char* st = smem + (it & 1) * STAGE;
    const char* rt = st + MAPS * Q_BYTES + O_BYTES;
    const int pt = start + t * QT;
    const bool skip = a.causal && pt + QT - 1 < kw0;  // no query of the tile sees this wave's keys
    if (MAPS == 1 && skip) continue;
#pragma unroll
    for (int sub = 0; sub < QT / 32; sub += NS) {
      const int pq = pt + 32 * sub;
      f32x16 s[NS], w[NS];
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        s[i] = zero16();
        if (MAPS == 2) {
          w[i] = zero16();
        } else {  // W - D out of the products at once (the kernel at 2 x 2048 causal, 16 heads of 128, bf16: 126 -> 116 us; 16 / 4 of 64: 67 -> 65)
#pragma unroll
          for (int rq = 0; rq < 4; ++rq) {
            const f32x4 D = *(const f32x4*)(rt + R_BYTES + (32 * (sub + i) + 8 * rq + 4 * h) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[i][4 * rq + e] = D[e];
          }
        }
      }
      if (MAPS == 1 || !skip) {
#pragma unroll
        for (int kk = 0; kk < KSV; ++kk)
#pragma unroll
          for (int i = 0; i < NS; ++i) w[i] = Num<T>::mfma(orr.get(st + MAPS * Q_BYTES, sub + i, kk), vf[kk], w[i]);
        if (MAPS == 2) put16(mine, w[0]);
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
#pragma unroll
          for (int i = 0; i < NS; ++i)
            s[i] = Num<T>::mfma(qr.get(st + m * Q_BYTES, sub + i, kk), kk < KS - KL ? kf[kk] : lds16(klds + (kk - (KS - KL)) * 1024), s[i]);
      }
      float mul = a.scale_log2, add = 0.f;
      if (BIAS) {
        if (kw0 + 31 - pq <= -a.R) add = far_lo;
        else if (kw0 - (pq + 32 * NS - 1) >= a.R) add = far_hi;
        else {
          const float* nb = near + (key - pq - 4 * h + a.R + E);
#pragma unroll
          for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[i][r] = fmaf(s[i][r], mul, nb[-32 * i - acc_row(r)]);
          mul = 1.f;
        }
      }
      if (kw0 + 31 >= len || (a.causal && kw0 + 31 > pq)) {
        const int dl = !valid ? 128 : (a.causal ? key - pq - 4 * h : -128);  // rows before dl do not see this lane's key
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[i][r] = 32 * i + acc_row(r) < dl ? -INFINITY : s[i][r];
      }
      // P' = 2^PSH P; rows_lse and rows_d carry 2^PSH and 2^-PSH
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
          const f32x4 nl = *(const f32x4*)(rt + m * R_BYTES + (32 * (sub + i) + 8 * rq + 4 * h) * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][4 * rq + e] = __builtin_amdgcn_exp2f(fmaf(s[i][4 * rq + e], mul, nl[e] + add));
        }
      u32x4 pv[NS][2];  // what meets dO in dV
      if (MAPS == 1) {
#pragma unroll
        for (int j = 0; j < NS; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) pv[j][i >> 2][i & 3] = Num<T>::pack(s[j][2 * i], s[j][2 * i + 1]);
      } else {
        if (!skip) put16(mine + 1024, s[0]);
        lds_barrier();
        if (skip) continue;
        const float f1 = ps * (m == 0 ? 1.f : -lam), f2 = ps * (m == 0 ? -lam : 1.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 w2 = *(const f32x4*)(theirs + i * 256), p2 = *(const f32x4*)(theirs + 1024 + i * 256);
          float pc[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[0][4 * i + e] += w2[e];
            pc[e] = fmaf(f1, s[0][4 * i + e], f2 * p2[e]);
          }
          pv[0][i >> 1][2 * (i & 1)] = Num<T>::pack(pc[0], pc[1]);
          pv[0][i >> 1][2 * (i & 1) + 1] = Num<T>::pack(pc[2], pc[3]);
        }
      }
#pragma unroll
      for (int kb2 = 0; kb2 < 2 * NS; ++kb2)
#pragma unroll
        for (int nt = 0; nt < VT; ++nt)
          if (MAPS == 1 || NT % 2 == 0 || m * VT + nt < NT) dv[nt] = Num<T>::mfma(ot.get(st + MAPS * Q_BYTES, 2 * sub + kb2, nt), pv[kb2 >> 1][kb2 & 1], dv[nt]);
      const float wf = (m == 0 ? PF : -lam * PF) * fs, wd = (m == 0 ? -1.f : lam) * fs;
      if (MAPS == 1) {
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[i][r] *= SCALED ? w[i][r] * wf : w[i][r];
      } else {
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
          const f32x4 D = *(const f32x4*)(rt + (MAPS + m) * R_BYTES + (8 * rq + 4 * h) * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[0][4 * rq + e] *= fmaf(w[0][4 * rq + e], wf, wd * D[e]);
        }
      }
#pragma unroll
      for (int kb2 = 0; kb2 < 2 * NS; ++kb2) {
        const f32x16& x = s[kb2 >> 1];
        u32x4 p;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = Num<T>::pack(x[8 * (kb2 & 1) + 2 * i], x[8 * (kb2 & 1) + 2 * i + 1]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) dk[dt] = Num<T>::mfma(qt.get(st + m * Q_BYTES, 2 * sub + kb2, dt), p, dk[dt]);
      }
    }
  }

  if (key >= a.Tk) return;  // keys behind len get zeros
  const float scale = a.scale * power(-fe), pf = PF * power(-pe);
  int at = key;
  opaque(at);  // (its 64-bit form of the loads above would wait through the walk)
  const int64_t row = ((int64_t)b * a.Tk + at) * a.Hkv + kvh;
  if (a.splits > 1) {  // 32-bit parts, (dk of each map, dv) of a key together
    float* pp = a.part_o + ((int64_t)split * a.B * a.Tk * a.Hkv + row) * (2 * a.dv);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        const int c0 = dt * 32 + rq * 8 + h * 4;
        const f32x16& x = dk[dt];
        if (c0 < a.d) *(f32x4*)(pp + m * a.d + c0) = f32x4{x[4 * rq] * scale, x[4 * rq + 1] * scale, x[4 * rq + 2] * scale, x[4 * rq + 3] * scale};
      }
#pragma unroll
    for (int nt = 0; nt < VT; ++nt)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        const int c0 = (m * VT + nt) * 32 + rq * 8 + h * 4;
        const f32x16& x = dv[nt];
        if (c0 < a.dv) *(f32x4*)(pp + a.dv + c0) = f32x4{x[4 * rq] * pf, x[4 * rq + 1] * pf, x[4 * rq + 2] * pf, x[4 * rq + 3] * pf};
      }
    return;
  }
  char* op = (char*)a.dk + (row * MAPS + m) * a.d * 2;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      const int c0 = dt * 32 + rq * 8 + h * 4;
      const f32x16& x = dk[dt];
      if (c0 < a.d)
        *(u32x2*)(op + c0 * 2) = u32x2{Num<T>::pack(x[4 * rq] * scale, x[4 * rq + 1] * scale), Num<T>::pack(x[4 * rq + 2] * scale, x[4 * rq + 3] * scale)};
    }
  op = (char*)a.dvo + row * a.dv * 2;
#pragma unroll
  for (int nt = 0; nt < VT; ++nt)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      const int c0 = (m * VT + nt) * 32 + rq * 8 + h * 4;
      const f32x16& x = dv[nt];
      if (c0 < a.dv)
        *(u32x2*)(op + c0 * 2) = u32x2{Num<T>::pack(x[4 * rq] * pf, x[4 * rq + 1] * pf), Num<T>::pack(x[4 * rq + 2] * pf, x[4 * rq + 3] * pf)};
    }
}

// dK, dV from the parts of a split walk: one thread per 4 channels
template <typename T>
__global__ __launch_bounds__(256) void mapattn_join_kernel(const MapAttnArgs a) {
  const int64_t rows = (int64_t)a.B * a.Tk * a.Hkv;
  const int qn = a.dv / 2;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * qn) return;
  const f32x4 t = add_parts(a.part_o + i * 4, a.splits, rows * qn * 4);
  const int64_t row = i / qn;
  const int c0 = (int)(i - row * qn) * 4;
  char* op = c0 < a.dv ? (char*)a.dk + (row * a.dv + c0) * 2 : (char*)a.dvo + (row * a.dv + c0 - a.dv) * 2;
  *(u32x2*)op = u32x2{Num<T>::pack(t[0], t[1]), Num<T>::pack(t[2], t[3])};
}

// D of rows whose walk was split, one thread per row: see the queries' kernel
template <int MAPS>
__global__ __launch_bounds__(256) void mapattn_rows_kernel(const MapAttnArgs a, float unit) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int m = MAPS == 2 ? blockIdx.y : 0;
  if (i >= (int64_t)a.B * a.H * a.Tq) return;
  const int64_t bh = i / a.Tq;
  const int q = (int)(i - bh * a.Tq), b = (int)(bh / a.H), head = (int)(bh - (int64_t)b * a.H);
  constexpr int NR = MAPS == 1 ? 3 : 2;
  const int64_t per = (int64_t)a.QW * 32;
  const float* p = a.rows3 + (((int64_t)head * a.B + b) * a.qsplits * NR + m) * per + q;
  float t = 0.f;
#pragma unroll 4
  for (int s = 0; s < a.qsplits; ++s) t += p[s * NR * per];
  float* d = a.rows_d + (bh * MAPS + m) * a.Tp + q;
  *d = MAPS == 1 ? *d - t : t * unit;
}

// dtable of many query groups: part sums of the diagonals, block (slots, part, head), one thread per slot; then a workgroup per head
__global__ __launch_bounds__(256) void mapattn_diag_kernel(const MapAttnArgs a) {
  const int slot = blockIdx.x * 256 + threadIdx.x, part = blockIdx.y, head = blockIdx.z;
  if (slot >= a.ND + 2) return;
  const int64_t rows = (int64_t)a.B * a.QW * a.qsplits, r0 = rows * part / a.parts, r1 = rows * (part + 1) / a.parts;
  const float* p = a.diag + ((int64_t)head * rows) * (a.ND + 2) + slot;
  float t = 0.f;
#pragma unroll 8
  for (int64_t r = r0; r < r1; ++r) t += p[r * (a.ND + 2)];
  a.diag_part[((int64_t)head * a.parts + part) * (a.ND + 2) + slot] = t;
}
template <typename T>
__global__ __launch_bounds__(512) void mapattn_dtable_kernel(const MapAttnArgs a) {
  __shared__ float sums[512];
  sum_table<T>(a, blockIdx.x, a.diag_part, a.parts, sums);
}

// ---- dispatch -----------------------------------------------------------------------------------------------------------
namespace {

template <typename T, int MAPS, int KS, int NT, int NG>
int run_dq(const MapAttnArgs& a, hipStream_t s) {
  constexpr int ROW = 16 * (MAPS * 4 * ((KS + 1) / 2) + 4 * NT);
  // tiles of 32 keys from 128 channels on: with 64 the kernel kept ten registers in scratch, reloaded in every step (16 x 500, 8 heads of
  // 128, the backward: 126.4 us against 125.3; 4 x 1500: 196 against 193; 160 channels, Q held in LDS for the same: 368 against 367)
  constexpr int KT = (MAPS == 2 || NG == 1 || KS >= 8) ? 32 : 64;
  // two sub-tiles of 32 at once where the registers allow two waves per SIMD all the same: two chains of products beside each other
  // (2 x 2048, 16 / 4 heads of 64: 54 us against 59, the keys' kernel 63 against 70; heads of 80: no difference)
  constexpr int NS = (KT == 64 && KS <= 4) ? 2 : 1;
  const int lds = 2 * KT * ROW + MAPS * NG * dq_held(MAPS, KS, NG) * 1024 + (MAPS == 1 ? (2 * (a.R + 32 * NG + KT) + 1) * 4 : 2 * NG * 4096);
  const void* f = (const void*)mapattn_dq_kernel<T, MAPS, KS, NT, KT, NG, NS>;
  if (anip_raise_lds_limit(f, lds) != 0) {
    anip_set_error("mapattn dq: cannot raise the dynamic LDS limit to %d bytes", lds);
    return -2;
  }
  const unsigned grid = mapattn_grid("mapattn_dq_kernel", (int64_t)(a.Tp / (32 * NG)) * a.splits * a.B * a.H, 64 * NG * MAPS);
  if (!grid) return -1;
  hipLaunchKernelGGL((mapattn_dq_kernel<T, MAPS, KS, NT, KT, NG, NS>), dim3(grid), dim3(64 * NG * MAPS), lds, s, a);
  ANIP_LAUNCH_CHECK("mapattn_dq_kernel");
  return 0;
}
template <typename T>
int table_sums(const MapAttnArgs& a, hipStream_t s) {
  if (a.diag_part != a.diag) {
    hipLaunchKernelGGL(mapattn_diag_kernel, dim3((unsigned)((a.ND + 2 + 255) / 256), (unsigned)a.parts, (unsigned)a.H), dim3(256), 0, s, a);
    ANIP_LAUNCH_CHECK("mapattn_diag_kernel");
  }
  hipLaunchKernelGGL((mapattn_dtable_kernel<T>), dim3((unsigned)a.H), dim3(512), 0, s, a);
  ANIP_LAUNCH_CHECK("mapattn_dtable_kernel");
  return 0;
}

template <typename T, int MAPS, int KS, int NT, int NG>
int run_dkv(const MapAttnArgs& a0, hipStream_t s) {
  MapAttnArgs a = a0;
  constexpr int ROW = 16 * (MAPS * 4 * ((KS + 1) / 2) + 4 * NT);
  constexpr int QT = (MAPS == 2 || NG == 1 || KS >= 8) ? 32 : 64;
  constexpr int NS = (QT == 64 && KS <= 4) ? 2 : 1;  // (see run_dq)
  const int lds = 2 * (QT * ROW + 2 * MAPS * 256) + MAPS * NG * dkv_held(MAPS, KS, NG) * 1024 + (MAPS == 1 ? (2 * (a.R + 32 * NG + QT) + 1) * 4 : 2 * NG * 8192);
  const void* f = (const void*)mapattn_dkv_kernel<T, MAPS, KS, NT, QT, NG, NS>;
  if (anip_raise_lds_limit(f, lds) != 0) {
    anip_set_error("mapattn dkv: cannot raise the dynamic LDS limit to %d bytes", lds);
    return -2;
  }
  // sums beside the keys' work: dlam always, dtable where a thread has few batches of loads, less time than the keys' work takes
  // (16 x 500, 8 heads of 64, 32 batches: 31 us, 26 + 11 in two kernels more; 4 heads of 32, 36 x 20, 24 of a lone wave: 22, 6 + 10)
  const int64_t groups = (int64_t)a.B * a.QW * a.qsplits;
  a.sum_blocks = MAPS == 2 || (cdiv64(groups, 16) * ((a.ND + 2 + 64 * NG - 1) / (64 * NG)) +
                                (a.qsplits > 1 ? cdiv64((int64_t)a.B * a.QW, 2 * NG) : 0)) <= (NG == 1 ? 12 : 48) ? a.H : 0;
  if (!a.sum_blocks) {
    const int r = table_sums<T>(a, s);
    if (r) return r;
  }
  const int64_t joins = a.qsplits > 1 ? cdiv64((int64_t)a.B * a.Tq * a.H * (a.dv / 4), 64 * NG * MAPS) : 0;
  const unsigned grid = mapattn_grid("mapattn_dkv_kernel", (int64_t)((a.Tk + 32 * NG - 1) / (32 * NG)) * a.splits * a.B * a.Hkv + a.sum_blocks + joins, 64 * NG * MAPS);
  if (!grid) return -1;
  a.join_blocks = (int)joins;
  hipLaunchKernelGGL((mapattn_dkv_kernel<T, MAPS, KS, NT, QT, NG, NS>), dim3(grid), dim3(64 * NG * MAPS), lds, s, a);
  ANIP_LAUNCH_CHECK("mapattn_dkv_kernel");
  return 0;
}

#define TRY1(KS, NT) if (ks <= KS) return nw == 1 ? run<T, 1, KS, NT, 1>(a, s) : run<T, 1, KS, NT, 4>(a, s);
#define TRY2(KS, NT) if (ks <= KS) return nw == 1 ? run<T, 2, KS, NT, 1>(a, s) : run<T, 2, KS, NT, 4>(a, s);
template <typename T>
int dq_t(const MapAttnArgs& a, int maps, int nw, hipStream_t s) {
  const int ks = (a.d + 15) / 16;
#define run run_dq
  if (maps == 1) { MAPATTN_GEOS_1(TRY1) } else { MAPATTN_GEOS_2(TRY2) }
#undef run
  return -1;
}
template <typename T>
int dkv_t(const MapAttnArgs& a, int maps, int nw, hipStream_t s) {
  const int ks = (a.d + 15) / 16;
#define run run_dkv
  if (maps == 1) { MAPATTN_GEOS_1(TRY1) } else { MAPATTN_GEOS_2(TRY2) }
#undef run
  return -1;
}

}  // namespace

int mapattn_dq(const MapAttnArgs& a, int maps, int bf16, int nw, hipStream_t s) { return bf16 ? dq_t<bf16_t>(a, maps, nw, s) : dq_t<f16>(a, maps, nw, s); }
int mapattn_dkv(const MapAttnArgs& a, int maps, int bf16, int nw, hipStream_t s) {
  if (a.qsplits > 1) {
    const dim3 rows((unsigned)cdiv64((int64_t)a.B * a.H * a.Tq, 256), (unsigned)maps);  // (fewer rows than the queries' kernel had threads)
    if (maps == 1) hipLaunchKernelGGL(mapattn_rows_kernel<1>, rows, dim3(256), 0, s, a, 1.0f);
    else hipLaunchKernelGGL(mapattn_rows_kernel<2>, rows, dim3(256), 0, s, a, bf16 ? 1.0f : 1.0f / (1 << Num<f16>::PSH));
    ANIP_LAUNCH_CHECK("mapattn_rows_kernel");
  }
  const int r = bf16 ? dkv_t<bf16_t>(a, maps, nw, s) : dkv_t<f16>(a, maps, nw, s);
  if (r || a.splits == 1) return r;
  const unsigned grid = mapattn_grid("mapattn_join_kernel", cdiv64((int64_t)a.B * a.Tk * a.Hkv * (a.dv / 2), 256), 256);
  if (!grid) return -1;
  if (bf16) hipLaunchKernelGGL((mapattn_join_kernel<bf16_t>), dim3(grid), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((mapattn_join_kernel<f16>), dim3(grid), dim3(256), 0, s, a);
  ANIP_LAUNCH_CHECK("mapattn_join_kernel");
  return 0;
}
