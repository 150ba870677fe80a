// Backward of the attention of mapattn.h.  With P_m the softmax maps, W = dO V^T (shared by both maps), D_m = rowsum(P_m W) =
// dO . o_m and w_1 = 1, w_2 = -lam:
//   dS_m = w_m P_m (W - D_m)   dQ_m = scale dS_m K_m   dK_m = scale dS_m^T Q_m   dV = (P_1 - lam P_2)^T dO
//   dlam = -sum P_2 W          dtable[bucket] = sum of dS over the pairs of the bucket
// Two kernels, one that owns queries (dQ, dlam, dtable's partial sums) and one that owns keys (dK, dV): each recomputes P and W
// (7 products instead of 5 at one map) and needs no atomics, so equal inputs give equal gradients.  P is recomputed from the row
// statistics of the forward; D from dO and the stored outputs.  dS and P are rounded to the inputs' type as operands of the
// matrix products (2^-9 or 2^-12 relative per term, averaged over a row); all sums are 32-bit.
#include "mapattn.h"

using namespace mapattn;

// ---- dQ: 32 queries per wave, tiles of KT keys ----------------------------------------------------------------------------
template <typename T, int MAPS, int KS, int NT, int KT, int NW>
__global__ __launch_bounds__(64 * NW, 1) void mapattn_dq_kernel(const MapAttnArgs a) {
  constexpr bool BIAS = MAPS == 1;
  constexpr int BQ = 32 * NW, DT = (KS + 1) / 2, KSV = MAPS == 1 ? KS : 2 * NT;
  constexpr int KCH = 4 * DT, VCH = 4 * NT;
  constexpr int K_BYTES = KT * KCH * 16, V_BYTES = KT * VCH * 16, STAGE = MAPS * K_BYTES + V_BYTES;
  constexpr int E = BQ + KT;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  float* near = (float*)(smem + 2 * STAGE);

  const int tid = threadIdx.x, lane = tid & 63, ql = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nqb = a.Tp / BQ;
  int qb, bh;
  if (!place(blockIdx.x, nqb, a.B * a.H, qb, bh)) return;
  qb = nqb - 1 - qb;
  const int b = bh / a.H, head = bh - b * a.H, kvh = head / a.G;
  const int len = seq_len(a, b), start = seq_start(a, b);
  const int q0 = qb * BQ + wave * 32, qi = q0 + ql, pw = start + q0;
  const bool valid = qi < a.Tq;
  const int lim = a.causal ? min(len - 1, start + qi) : len - 1;
  int kend = len;
  if (a.causal) kend = min(kend, start + min(qb * BQ + BQ, a.Tq));
  if (qb * BQ >= a.Tq) kend = 0;  // padding rows: only their row statistics are written
  const int nt_all = kend > 0 ? (kend + KT - 1) / KT : 0;

  const float lam = MAPS == 2 ? a.lam[head] : 0.f;
  u32x4 qf[MAPS][KS], df[KSV];
#pragma unroll
  for (int m = 0; m < MAPS; ++m)
    load_row<KS>(qf[m], (const char*)a.q + 2 * (b * a.q_sb + (int64_t)qi * a.q_st + (int64_t)(head * MAPS + m) * a.q_sh), valid, h, a.d);
  load_row<KSV>(df, (const char*)a.dout + 2 * (b * a.do_sb + (int64_t)qi * a.do_st + (int64_t)head * a.do_sh), valid, h, a.dv);

  // ---- row statistics: D_m = dO . o_m (o_1 = o + lam o_2), -lse in base 2 -------------------------------------------------
  float nl[MAPS], D[MAPS];
  {
    const int64_t orow = (((int64_t)b * a.Tq + qi) * a.H + head) * a.dv * 2;
    float dot[MAPS];
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      u32x4 of[KSV];
      load_row<KSV>(of, (const char*)(m == 0 ? a.out : a.out2) + orow, valid, h, a.dv);
      float t = 0.f;
#pragma unroll
      for (int kk = 0; kk < KSV; ++kk)
#pragma unroll
        for (int i = 0; i < 4; ++i) t = fmaf(Num<T>::lo(df[kk][i]), Num<T>::lo(of[kk][i]), fmaf(Num<T>::hi(df[kk][i]), Num<T>::hi(of[kk][i]), t));
      dot[m] = xor32_sum(t);
    }
    D[0] = dot[0];
    if (MAPS == 2) {
      D[MAPS - 1] = dot[MAPS - 1];
      D[0] = fmaf(lam, D[MAPS - 1], dot[0]);
    }
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      const float l = valid ? a.lse[((int64_t)bh * MAPS + m) * a.Tq + qi] * LOG2E : -INFINITY;
      nl[m] = l == -INFINITY ? -INFINITY : -l;  // rows without keys: P = 2^-inf = 0
      if (h == 0) {
        const int64_t at = ((int64_t)bh * MAPS + m) * a.Tp + qi;
        a.rows_lse[at] = nl[m] + Num<T>::PSH;
        a.rows_d[at] = D[m] * (1.0f / (1 << Num<T>::PSH));
      }
    }
  }

  float* diag = nullptr;
  if (BIAS && q0 < a.Tq) {
    diag = a.diag + (((int64_t)head * a.B + b) * a.QW + q0 / 32) * (a.ND + 2);
    for (int x = lane; x < a.ND + 2; x += 64) diag[x] = 0.f;  // (complete before the first tile's wait; later stores are this wave's own)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }

  const char* kb[MAPS];
#pragma unroll
  for (int m = 0; m < MAPS; ++m) kb[m] = (const char*)a.k + 2 * (b * a.k_sb + (int64_t)(kvh * MAPS + m) * a.k_sh);
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
    for (int m = 0; m < MAPS; ++m) kd.issue(kb[m] + row * a.k_st * 2, n, st + m * K_BYTES, wave);
    vd.issue(vb + row * a.v_st * 2, n, st + MAPS * K_BYTES, wave);
  };
  RowRead<KCH, KS> kr;
  RowRead<VCH, KSV> vr;
  TrRead<KCH, DT> kt;
  kr.init(lane);
  vr.init(lane);
  kt.init(lane);

  f32x16 dq[MAPS][DT];
#pragma unroll
  for (int m = 0; m < MAPS; ++m)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) dq[m][dt] = zero16();
  float far_lo = 0.f, far_hi = 0.f, sum_lo = 0.f, sum_hi = 0.f, dl_sum = 0.f;
  float dpos = 0.f, dneg = 0.f;  // diagonals rel = base + ql and base - 32 + ql of the current 32 keys, base = k0 - pw
  int next_base = 0;
  bool open = false;
  if (BIAS) {
    fill_near<T>(a, head, E, near, tid, 64 * NW);
    far_lo = bias_at<T>(a, head, -a.R);
    far_hi = bias_at<T>(a, head, a.R);
  }

  if (nt_all > 0) issue(0);
  for (int t = 0; t < nt_all; ++t) {
    MAPATTN_WAIT_DMA();
    __syncthreads();
    if (t + 1 < nt_all) issue(t + 1);
    const char* st = smem + (t & 1) * STAGE;
    const int kt0 = t * KT;
    if (a.causal && kt0 > pw + 31) continue;
#pragma unroll
    for (int sub = 0; sub < KT / 32; ++sub) {
      const int k0 = kt0 + 32 * sub;
      f32x16 s[MAPS], w = zero16();
#pragma unroll
      for (int m = 0; m < MAPS; ++m) {
        s[m] = zero16();
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) s[m] = Num<T>::mfma(kr.get(st + m * K_BYTES, sub, kk), qf[m][kk], s[m]);
      }
#pragma unroll
      for (int kk = 0; kk < KSV; ++kk) w = Num<T>::mfma(vr.get(st + MAPS * K_BYTES, sub, kk), df[kk], w);

      float mul = a.scale_log2, add = 0.f;
      int zone = 0;  // -1, 1: the whole of these 32 x 32 pairs beyond the bias's reach
      if (BIAS) {
        if (k0 + 31 - pw <= -a.R) { add = far_lo; zone = -1; }
        else if (k0 - (pw + 31) >= a.R) { add = far_hi; zone = 1; }
        else {
          const float* nb = near + (k0 + 4 * h - (pw + ql) + a.R + E);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[0][r] = fmaf(s[0][r], mul, nb[acc_row(r)]);
          mul = 1.f;
        }
      }
      if (k0 + 31 >= len || (a.causal && k0 + 31 > pw)) {
        const int dl = lim - k0 - 4 * h;
#pragma unroll
        for (int m = 0; m < MAPS; ++m)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[m][r] = acc_row(r) > dl ? -INFINITY : s[m][r];
      }
#pragma unroll
      for (int m = 0; m < MAPS; ++m) {
        const float c = add + nl[m];
        const float wf = m == 0 ? 1.f : -lam, wd = m == 0 ? -D[0] : lam * D[MAPS - 1];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[m][r], mul, c));
          if (MAPS == 2 && m == 1) dl_sum = fmaf(p, w[r], dl_sum);
          s[m][r] = p * (m == 0 ? w[r] + wd : fmaf(w[r], wf, wd));
        }
      }
      if (BIAS) {
        if (zone != 0) {
          float t16 = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) t16 += s[0][r];
          if (zone < 0) sum_lo += t16;
          else sum_hi += t16;
        } else {
          // value of (key k0 + ko, query ql) belongs to diagonal ko - ql: lane x takes it from lane (ko - x) mod 32 of its half
          open = true;
          next_base = k0 + 32 - pw;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int ko = acc_row(r) + 4 * h;
            const float v = __uint_as_float(__builtin_amdgcn_ds_bpermute((((ko - ql) & 31) | (lane & 32)) << 2, __float_as_uint(s[0][r])));
            dpos += ql <= ko ? v : 0.f;
            dneg += ql <= ko ? 0.f : v;
          }
          const float done = xor32_sum(dneg);  // no later key reaches these 32 diagonals
          if (diag && h == 0) diag[k0 - pw - 32 + ql + a.R + 64] = done;
          dneg = dpos;
          dpos = 0.f;
        }
      }
#pragma unroll
      for (int m = 0; m < MAPS; ++m) {
        u32x4 p[2];
#pragma unroll
        for (int kb2 = 0; kb2 < 2; ++kb2) {
#pragma unroll
          for (int i = 0; i < 4; ++i) p[kb2][i] = Num<T>::pack(s[m][8 * kb2 + 2 * i], s[m][8 * kb2 + 2 * i + 1]);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) dq[m][dt] = Num<T>::mfma(kt.get(st + m * K_BYTES, 2 * sub + kb2, dt), p[kb2], dq[m][dt]);
        }
      }
    }
  }

  if (BIAS && diag) {
    const float done = xor32_sum(dneg);
    if (open && h == 0) diag[next_base - 32 + ql + a.R + 64] = done;
    const float lo = wave_sum(sum_lo), hi = wave_sum(sum_hi);
    if (lane == 0) {
      diag[a.ND] = lo;
      diag[a.ND + 1] = hi;
    }
  }
  if (MAPS == 2 && q0 < a.Tq) {
    const float t = wave_sum(dl_sum);
    if (lane == 0) a.dlam_part[((int64_t)head * a.B + b) * a.QW + q0 / 32] = -t;
  }
  if (!valid) return;
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    char* op = (char*)a.dq + ((((int64_t)b * a.Tq + qi) * a.H + head) * MAPS + m) * a.d * 2;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        const int c0 = dt * 32 + rq * 8 + h * 4;
        const f32x16& x = dq[m][dt];
        if (c0 < a.d)
          *(u32x2*)(op + c0 * 2) = u32x2{Num<T>::pack(x[4 * rq] * a.scale, x[4 * rq + 1] * a.scale), Num<T>::pack(x[4 * rq + 2] * a.scale, x[4 * rq + 3] * a.scale)};
      }
  }
}

// ---- dK, dV: 32 keys per wave (K and V rows in registers), tiles of QT queries of every head that shares them ------------------
template <typename T, int MAPS, int KS, int NT, int QT, int NW>
__global__ __launch_bounds__(64 * NW, 1) void mapattn_dkv_kernel(const MapAttnArgs a) {
  constexpr bool BIAS = MAPS == 1;
  constexpr int BK = 32 * NW, DT = (KS + 1) / 2, KSV = MAPS == 1 ? KS : 2 * NT;
  constexpr int QCH = 4 * DT, OCH = 4 * NT;
  constexpr int Q_BYTES = QT * QCH * 16, O_BYTES = QT * OCH * 16, R_BYTES = 256;
  constexpr int STAGE = MAPS * Q_BYTES + O_BYTES + 2 * MAPS * R_BYTES;
  constexpr int E = BK + QT;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  float* near = (float*)(smem + 2 * STAGE);

  const int tid = threadIdx.x, lane = tid & 63, kl = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nkb = (a.Tk + BK - 1) / BK;
  int kblk, bk;
  if (!place(blockIdx.x, nkb, a.B * a.Hkv, kblk, bk)) return;  // causal: the first keys meet the most queries
  const int b = bk / a.Hkv, kvh = bk - b * a.Hkv;
  const int len = seq_len(a, b), start = seq_start(a, b);
  const int kw0 = kblk * BK + wave * 32, key = kw0 + kl;
  const bool valid = key < len;

  u32x4 kf[MAPS][KS], vf[KSV];
#pragma unroll
  for (int m = 0; m < MAPS; ++m)
    load_row<KS>(kf[m], (const char*)a.k + 2 * (b * a.k_sb + (int64_t)key * a.k_st + (int64_t)(kvh * MAPS + m) * a.k_sh), valid, h, a.d);
  load_row<KSV>(vf, (const char*)a.v + 2 * (b * a.v_sb + (int64_t)key * a.v_st + (int64_t)kvh * a.v_sh), valid, h, a.dv);

  // ---- query tiles that meet these keys -----------------------------------------------------------------------------------
  const int nqt = (a.Tq + QT - 1) / QT;
  int tq0 = 0;
  if (a.causal) {
    const int first = kblk * BK - start;  // first query that sees the workgroup's first key
    tq0 = first <= 0 ? 0 : min(first / QT, nqt);
  }
  const int per = kblk * BK < len ? nqt - tq0 : 0, total = per * a.G;

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
    for (int m = 0; m < MAPS; ++m)
      qd.issue((const char*)a.q + 2 * (b * a.q_sb + row * a.q_st + (int64_t)(head * MAPS + m) * a.q_sh), n, st + m * Q_BYTES, wave);
    od.issue((const char*)a.dout + 2 * (b * a.do_sb + row * a.do_st + (int64_t)head * a.do_sh), n, st + MAPS * Q_BYTES, wave);
    char* rt = st + MAPS * Q_BYTES + O_BYTES;
#pragma unroll
    for (int i = 0; i < 2 * MAPS; ++i)
      if (i % NW == wave) {
        const float* src = (i < MAPS ? a.rows_lse : a.rows_d) + ((int64_t)(b * a.H + head) * MAPS + i % MAPS) * a.Tp + row;
        dma4(src, QT * 4, rt + i * R_BYTES, lane * 4);
      }
  };
  RowRead<QCH, KS> qr;
  RowRead<OCH, KSV> orr;
  TrRead<QCH, DT> qt;
  TrRead<OCH, NT> ot;
  qr.init(lane);
  orr.init(lane);
  qt.init(lane);
  ot.init(lane);

  f32x16 dk[MAPS][DT], dv[NT];
#pragma unroll
  for (int m = 0; m < MAPS; ++m)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) dk[m][dt] = zero16();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) dv[nt] = zero16();
  float far_lo = 0.f, far_hi = 0.f, lam = 0.f;
  constexpr float PF = 1.0f / (1 << Num<T>::PSH);

  if (total > 0) issue(0);
  for (int it = 0; it < total; ++it) {
    const int g = it / per, t = tq0 + it - g * per;
    if (it - g * per == 0) {  // the next head: its bias, its lam
      const int head = kvh * a.G + g;
      if (BIAS) {
        if (g > 0) __syncthreads();  // the head before is read to the end
        fill_near<T>(a, head, E, near, tid, 64 * NW);
        far_lo = bias_at<T>(a, head, -a.R);
        far_hi = bias_at<T>(a, head, a.R);
      } else {
        lam = a.lam[head];
      }
    }
    MAPATTN_WAIT_DMA();
    __syncthreads();
    if (it + 1 < total) issue(it + 1);
    const char* st = smem + (it & 1) * STAGE;
    const char* rt = st + MAPS * Q_BYTES + O_BYTES;
    const int pt = start + t * QT;
    if (a.causal && pt + QT - 1 < kw0) continue;  // no query of the tile sees this wave's keys
#pragma unroll
    for (int sub = 0; sub < QT / 32; ++sub) {
      const int pq = pt + 32 * sub;
      f32x16 s[MAPS], w = zero16();
#pragma unroll
      for (int m = 0; m < MAPS; ++m) {
        s[m] = zero16();
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) s[m] = Num<T>::mfma(qr.get(st + m * Q_BYTES, sub, kk), kf[m][kk], s[m]);
      }
#pragma unroll
      for (int kk = 0; kk < KSV; ++kk) w = Num<T>::mfma(orr.get(st + MAPS * Q_BYTES, sub, kk), vf[kk], w);
      float mul = a.scale_log2, add = 0.f;
      if (BIAS) {
        if (kw0 + 31 - pq <= -a.R) add = far_lo;
        else if (kw0 - (pq + 31) >= a.R) add = far_hi;
        else {
          const float* nb = near + (key - pq - 4 * h + a.R + E);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[0][r] = fmaf(s[0][r], mul, nb[-acc_row(r)]);
          mul = 1.f;
        }
      }
      if (kw0 + 31 >= len || (a.causal && kw0 + 31 > pq)) {
        const int dl = !valid ? 64 : (a.causal ? key - pq - 4 * h : -64);  // rows before dl do not see this lane's key
#pragma unroll
        for (int m = 0; m < MAPS; ++m)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[m][r] = acc_row(r) < dl ? -INFINITY : s[m][r];
      }
      // P' = 2^PSH P; rows_lse and rows_d carry 2^PSH and 2^-PSH
      f32x16 ds[MAPS];
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        f32x4 nl[MAPS], D[MAPS];
#pragma unroll
        for (int m = 0; m < MAPS; ++m) {
          nl[m] = *(const f32x4*)(rt + m * R_BYTES + (32 * sub + 8 * rq + 4 * h) * 4);
          D[m] = *(const f32x4*)(rt + (MAPS + m) * R_BYTES + (32 * sub + 8 * rq + 4 * h) * 4);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * rq + e;
#pragma unroll
          for (int m = 0; m < MAPS; ++m) s[m][r] = __builtin_amdgcn_exp2f(fmaf(s[m][r], mul, nl[m][e] + add));
          ds[0][r] = s[0][r] * fmaf(w[r], PF, -D[0][e]);
          if (MAPS == 2) {
            ds[MAPS - 1][r] = -lam * (s[MAPS - 1][r] * fmaf(w[r], PF, -D[MAPS - 1][e]));
            s[0][r] = fmaf(-lam, s[MAPS - 1][r], s[0][r]);
          }
        }
      }
#pragma unroll
      for (int kb2 = 0; kb2 < 2; ++kb2) {
        u32x4 p;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = Num<T>::pack(s[0][8 * kb2 + 2 * i], s[0][8 * kb2 + 2 * i + 1]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) dv[nt] = Num<T>::mfma(ot.get(st + MAPS * Q_BYTES, 2 * sub + kb2, nt), p, dv[nt]);
#pragma unroll
        for (int m = 0; m < MAPS; ++m) {
#pragma unroll
          for (int i = 0; i < 4; ++i) p[i] = Num<T>::pack(ds[m][8 * kb2 + 2 * i], ds[m][8 * kb2 + 2 * i + 1]);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) dk[m][dt] = Num<T>::mfma(qt.get(st + m * Q_BYTES, 2 * sub + kb2, dt), p, dk[m][dt]);
        }
      }
    }
  }

  if (key >= a.Tk) return;  // keys behind len get zeros
  const int64_t row = ((int64_t)b * a.Tk + key) * a.Hkv + kvh;
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    char* op = (char*)a.dk + (row * MAPS + m) * a.d * 2;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        const int c0 = dt * 32 + rq * 8 + h * 4;
        const f32x16& x = dk[m][dt];
        if (c0 < a.d)
          *(u32x2*)(op + c0 * 2) = u32x2{Num<T>::pack(x[4 * rq] * a.scale, x[4 * rq + 1] * a.scale), Num<T>::pack(x[4 * rq + 2] * a.scale, x[4 * rq + 3] * a.scale)};
      }
  }
  char* op = (char*)a.dvo + row * a.dv * 2;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      const int c0 = nt * 32 + rq * 8 + h * 4;
      const f32x16& x = dv[nt];
      if (c0 < a.dv)
        *(u32x2*)(op + c0 * 2) = u32x2{Num<T>::pack(x[4 * rq] * PF, x[4 * rq + 1] * PF), Num<T>::pack(x[4 * rq + 2] * PF, x[4 * rq + 3] * PF)};
    }
}

// ---- sums of the query groups' parts, in a fixed order --------------------------------------------------------------------
// part sums of dtable's diagonals: block (slots, part, head), one thread per slot
__global__ __launch_bounds__(256) void mapattn_diag_kernel(const MapAttnArgs a) {
  const int slot = blockIdx.x * 256 + threadIdx.x, part = blockIdx.y, head = blockIdx.z;
  if (slot >= a.ND + 2) return;
  const int64_t rows = (int64_t)a.B * a.QW, r0 = rows * part / a.parts, r1 = rows * (part + 1) / a.parts;
  const float* p = a.diag + ((int64_t)head * rows) * (a.ND + 2) + slot;
  float t = 0.f;
  for (int64_t r = r0; r < r1; ++r) t += p[r * (a.ND + 2)];
  a.diag_part[((int64_t)head * a.parts + part) * (a.ND + 2) + slot] = t;
}
template <typename T>
__global__ __launch_bounds__(256) void mapattn_dtable_kernel(const MapAttnArgs a) {
  extern __shared__ float sums[];
  const int head = blockIdx.x, n = a.ND + 2;
  for (int x = threadIdx.x; x < n; x += 256) {
    float t = 0.f;
    for (int p = 0; p < a.parts; ++p) t += a.diag_part[((int64_t)head * a.parts + p) * n + x];
    sums[x] = t;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.NB; c += 256) {
    float t = 0.f;
    for (int x = 0; x <= 2 * a.R; ++x) {
      int bx = a.buckets[x];
      bx = bx < 0 ? 0 : (bx >= a.NB ? a.NB - 1 : bx);
      if (bx != c) continue;
      t += sums[x + 64];
      if (x == 0) {
        t += sums[a.ND];
        for (int i = 0; i < 64; ++i) t += sums[i];
      }
      if (x == 2 * a.R) {
        t += sums[a.ND + 1];
        for (int i = 2 * a.R + 65; i < a.ND; ++i) t += sums[i];
      }
    }
    ((T*)a.dtable)[(int64_t)head * a.NB + c] = (T)t;
  }
}
__global__ __launch_bounds__(256) void mapattn_dlam_kernel(const MapAttnArgs a) {
  __shared__ float part[4];
  const int64_t rows = (int64_t)a.B * a.QW;
  const float* p = a.dlam_part + blockIdx.x * rows;
  float t = 0.f;
  for (int64_t r = threadIdx.x; r < rows; r += 256) t += p[r];
  t = wave_sum(t);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x == 0) a.dlam[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// ---- dispatch -----------------------------------------------------------------------------------------------------------
namespace {

template <typename T, int MAPS, int KS, int NT, int NW>
int run_dq(const MapAttnArgs& a, hipStream_t s) {
  constexpr int ROW = 16 * (MAPS * 4 * ((KS + 1) / 2) + 4 * NT);
  constexpr int KT = (NW == 1 || 2 * 64 * ROW > 64 * 1024) ? 32 : 64;
  const int lds = 2 * KT * ROW + (MAPS == 1 ? (2 * (a.R + 32 * NW + KT) + 1) * 4 : 0);
  const void* f = (const void*)mapattn_dq_kernel<T, MAPS, KS, NT, KT, NW>;
  if (anip_raise_lds_limit(f, lds) != 0) {
    anip_set_error("mapattn dq: cannot raise the dynamic LDS limit to %d bytes", lds);
    return -2;
  }
  hipLaunchKernelGGL((mapattn_dq_kernel<T, MAPS, KS, NT, KT, NW>), dim3((unsigned)(a.Tp / (32 * NW) * a.B * a.H)), dim3(64 * NW), lds, s, a);
  ANIP_LAUNCH_CHECK("mapattn_dq_kernel");
  return 0;
}
template <typename T, int MAPS, int KS, int NT, int NW>
int run_dkv(const MapAttnArgs& a, hipStream_t s) {
  constexpr int ROW = 16 * (MAPS * 4 * ((KS + 1) / 2) + 4 * NT);
  constexpr int QT = (NW == 1 || 2 * 64 * ROW > 64 * 1024) ? 32 : 64;
  const int lds = 2 * (QT * ROW + 2 * MAPS * 256) + (MAPS == 1 ? (2 * (a.R + 32 * NW + QT) + 1) * 4 : 0);
  const void* f = (const void*)mapattn_dkv_kernel<T, MAPS, KS, NT, QT, NW>;
  if (anip_raise_lds_limit(f, lds) != 0) {
    anip_set_error("mapattn dkv: cannot raise the dynamic LDS limit to %d bytes", lds);
    return -2;
  }
  hipLaunchKernelGGL((mapattn_dkv_kernel<T, MAPS, KS, NT, QT, NW>), dim3((unsigned)((a.Tk + 32 * NW - 1) / (32 * NW) * a.B * a.Hkv)), dim3(64 * NW), lds, s, a);
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
int mapattn_dkv(const MapAttnArgs& a, int maps, int bf16, int nw, hipStream_t s) { return bf16 ? dkv_t<bf16_t>(a, maps, nw, s) : dkv_t<f16>(a, maps, nw, s); }
int mapattn_reduce(const MapAttnArgs& a, int maps, int bf16, hipStream_t s) {
  if (maps == 2) {
    hipLaunchKernelGGL(mapattn_dlam_kernel, dim3((unsigned)a.H), dim3(256), 0, s, a);
    ANIP_LAUNCH_CHECK("mapattn_dlam_kernel");
    return 0;
  }
  hipLaunchKernelGGL(mapattn_diag_kernel, dim3((unsigned)((a.ND + 2 + 255) / 256), (unsigned)a.parts, (unsigned)a.H), dim3(256), 0, s, a);
  ANIP_LAUNCH_CHECK("mapattn_diag_kernel");
  const int lds = (a.ND + 2) * 4;
  if (bf16) hipLaunchKernelGGL((mapattn_dtable_kernel<bf16_t>), dim3((unsigned)a.H), dim3(256), lds, s, a);
  else hipLaunchKernelGGL((mapattn_dtable_kernel<f16>), dim3((unsigned)a.H), dim3(256), lds, s, a);
  ANIP_LAUNCH_CHECK("mapattn_dtable_kernel");
  return 0;
}
