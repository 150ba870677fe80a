// Forward of the attention of mapattn.h: QG x 32 queries of one head per workgroup, a wave for each 32, tiles of KT keys in two LDS
// stages, one pass over the keys with running maxima and sums (base 2).  S^T = K Q^T per 32 keys, so that a lane owns one query:
// its maximum and sum are 16 register operations and one exchange between the half-waves, and P^T is the B operand of
// O^T += V^T P^T as it lies.  Differential attention gives each of its two
// maps a wave of its own (two accumulators of 2 d channels would not fit one wave's registers from d = 64 on); both read the same
// V tile, and the second hands its share to the first at the end.
#include "mapattn.h"

using namespace mapattn;

namespace {

constexpr float THR = 8.0f;  // the running maximum is raised when a score exceeds it by more: P <= 2^8

// a running softmax over NS x 32 keys: scores s (x = mul s + add in base 2) -> P fragments
template <typename T, int NT, int NS>
__device__ __forceinline__ void soft_step(f32x16 (&s)[NS], float mul, float add, float& m, float& l, f32x16 (&o)[NT], u32x4 (&p)[NS][2]) {
  float mx = fmaxf(fmaxf(s[0][0], s[0][1]), s[0][2]);
#pragma unroll
  for (int r = 3; r < 15; r += 2) mx = fmaxf(fmaxf(mx, s[0][r]), s[0][r + 1]);
  if (NS == 1) {
    mx = fmaxf(mx, s[0][15]);
  } else {
    mx = fmaxf(fmaxf(mx, s[0][15]), s[NS - 1][0]);
#pragma unroll
    for (int r = 1; r < 15; r += 2) mx = fmaxf(fmaxf(mx, s[NS - 1][r]), s[NS - 1][r + 1]);
    mx = fmaxf(mx, s[NS - 1][15]);
  }
  mx = fmaf(xor32_max(mx), mul, add);
  if (__any(mx - m > THR)) {  // always on the first seen key (m = -inf); never while both are -inf (NaN > THR is false)
    const float mn = fmaxf(m, mx);
    const float alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
    m = mn;
    l *= alpha;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[nt][r] *= alpha;
  }
  const float c = add - (m == -INFINITY ? 0.f : m);
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[i][r] = __builtin_amdgcn_exp2f(fmaf(s[i][r], mul, c));
      t += s[i][r];
    }
    l += t;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int j = 0; j < 4; ++j) p[i][kb][j] = Num<T>::pack(s[i][8 * kb + 2 * j], s[i][8 * kb + 2 * j + 1]);
  }
}

}  // namespace

template <typename T, int MAPS, int KS, int NT, int KT, int NS, int QG>
__global__ __launch_bounds__(64 * QG * MAPS, 2) void mapattn_fwd_kernel(const MapAttnArgs a) {
  constexpr bool BIAS = MAPS == 1;
  constexpr int NW = QG * MAPS, BQ = 32 * QG;
  constexpr int KCH = 4 * ((KS + 1) / 2), VCH = 4 * NT;
  constexpr int K_BYTES = KT * KCH * 16, V_BYTES = KT * VCH * 16, STAGE = MAPS * K_BYTES + V_BYTES;
  constexpr int E = BQ + KT;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  float* near = (float*)(smem + 2 * STAGE);

  const int tid = threadIdx.x, lane = tid & 63, ql = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave / MAPS, m = wave % MAPS;  // 32 queries, and the map that this wave computes for them
  const int nqb = (a.Tq + BQ - 1) / BQ;
  int slot, bh;
  place<MAPS == 1 || (NT < 8)>(blockIdx.x, nqb * a.splits, a.B * a.H, a.causal, slot, bh);
  const int split = slot % a.splits, qb = nqb - 1 - slot / a.splits;  // causal: the longest rows first
  const int b = bh / a.H, head = bh - b * a.H, kvh = head / a.G;
  const int len = seq_len(a, b), start = seq_start(a, b);
  const int qi = qb * BQ + grp * 32 + ql;      // this lane's query
  const int pw = start + qb * BQ + grp * 32;   // position of the wave's first query
  const int lim = a.causal ? min(len - 1, start + qi) : len - 1;  // last key this lane sees

  // ---- the keys this workgroup walks over -------------------------------------------------------------------------------
  int kend = len;
  if (a.causal) kend = min(kend, start + min(qb * BQ + BQ, a.Tq));
  const int nt_all = kend > 0 ? (kend + KT - 1) / KT : 0;
  const int t0 = (int)((int64_t)nt_all * split / a.splits), t1 = (int)((int64_t)nt_all * (split + 1) / a.splits);

  u32x4 qf[KS];
  load_row<KS>(qf, (const char*)a.q + 2 * (b * a.q_sb + (int64_t)qi * a.q_st + (int64_t)(head * MAPS + m) * a.q_sh), qi < a.Tq, h, a.d);

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
    const int valid = len - t * KT;
#pragma unroll
    for (int i = 0; i < MAPS; ++i) kd.issue(kb[i] + row * a.k_st * 2, valid, st + i * K_BYTES, wave);
    vd.issue(vb + row * a.v_st * 2, valid, st + MAPS * K_BYTES, wave);
  };
  RowRead<KCH> kr;
  TrRead<VCH> vr;
  kr.init(lane);
  vr.init(lane);

  f32x16 o[NT];
  float mrun = -INFINITY, lrun = 0.f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) o[nt] = zero16();
  float far_lo = 0.f, far_hi = 0.f;
  if (BIAS) {
    fill_near<T>(a, head, E, near, tid, 64 * NW);
    far_lo = bias_at<T>(a, head, -a.R);
    far_hi = bias_at<T>(a, head, a.R);
  }

  if (t0 < t1) issue(t0);
  for (int t = t0; t < t1; ++t) {
    MAPATTN_WAIT_DMA();
    __syncthreads();  // tile t is there for all waves; nobody reads the other stage any more
    if (t + 1 < t1) issue(t + 1);
    if (MAPS * NT >= 16) {
      opaque(kr.base);
      opaque(vr.base);
    }
    const char* st = smem + (t & 1) * STAGE;
    const int kt0 = t * KT;
    if (a.causal && kt0 > pw + 31) continue;  // nothing of this tile is seen by this wave
#pragma unroll
    for (int sub = 0; sub < KT / 32; sub += NS) {
      const int k0 = kt0 + 32 * sub;
      f32x16 s[NS];
#pragma unroll
      for (int i = 0; i < NS; ++i) s[i] = zero16();
#pragma unroll
      for (int kk = 0; kk < KS; ++kk)
#pragma unroll
        for (int i = 0; i < NS; ++i) s[i] = Num<T>::mfma(kr.get(st + m * K_BYTES, sub + i, kk), qf[kk], s[i]);
      float mul = a.scale_log2, add = 0.f;
      if (BIAS) {
        if (k0 + 32 * NS - 1 - pw <= -a.R) add = far_lo;
        else if (k0 - (pw + 31) >= a.R) add = far_hi;
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
      u32x4 p[NS][2];
      soft_step<T, NT, NS>(s, mul, add, mrun, lrun, o, p);
#pragma unroll
      for (int kb2 = 0; kb2 < 2 * NS; ++kb2)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) o[nt] = Num<T>::mfma(vr.get(st + MAPS * K_BYTES, 2 * sub + kb2, nt), p[kb2 >> 1][kb2 & 1], o[nt]);
    }
  }

  // ---- epilogue ---------------------------------------------------------------------------------------------------------
  const float l = xor32_sum(lrun);
  const bool none = l == 0.f;  // no key seen: the row is zeros.  (Not where all scores are NaN: their sum is, while no maximum was set)
  const float inv = none ? 0.f : 1.0f / l;
  const float lse2 = none ? -INFINITY : mrun + __builtin_amdgcn_logf(l);
  if (MAPS == 2 && a.splits == 1) {
    // the second map's wave hands lam o2 to the first one's, lane for lane
    float* x = (float*)smem + grp * (NT * 16 * 64) + lane;
    __syncthreads();  // all tiles read
    if (m == 1) {
      const float f = inv * a.lam[head];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[(nt * 16 + r) * 64] = o[nt][r] * f;
    }
    __syncthreads();
    if (m == 0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[nt][r] = o[nt][r] * inv - x[(nt * 16 + r) * 64];
    }
  }
  if (qi >= a.Tq) return;
  const int64_t row = ((int64_t)b * a.Tq + qi) * a.H + head;
  if (a.splits > 1) {
    const int64_t at = ((int64_t)split * a.B * a.Tq * a.H + row) * MAPS + m;
    float* op = a.part_o + at * a.dv;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        const int c0 = nt * 32 + rq * 8 + h * 4;
        if (c0 < a.dv) *(f32x4*)(op + c0) = f32x4{o[nt][4 * rq] * inv, o[nt][4 * rq + 1] * inv, o[nt][4 * rq + 2] * inv, o[nt][4 * rq + 3] * inv};
      }
    if (h == 0) a.part_l[at] = lse2;
    return;
  }
  if (a.lse && h == 0) a.lse[((int64_t)bh * MAPS + m) * a.Tq + qi] = lse2 * LN2;
  char* op = (char*)(m == 0 ? a.out : a.out2);
  if (op == nullptr) return;
  op += row * a.dv * 2;
  const float f = (MAPS == 2 && m == 0) ? 1.0f : inv;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      const int c0 = nt * 32 + rq * 8 + h * 4;
      if (c0 < a.dv)
        *(u32x2*)(op + c0 * 2) = u32x2{Num<T>::pack(o[nt][4 * rq] * f, o[nt][4 * rq + 1] * f), Num<T>::pack(o[nt][4 * rq + 2] * f, o[nt][4 * rq + 3] * f)};
    }
}

// ---- single tokens: few queries against many keys -----------------------------------------------------------------------
// The Tq x G queries that share a key head are at most 32 columns of one tile.  Bound by reading the keys and values once, so a
// team of MAPS waves (one for each map, sharing the V tile) walks its own 32-key tiles; the kw = teams teams of a workgroup share a
// problem (tiles t, t + kw, ..) and join their results in LDS, or each team has its own problem (kw = 1: many short sequences).
// One map: a team is one wave and needs no barrier; it has one K and one V tile in LDS and refills each as soon as it is read, so
// that eight waves fit a CU and nearly a tile of each is in flight.  Two maps: two stages, a barrier per tile.
template <typename T, int MAPS, int KS, int NT, int MAXT>
__global__ __launch_bounds__(64 * MAXT * MAPS, (MAPS == 1 ? 2 : 1)) void mapattn_token_kernel(const MapAttnArgs a) {
  constexpr bool BIAS = MAPS == 1;
  constexpr int KT = 32;
  constexpr int KCH = 4 * ((KS + 1) / 2), VCH = 4 * NT;
  constexpr int K_BYTES = KT * KCH * 16, V_BYTES = KT * VCH * 16, STAGE = MAPS * K_BYTES + V_BYTES;
  constexpr int TEAM = MAPS == 1 ? STAGE : 2 * STAGE;
  constexpr int OW = NT * 16 * 64;  // floats of a wave's result
  extern __shared__ __attribute__((aligned(1024))) char smem[];

  const int tid = threadIdx.x, lane = tid & 63, ql = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int team = wave / MAPS, m = wave % MAPS;
  const int ppb = a.teams / a.kw, kwi = team % a.kw;
  const int problems = a.B * a.Hkv * a.splits;  // (fewer than 2^31: mapattn_grid)
  const int prob = blockIdx.x * ppb + team / a.kw;
  const bool live = prob < problems;  // (kw = teams: the same for all waves)
  const int split = prob % a.splits, bk = live ? prob / a.splits : 0;
  const int b = bk / a.Hkv, kvh = bk - b * a.Hkv;
  const int len = live ? seq_len(a, b) : 0, start = seq_start(a, b);
  const int nrow = a.Tq * a.G;
  const int qi = ql / a.G, head = kvh * a.G + (ql - qi * a.G);
  const bool mine = live && ql < nrow;
  const int lim = mine ? (a.causal ? min(len - 1, start + qi) : len - 1) : -1;

  const int nt_all = (len + KT - 1) / KT;
  const int t0 = (int)((int64_t)nt_all * split / a.splits), t1 = (int)((int64_t)nt_all * (split + 1) / a.splits);
  // turns of the loop: with barriers inside, the same for all teams of the workgroup
  const int turns = MAPS == 1 ? (t1 - t0 - kwi + a.kw - 1) / a.kw : (a.kw == 1 ? (a.Tk + KT - 1) / KT : (t1 - t0 + a.kw - 1) / a.kw);

  const char* kb[MAPS];
#pragma unroll
  for (int i = 0; i < MAPS; ++i) kb[i] = (const char*)a.k + 2 * (b * a.k_sb + (int64_t)(kvh * MAPS + i) * a.k_sh);
  const char* vb = (const char*)a.v + 2 * (b * a.v_sb + (int64_t)kvh * a.v_sh);
  TileDma<KCH, KT, MAPS> kd;
  TileDma<VCH, KT, MAPS> vd;
  kd.init(m, lane, a.k_st, a.d);
  vd.init(m, lane, a.v_st, a.dv);
  char* mem = smem + team * TEAM;
  auto issue_k = [&](int t, char* p) {
#pragma unroll
    for (int i = 0; i < MAPS; ++i) kd.issue(kb[i] + (int64_t)t * KT * a.k_st * 2, len - t * KT, p + i * K_BYTES, m);
  };
  auto issue_v = [&](int t, char* p) { vd.issue(vb + (int64_t)t * KT * a.v_st * 2, len - t * KT, p + MAPS * K_BYTES, m); };
  constexpr int KP = TileDma<KCH, KT, 1>::P, VP = TileDma<VCH, KT, 1>::P;  // pieces of a tile (one map: all of them this wave's)

  u32x4 qf[KS];
  load_row<KS>(qf, (const char*)a.q + 2 * (b * a.q_sb + (int64_t)qi * a.q_st + (int64_t)(head * MAPS + m) * a.q_sh), mine, h, a.d);
  const float far_lo = BIAS && mine ? bias_at<T>(a, head, -a.R) : 0.f, far_hi = BIAS && mine ? bias_at<T>(a, head, a.R) : 0.f;
  // (one map) bias of a tile near the queries: [G][31 + Tq] relative positions k0 - (start + Tq - 1) ..
  float* near = (float*)(smem + a.teams * TEAM) + team * (a.G * (31 + a.Tq));
  const float* nq = mine ? near + (ql - qi * a.G) * (31 + a.Tq) + (a.Tq - 1 - qi) + 4 * h : near;
  if (t0 + kwi < t1) {
    issue_k(t0 + kwi, mem);
    issue_v(t0 + kwi, mem);
  }
  RowRead<KCH> kr;
  TrRead<VCH> vr;
  kr.init(lane);
  vr.init(lane);

  f32x16 o[NT];
  float mrun = -INFINITY, lrun = 0.f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) o[nt] = zero16();

  for (int it = 0; it < turns; ++it) {
    const int t = t0 + kwi + it * a.kw;
    const int k0 = t * KT;
    const bool more = t + a.kw < t1;
    float mul = a.scale_log2, add = 0.f;
    bool close = false;
    if (BIAS) {
      if (k0 + 31 - start <= -a.R) add = far_lo;
      else if (k0 - (start + a.Tq - 1) >= a.R) add = far_hi;
      else {
        close = true;
        const int w = 31 + a.Tq;
        for (int e = lane; e < a.G * w; e += 64) near[e] = bias_at<T>(a, kvh * a.G + e / w, k0 - (start + a.Tq - 1) + e % w);
      }
    }
    const char* tile = mem;
    if (MAPS == 1) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(VP) : "memory");  // K is there; V, issued behind it, may be on its way
    } else {
      MAPATTN_WAIT_DMA();
      __syncthreads();
      if (more) {
        issue_k(t + a.kw, mem + ((it + 1) & 1) * STAGE);
        issue_v(t + a.kw, mem + ((it + 1) & 1) * STAGE);
      }
      if (t >= t1) continue;
      tile = mem + (it & 1) * STAGE;
    }
    f32x16 s[1] = {zero16()};
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) s[0] = Num<T>::mfma(kr.get(tile + m * K_BYTES, 0, kk), qf[kk], s[0]);
    if (MAPS == 1) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K is read: its place may be filled again
      if (more) issue_k(t + a.kw, mem);
    }
    if (BIAS && close) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[0][r] = fmaf(s[0][r], mul, nq[acc_row(r)]);
      mul = 1.f;
    }
    if (k0 + 31 >= len || (a.causal && k0 + 31 > start)) {
      const int dl = lim - k0 - 4 * h;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[0][r] = acc_row(r) > dl ? -INFINITY : s[0][r];
    }
    u32x4 p[1][2];
    soft_step<T, NT, 1>(s, mul, add, mrun, lrun, o, p);
    if (MAPS == 1) {
      if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(KP) : "memory");
      else MAPATTN_WAIT_DMA();
    }
#pragma unroll
    for (int kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) o[nt] = Num<T>::mfma(vr.get(tile + MAPS * K_BYTES, kb2, nt), p[0][kb2], o[nt]);
    if (MAPS == 1) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (more) issue_v(t + a.kw, mem);
    }
  }
  lrun = xor32_sum(lrun);

  // ---- join the teams of a problem: team 0 adds the others' results scaled to the common maximum ---------------------------
  if (a.kw > 1) {
    float* jo = (float*)smem;
    float* jm = jo + (a.teams - 1) * MAPS * OW;
    __syncthreads();  // all tiles read
    if (kwi > 0) {
      const int w = (kwi - 1) * MAPS + m;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 16; ++r) jo[w * OW + (nt * 16 + r) * 64 + lane] = o[nt][r];
      jm[w * 128 + lane] = mrun;
      jm[w * 128 + 64 + lane] = lrun;
    }
    __syncthreads();
    if (kwi == 0) {
      float all = mrun;
      for (int i = 0; i < a.teams - 1; ++i) all = fmaxf(all, jm[(i * MAPS + m) * 128 + lane]);
      const float base = all == -INFINITY ? 0.f : all;
      float f = __builtin_amdgcn_exp2f(mrun - base);
      lrun *= f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[nt][r] *= f;
      for (int i = 0; i < a.teams - 1; ++i) {
        const int w = i * MAPS + m;
        f = __builtin_amdgcn_exp2f(jm[w * 128 + lane] - base);
        lrun += f * jm[w * 128 + 64 + lane];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[nt][r] += f * jo[w * OW + (nt * 16 + r) * 64 + lane];
      }
      mrun = all;
    }
  }
  const bool none = lrun == 0.f;
  const float inv = none ? 0.f : 1.0f / lrun;
  const float lse2 = none ? -INFINITY : mrun + __builtin_amdgcn_logf(lrun);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[nt][r] *= inv;
  const int64_t row = ((int64_t)b * a.Tq + qi) * a.H + head;
  if (MAPS == 2 && a.splits == 1) {
    float* x = (float*)smem + team * OW + lane;
    __syncthreads();  // tiles and joined results read
    if (m == 1 && mine) {
      const float lam = a.lam[head];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[(nt * 16 + r) * 64] = o[nt][r] * lam;
    }
    __syncthreads();
    if (m == 0)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[nt][r] -= x[(nt * 16 + r) * 64];
  }
  if (!mine || kwi > 0) return;
  if (a.splits > 1) {
    const int64_t at = ((int64_t)split * a.B * a.Tq * a.H + row) * MAPS + m;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        const int c0 = nt * 32 + rq * 8 + h * 4;
        if (c0 < a.dv) *(f32x4*)(a.part_o + at * a.dv + c0) = f32x4{o[nt][4 * rq], o[nt][4 * rq + 1], o[nt][4 * rq + 2], o[nt][4 * rq + 3]};
      }
    if (h == 0) a.part_l[at] = lse2;
    return;
  }
  if (a.lse && h == 0) a.lse[((int64_t)(b * a.H + head) * MAPS + m) * a.Tq + qi] = lse2 * LN2;
  char* op = (char*)(m == 0 ? a.out : a.out2);
  if (op == nullptr) return;
  op += row * a.dv * 2;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      const int c0 = nt * 32 + rq * 8 + h * 4;
      if (c0 < a.dv) *(u32x2*)(op + c0 * 2) = u32x2{Num<T>::pack(o[nt][4 * rq], o[nt][4 * rq + 1]), Num<T>::pack(o[nt][4 * rq + 2], o[nt][4 * rq + 3])};
    }
}

// ---- joins the parts of a split forward: o = sum_s 2^(l_s - l) o_s, l = log2 sum_s 2^l_s -----------------------------------------
// Up to PARTS of them: LR lanes of 4 channels per row.  More (PARTS = 0): a wave per row; lane s holds the weight of parts s, s + 64,
// ..; 64 / LR parts are added at once by LR lanes of 4 channels each.  Bound by latency: rows are few and each load is some 600 ns
// away, so all loads of a row, of both maps (of many parts, the first 8 steps'), are on their way before the first weight is needed.
template <typename T, int MAPS, int LR, int PARTS>
__global__ __launch_bounds__(256) void mapattn_combine_kernel(const MapAttnArgs a) {
  constexpr bool SHORT = PARTS > 0;
  constexpr int PG = 64 / LR, MW = 4, N = SHORT ? PARTS : 8;  // parts at once; weights of a lane (256 parts at most); loads in flight
  const int64_t rows = (int64_t)a.B * a.Tq * a.H;
  const int lane = threadIdx.x & 63, c0 = (lane % LR) * 4, sg = SHORT ? 0 : lane / LR;
  const int64_t row = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / (SHORT ? LR : 64);
  if (row >= rows) return;
  constexpr int NW = SHORT ? N : MW;
  float lw[MAPS][NW], x[MAPS][4], lse2[MAPS];
  f32x4 v[MAPS][N];
  auto load = [&](int m, int s) {
    f32x4 r = {0.f, 0.f, 0.f, 0.f};
    if (s < a.splits && c0 < a.dv) r = *(const f32x4*)(a.part_o + (((int64_t)s * rows + row) * MAPS + m) * a.dv + c0);
    return r;
  };
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const int s = SHORT ? i : lane + 64 * i;
      lw[m][i] = s < a.splits ? a.part_l[((int64_t)s * rows + row) * MAPS + m] : -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < N; ++k) v[m][k] = load(m, SHORT ? k : k * PG + sg);
  }
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    float mx = lw[m][0];
#pragma unroll
    for (int i = 1; i < NW; ++i) mx = fmaxf(mx, lw[m][i]);
    if (!SHORT) mx = wave_max(mx);
    const float base = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      lw[m][i] = __builtin_amdgcn_exp2f(lw[m][i] - base);
      sum += lw[m][i];
    }
    if (!SHORT) sum = wave_sum(sum);
    const bool none = sum == 0.f;
    const float inv = none ? 0.f : 1.0f / sum;
    lse2[m] = none ? -INFINITY : base + __builtin_amdgcn_logf(sum);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](float w, const f32x4& p) {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(w, p[e], acc[e]);
    };
    if (SHORT) {
#pragma unroll
      for (int k = 0; k < N; ++k) add(lw[m][k % NW], v[m][k]);
    } else {
      // (64 parts are a whole number of steps, and a part behind the last is zeros)
#pragma unroll
      for (int i = 0; i < MW; ++i) {
        for (int s0 = 0; s0 < 64 && 64 * i + s0 < a.splits; s0 += N * PG) {
          if (i + s0 > 0) {
#pragma unroll
            for (int k = 0; k < N; ++k) v[m][k] = load(m, 64 * i + s0 + k * PG + sg);
          }
#pragma unroll
          for (int k = 0; k < N; ++k) add(__shfl(lw[m][i % NW], s0 + k * PG + sg, 64), v[m][k]);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float t = acc[e];
      if (!SHORT) {
#pragma unroll
        for (int o = LR; o < 64; o <<= 1) t += __shfl_xor(t, o, 64);
      }
      x[m][e] = t * inv;
    }
  }
  const int head = (int)(row % a.H);
  const int64_t bt = row / a.H;
  if (a.lse && sg == 0 && c0 == 0) {
    const int64_t b = bt / a.Tq, qi = bt - b * a.Tq;
#pragma unroll
    for (int m = 0; m < MAPS; ++m) a.lse[((b * a.H + head) * MAPS + m) * a.Tq + qi] = lse2[m] * LN2;
  }
  if (sg != 0 || c0 >= a.dv) return;
  if (MAPS == 2) {
    if (a.out2) *(u32x2*)((char*)a.out2 + (row * a.dv + c0) * 2) = u32x2{Num<T>::pack(x[MAPS - 1][0], x[MAPS - 1][1]), Num<T>::pack(x[MAPS - 1][2], x[MAPS - 1][3])};
    const float lam = a.lam[head];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[0][e] -= lam * x[MAPS - 1][e];
  }
  *(u32x2*)((char*)a.out + (row * a.dv + c0) * 2) = u32x2{Num<T>::pack(x[0][0], x[0][1]), Num<T>::pack(x[0][2], x[0][3])};
}

// ---- dispatch -----------------------------------------------------------------------------------------------------------
namespace {

constexpr int fwd_groups(int maps, int nt) { return maps == 1 || nt >= 8 ? 4 : 2; }

template <typename T, int MAPS, int KS, int NT>
int run_fwd(const MapAttnArgs& a, hipStream_t s) {
  // One map: 128 queries, 64 keys between two maxima (32: 102 us against 94 at 2 x 4096, 8 heads of 40; two waves per 32 queries
  // on alternating keys, twice the waves, 93).  Two maps: small workgroups of 64 queries and tiles of 32 keys, three to a CU and
  // each in its own phase (487 us against 527 - 583 with 128 queries or 64 keys at 8192 causal, 16 heads of 64 + 64); the widest
  // heads' accumulators allow two waves per SIMD either way (237 us against 242 at 2 x 4096 causal, 8 heads of 128 + 128).
  constexpr bool WIDE = NT >= 8;
  constexpr int KT = (MAPS == 1 || WIDE) ? 64 : 32, NS = MAPS == 1 ? 2 : 1, QG = fwd_groups(MAPS, NT);
  constexpr int KCH = 4 * ((KS + 1) / 2), VCH = 4 * NT;
  constexpr int tiles = 2 * KT * 16 * (MAPS * KCH + VCH), hand = MAPS == 2 ? QG * NT * 16 * 64 * 4 : 0;
  const int lds = (tiles > hand ? tiles : hand) + (MAPS == 1 ? (2 * (a.R + 32 * QG + KT) + 1) * 4 : 0);
  const void* f = (const void*)mapattn_fwd_kernel<T, MAPS, KS, NT, KT, NS, QG>;
  if (anip_raise_lds_limit(f, lds) != 0) {
    anip_set_error("mapattn forward: cannot raise the dynamic LDS limit to %d bytes", lds);
    return -2;
  }
  const int nqb = (a.Tq + 32 * QG - 1) / (32 * QG);
  const unsigned grid = mapattn_grid("mapattn_fwd_kernel", (int64_t)nqb * a.splits * a.B * a.H, 64 * QG * MAPS);
  if (!grid) return -1;
  hipLaunchKernelGGL((mapattn_fwd_kernel<T, MAPS, KS, NT, KT, NS, QG>), dim3(grid), dim3(64 * QG * MAPS), lds, s, a);
  ANIP_LAUNCH_CHECK("mapattn_fwd_kernel");
  return 0;
}

// LDS of a team without the near bias, and the most teams of a workgroup: eight waves, fewer where the CU's LDS does not hold them
constexpr int token_team_lds(int maps, int ks, int nt) { return maps * 32 * 16 * (maps * 4 * ((ks + 1) / 2) + 4 * nt); }
constexpr int token_max_teams(int maps, int ks, int nt) {
  const int fit = 160 * 1024 / (token_team_lds(maps, ks, nt) + (maps == 1 ? 4096 : 0)), most = maps == 1 ? 8 : 4;
  return fit < most ? fit : most;
}

template <typename T, int MAPS, int KS, int NT>
int run_token(const MapAttnArgs& a0, hipStream_t s) {
  constexpr int MAXT = token_max_teams(MAPS, KS, NT), OW = NT * 16 * 64 * 4;
  MapAttnArgs a = a0;
  a.teams = MAXT;  // (4 of 8 teams to a workgroup at one each: 20.2 us against 19.2 at 1024 x 24, 8 heads of 40)
  if (a.kw > 1) a.kw = a.teams;
  const int tiles = a.teams * (token_team_lds(MAPS, KS, NT) + (MAPS == 1 ? a.G * (31 + a.Tq) * 4 : 0));
  const int join = a.kw > 1 ? (a.teams - 1) * MAPS * (OW + 512) : 0, hand = MAPS == 2 ? a.teams * OW : 0;
  const int lds = tiles > join ? (tiles > hand ? tiles : hand) : (join > hand ? join : hand);
  static_assert(MAXT >= 2 && (MAXT - 1) * MAPS * (OW + 512) <= 160 * 1024 && MAXT * (token_team_lds(MAPS, KS, NT) + (MAPS == 1 ? 4096 : 0)) <= 160 * 1024, "LDS of a CU");
  const void* f = (const void*)mapattn_token_kernel<T, MAPS, KS, NT, MAXT>;
  if (anip_raise_lds_limit(f, lds) != 0) {
    anip_set_error("mapattn token: cannot raise the dynamic LDS limit to %d bytes", lds);
    return -2;
  }
  const int ppb = a.teams / a.kw;
  const unsigned grid = mapattn_grid("mapattn_token_kernel", cdiv64((int64_t)a.B * a.Hkv * a.splits, ppb), 64 * a.teams * MAPS);
  if (!grid) return -1;
  hipLaunchKernelGGL((mapattn_token_kernel<T, MAPS, KS, NT, MAXT>), dim3(grid), dim3(64 * a.teams * MAPS), lds, s, a);
  ANIP_LAUNCH_CHECK("mapattn_token_kernel");
  return 0;
}

template <typename T, int MAPS, int LR>
int run_combine_lr(const MapAttnArgs& a, hipStream_t s) {
  // (up to 16 parts by LR lanes: 4.9 us at 128 rows x 16, two maps, 7 by a wave; with room for 16 where there are 2: 10.8 at 29 688
  // rows, 7.4 with 8.  Workgroups of one wave where rows are few: 16 parts by waves, 7 us against 7.8)
  const int64_t rows = (int64_t)a.B * a.Tq * a.H;
  const int64_t lanes = rows * (a.splits <= 16 ? LR : 64);
  const int threads = lanes <= 32768 ? 64 : 256;
  const unsigned grid = mapattn_grid("mapattn_combine_kernel", cdiv64(lanes, threads), threads);
  if (!grid) return -1;
  if (a.splits <= 8) hipLaunchKernelGGL((mapattn_combine_kernel<T, MAPS, LR, 8>), dim3(grid), dim3(threads), 0, s, a);
  else if (a.splits <= 16) hipLaunchKernelGGL((mapattn_combine_kernel<T, MAPS, LR, 16>), dim3(grid), dim3(threads), 0, s, a);
  else hipLaunchKernelGGL((mapattn_combine_kernel<T, MAPS, LR, 0>), dim3(grid), dim3(threads), 0, s, a);
  ANIP_LAUNCH_CHECK("mapattn_combine_kernel");
  return 0;
}
template <typename T, int MAPS>
int run_combine(const MapAttnArgs& a, hipStream_t s) {
  return a.dv <= 64 ? run_combine_lr<T, MAPS, 16>(a, s) : a.dv <= 128 ? run_combine_lr<T, MAPS, 32>(a, s) : run_combine_lr<T, MAPS, 64>(a, s);
}

#define TRY1(KS, NT) if (ks <= KS) return run<T, 1, KS, NT>(a, s);
#define TRY2(KS, NT) if (ks <= KS) return run<T, 2, KS, NT>(a, s);
template <typename T>
int fwd_t(const MapAttnArgs& a, int maps, hipStream_t s) {
  const int ks = (a.d + 15) / 16;
#define run run_fwd
  if (maps == 1) { MAPATTN_GEOS_1(TRY1) } else { MAPATTN_GEOS_2(TRY2) }
#undef run
  return -1;
}
template <typename T>
int token_t(const MapAttnArgs& a, int maps, hipStream_t s) {
  const int ks = (a.d + 15) / 16;
#define run run_token
  if (maps == 1) { MAPATTN_GEOS_1(TRY1) } else { MAPATTN_GEOS_2(TRY2) }
#undef run
  return -1;
}

}  // namespace

int mapattn_forward(const MapAttnArgs& a, int maps, int bf16, hipStream_t s) { return bf16 ? fwd_t<bf16_t>(a, maps, s) : fwd_t<f16>(a, maps, s); }
int mapattn_token(const MapAttnArgs& a, int maps, int bf16, hipStream_t s) { return bf16 ? token_t<bf16_t>(a, maps, s) : token_t<f16>(a, maps, s); }
int mapattn_combine(const MapAttnArgs& a, int maps, int bf16, hipStream_t s) {
  if (maps == 1) return bf16 ? run_combine<bf16_t, 1>(a, s) : run_combine<f16, 1>(a, s);
  return bf16 ? run_combine<bf16_t, 2>(a, s) : run_combine<f16, 2>(a, s);
}
