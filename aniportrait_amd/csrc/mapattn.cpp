// C entry points of the attention of mapattn.h: checks, workspaces, and which kernel a call takes.
#include "mapattn.h"

namespace {

constexpr int MAX_R = 4096;  // reach of the learned bias: 2 R + 1 floats of it lie in LDS

int check(const char* what, const anip_attn_params* p, int maps, bool backward) {
  ANIP_REQUIRE(p != nullptr, "%s: NULL parameters", what);
  ANIP_REQUIRE(p->dtype == 0 || p->dtype == 1, "%s: dtype must be 0 (fp16) or 1 (bf16)", what);
  ANIP_REQUIRE(p->B >= 1 && p->Tq >= 1 && p->Tk >= 1 && p->H >= 1 && p->Hkv >= 1, "%s: sizes must be positive", what);
  ANIP_REQUIRE(p->H % p->Hkv == 0, "%s: %d query heads do not divide into %d key heads", what, p->H, p->Hkv);
  ANIP_REQUIRE(p->Tq <= (1 << 28) && p->Tk <= (1 << 28), "%s: sequences are longer than 2^28", what);
  ANIP_REQUIRE(p->H <= (1 << 20) && (int64_t)p->B * p->H < (1ll << 31), "%s: too many heads", what);
  const int dmax = maps == 1 ? 160 : 128;
  ANIP_REQUIRE(p->d >= 8 && p->d <= dmax && p->d % 8 == 0, "%s: head width %d: a multiple of 8 up to %d is wanted", what, p->d, dmax);
  ANIP_REQUIRE(p->scale > 0.f && p->scale < 1e30f, "%s: scale must be positive and finite", what);
  struct Side {
    const char* name;
    const void* x;
    const int64_t* s;
    int T;
  } sides[4] = {{"q", p->q, p->q_stride, p->Tq}, {"k", p->k, p->k_stride, p->Tk}, {"v", p->v, p->v_stride, p->Tk}, {"dout", p->dout, p->dout_stride, p->Tq}};
  for (int i = 0; i < (backward ? 4 : 3); ++i) {
    const Side& t = sides[i];
    ANIP_REQUIRE(t.x != nullptr && ((uintptr_t)t.x & 15) == 0, "%s: %s must be a 16-byte aligned device pointer", what, t.name);
    ANIP_REQUIRE(t.s[0] % 8 == 0 && t.s[1] % 8 == 0 && t.s[2] % 8 == 0, "%s: %s: strides must be multiples of 8 elements", what, t.name);
    ANIP_REQUIRE(t.T == 1 || (t.s[1] >= 0 && t.s[1] < (1 << 24)), "%s: %s: the distance between tokens must be below 2^24 elements", what, t.name);
  }
  ANIP_REQUIRE(p->out != nullptr && (((uintptr_t)p->out | (uintptr_t)p->out2) & 15) == 0, "%s: out and out2 must be 16-byte aligned device pointers", what);
  if (maps == 1) {
    ANIP_REQUIRE(p->table != nullptr && p->buckets != nullptr && p->n_buckets >= 1, "%s: the bias needs its table and the buckets of the relative positions", what);
    ANIP_REQUIRE(p->max_distance >= 0 && p->max_distance <= MAX_R, "%s: relative positions up to %d can be told apart, %d are asked for", what, MAX_R, p->max_distance);
  } else {
    ANIP_REQUIRE(p->lam != nullptr, "%s: lam is wanted", what);
  }
  if (backward) {
    ANIP_REQUIRE(p->lse != nullptr && p->dq != nullptr && p->dk != nullptr && p->dv != nullptr, "%s: lse, dq, dk and dv are wanted", what);
    ANIP_REQUIRE((((uintptr_t)p->dq | (uintptr_t)p->dk | (uintptr_t)p->dv) & 15) == 0, "%s: dq, dk and dv must be 16-byte aligned", what);
    ANIP_REQUIRE(maps == 1 ? p->dtable != nullptr : (p->dlam != nullptr && p->out2 != nullptr), "%s: %s wanted", what, maps == 1 ? "dtable is" : "out2 and dlam are");
  }
  return 0;
}

// the distance between tokens; of a lone one it may be anything, and any that clears its channels does
int64_t token_stride(int T, const int64_t* s) { return T == 1 ? 256 : s[1]; }

MapAttnArgs args(const anip_attn_params* p, int maps) {
  MapAttnArgs a{};
  a.q = p->q, a.q_sb = p->q_stride[0], a.q_st = token_stride(p->Tq, p->q_stride), a.q_sh = p->q_stride[2];
  a.k = p->k, a.k_sb = p->k_stride[0], a.k_st = token_stride(p->Tk, p->k_stride), a.k_sh = p->k_stride[2];
  a.v = p->v, a.v_sb = p->v_stride[0], a.v_st = token_stride(p->Tk, p->v_stride), a.v_sh = p->v_stride[2];
  a.B = p->B, a.Tq = p->Tq, a.Tk = p->Tk, a.H = p->H, a.Hkv = p->Hkv, a.G = p->H / p->Hkv;
  a.d = p->d, a.dv = p->d * maps, a.causal = p->causal != 0;
  a.scale = p->scale, a.scale_log2 = p->scale * mapattn::LOG2E;
  a.kv_lens = p->kv_lens, a.q_start = p->q_start, a.start0 = p->Tk - p->Tq;
  a.table = p->table, a.buckets = p->buckets, a.NB = p->n_buckets, a.R = p->max_distance;
  a.lam = p->lam;
  a.out = p->out, a.out2 = p->out2, a.lse = p->lse;
  a.splits = 1, a.kw = 1;
  return a;
}

bool few_rows(const anip_attn_params* p) { return (int64_t)p->Tq * (p->H / p->Hkv) <= 32; }

// how the keys are split over workgroups where the queries alone do not fill the chip (256 CUs): towards two workgroups per CU of
// the kernel for many queries (8 tiles of 64 keys at the least for each: 4 x 500, 8 heads of 64 take 12.7 us whole, 17.4 in two), and
// of the single-token kernel (4 of 128)
int splits_of(const anip_attn_params* p) {
  const bool few = few_rows(p);
  const int64_t blocks = few ? (int64_t)p->B * p->Hkv : (int64_t)((p->Tq + 127) / 128) * p->B * p->H;
  const int64_t tiles = few ? (p->Tk + 127) / 128 : (p->Tk + 63) / 64;
  if (blocks * 2 > 512) return 1;
  int64_t s = 512 / blocks;  // (single tokens, 256 and 1024: 33 and 39 us against 29 at 8 x 16384; 59 and 68 against 59 at 16 x 8192)
  const int64_t most = tiles / (few ? 4 : 8);
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : (s > 256 ? 256 : s));
}
int64_t fwd_ws(const anip_attn_params* p, int maps) {
  const int s = splits_of(p);
  return s == 1 ? 0 : (int64_t)s * p->B * p->Tq * p->H * maps * (p->d * maps + 1) * 4;
}

int forward(const char* what, const anip_attn_params* p, int maps, int kid, void* stream) {
  const int rc = check(what, p, maps, false);
  if (rc) return rc;
  MapAttnArgs a = args(p, maps);
  a.splits = splits_of(p);
  const int64_t need = fwd_ws(p, maps);
  ANIP_REQUIRE(need == 0 || (p->workspace != nullptr && ((uintptr_t)p->workspace & 15) == 0 && p->workspace_bytes >= need), "%s: a workspace of %lld bytes is wanted, 16-byte aligned", what, (long long)need);
  if (a.splits > 1) {
    a.part_o = (float*)p->workspace;
    a.part_l = a.part_o + (int64_t)a.splits * p->B * p->Tq * p->H * maps * a.dv;
  }
  hipStream_t s = (hipStream_t)stream;
  AnipProfScope prof_(kid, stream);
  int r;
  if (few_rows(p)) {
    // a team per problem where there are enough of them or few keys, else the workgroup's teams share one
    a.kw = (a.splits == 1 && ((int64_t)p->B * p->Hkv >= 2048 || p->Tk <= 64)) ? 1 : 4;
    r = mapattn_token(a, maps, p->dtype, s);
  } else {
    r = mapattn_forward(a, maps, p->dtype, s);
  }
  if (r || a.splits == 1) return r;
  return mapattn_combine(a, maps, p->dtype, s);
}

// one wave per workgroup on short sequences, which would leave three of four idle
int waves_for(int T) { return T <= 64 ? 1 : 4; }

// Both kernels of the backward walk over tiles of the other side.  The chip holds two workgroups of 4 wave groups per CU (one, with
// two maps or the widest heads); where there are fewer, a walk of 12 tiles or more is split towards that, with 4 at the least for each
// part (whole step at 1 x 1000, 8 heads of 128: 95 us, 114 with 8; at 4 x 500, 8 heads of 64, 8 tiles: 69 split, 62 whole).
int walk_splits(int64_t blocks, int64_t tiles) {
  if (tiles < 12) return 1;
  if (blocks < 1) blocks = 1;
  int64_t s = 512 / blocks;
  s = s < tiles / 4 ? s : tiles / 4;
  return (int)(s < 1 ? 1 : (s > 16 ? 16 : s));
}

struct BwdLayout {
  int nwq, nwk, Tp, QW, ND, DR, parts, qsplits, ksplits;
  int64_t rows, rows3, diag, dlam, part, dkv, dq, sizes, total;  // floats
};
BwdLayout layout(const anip_attn_params* p, int maps) {
  BwdLayout l{};
  l.nwq = waves_for(p->Tq);
  l.nwk = waves_for(p->Tk);
  l.Tp = l.nwq == 1 ? (p->Tq + 63) / 64 * 64 : (p->Tq + 127) / 128 * 128;
  l.QW = (p->Tq + 31) / 32;
  l.rows = (int64_t)p->B * p->H * maps * l.Tp;
  l.qsplits = walk_splits((int64_t)l.Tp / 32 * p->B * p->H / 4, (p->Tk + 63) / 64);
  l.ksplits = walk_splits((int64_t)((p->Tk + 31) / 32) * p->B * p->Hkv / 4, (int64_t)((p->Tq + 63) / 64) * (p->H / p->Hkv));
  if (maps == 1) {
    // the diagonals that exist: queries at the keys' end lie max(Tq, Tk) - 1 from any key; those of q_start may lie anywhere (1024 x 24,
    // 8 heads, reach 4096: 8 MB of sums instead of 275)
    const int far = p->Tq > p->Tk ? p->Tq : p->Tk;
    l.DR = p->q_start != nullptr || p->max_distance < far ? p->max_distance : far;
    l.ND = 2 * l.DR + 2 * mapattn::DIAG_PAD;
    const int64_t groups = (int64_t)p->B * l.QW * l.qsplits;
    l.parts = (int)(groups < 32 ? groups : 32);  // few query groups: their own sums are the parts
    l.diag = (int64_t)p->H * groups * (l.ND + 2);
    l.part = groups > 32 ? (int64_t)p->H * l.parts * (l.ND + 2) : 0;
  } else {
    l.dlam = (int64_t)p->H * p->B * l.QW * l.qsplits;
  }
  if (l.qsplits > 1) l.rows3 = (int64_t)p->H * p->B * l.QW * l.qsplits * (maps == 1 ? 3 : 2) * 32;
  if (l.qsplits > 1) l.dq = (int64_t)l.qsplits * p->B * p->Tq * p->H * maps * p->d;
  if (l.ksplits > 1) l.dkv = (int64_t)l.ksplits * p->B * p->Tk * p->Hkv * 2 * maps * p->d;
  if (p->dtype == 0) l.sizes = (int64_t)p->B * p->H * maps * l.QW * 2;
  l.total = l.dq + l.dkv + 2 * l.rows + l.sizes + l.diag + l.part + l.dlam + l.rows3;
  return l;
}

int backward(const char* what, const anip_attn_params* p, int maps, int kid, void* stream) {
  const int rc = check(what, p, maps, true);
  if (rc) return rc;
  const BwdLayout l = layout(p, maps);
  ANIP_REQUIRE(p->workspace != nullptr && ((uintptr_t)p->workspace & 15) == 0 && p->workspace_bytes >= l.total * 4, "%s: a workspace of %lld bytes is wanted, 16-byte aligned", what, (long long)l.total * 4);
  ANIP_REQUIRE((int64_t)((p->Tq + 31) / 32) * (p->H / p->Hkv) < (1ll << 31), "%s: too many query tiles", what);
  MapAttnArgs a = args(p, maps);
  a.dout = p->dout, a.do_sb = p->dout_stride[0], a.do_st = token_stride(p->Tq, p->dout_stride), a.do_sh = p->dout_stride[2];
  a.dq = p->dq, a.dk = p->dk, a.dvo = p->dv, a.dtable = p->dtable, a.dlam = p->dlam;
  a.Tp = l.Tp, a.QW = l.QW, a.ND = l.ND, a.DR = l.DR, a.parts = l.parts;
  a.part_q = (float*)p->workspace;
  a.part_o = a.part_q + l.dq;
  a.rows_lse = a.part_o + l.dkv;
  a.rows_d = a.rows_lse + l.rows;
  a.sizes = (f32x2*)(a.rows_d + l.rows);  // (each part before it holds a multiple of 8 floats)
  a.diag = a.rows_d + l.rows + l.sizes;
  a.diag_part = l.part ? a.diag + l.diag : a.diag;
  a.dlam_part = a.diag + l.diag + l.part;
  a.rows3 = a.dlam_part + l.dlam;
  hipStream_t s = (hipStream_t)stream;
  AnipProfScope prof_(kid, stream);
  a.splits = a.qsplits = l.qsplits;
  int r = mapattn_dq(a, maps, p->dtype, l.nwq, s);
  a.splits = l.ksplits;
  if (!r) r = mapattn_dkv(a, maps, p->dtype, l.nwk, s);
  return r;
}

}  // namespace

extern "C" int64_t anip_relative_attention_ws_bytes(const anip_attn_params* p, int backward) {
  const int rc = check("anip_relative_attention_ws_bytes", p, 1, false);
  return rc ? rc : (backward ? layout(p, 1).total * 4 : fwd_ws(p, 1));
}
extern "C" int anip_relative_attention(const anip_attn_params* p, void* stream) { return forward("anip_relative_attention", p, 1, ANIP_K_REL_ATTN, stream); }
extern "C" int anip_relative_attention_backward(const anip_attn_params* p, void* stream) { return backward("anip_relative_attention_backward", p, 1, ANIP_K_REL_ATTN, stream); }

extern "C" int64_t anip_differential_attention_ws_bytes(const anip_attn_params* p, int backward) {
  const int rc = check("anip_differential_attention_ws_bytes", p, 2, false);
  return rc ? rc : (backward ? layout(p, 2).total * 4 : fwd_ws(p, 2));
}
extern "C" int anip_differential_attention(const anip_attn_params* p, void* stream) { return forward("anip_differential_attention", p, 2, ANIP_K_DIFF_ATTN, stream); }
extern "C" int anip_differential_attention_backward(const anip_attn_params* p, void* stream) { return backward("anip_differential_attention_backward", p, 2, ANIP_K_DIFF_ATTN, stream); }
