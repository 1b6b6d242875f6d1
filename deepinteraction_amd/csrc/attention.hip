// Entry points of the attention to another sequence (attention.h, attention_fwd.h, attention_bwd.h): checks, plans, dispatch.
// Reference: the decoder layer's attention to the BEV map (decoder_utils.py:96-103, :421-485), the RoI blocks' attention among the
// queries of a view (:743-746) and the ray decoder's attention to an image column (fusion_transformerv4.py:715-769).
#include <math.h>

#include "attention_plan.h"

namespace di {
namespace at {

// Blocks, and - where they are fewer than `want` - ranges of the walked side (whole tiles) so that about `want` workgroups run: at
// least `least` tiles each, or up to `some` ranges whatever their length.
static void cut(Plan &p, long long problems, int rows, int per_block, int walked, int tile, int least, int some, long long want) {
  p.blocks = (rows + per_block - 1) / per_block;
  const long long n = problems * (p.blocks > 0 ? p.blocks : 1);
  const int tiles = walked > 0 ? (int)(((long long)walked + tile - 1) / tile) : 1;
  int most = tiles / least;
  if (most < some) most = some < tiles ? some : tiles;
  long long splits = n > 0 ? want / n : 1;
  if (splits > most) splits = most;
  if (splits < 1) splits = 1;
  const int per = (int)((tiles + splits - 1) / splits);
  p.range = per > 0x7fffffff / tile ? 0x7fffffff : per * tile;
  p.splits = (tiles + per - 1) / per;
}

// Rows per workgroup and ranges of the keys.  Up to 16 rows (single queries): 24 workgroups a CU, the memory streams best through many
// short ranges (16 samples x 8 key heads of 128, up to 32 768 keys, with the join: 8 a CU 246 us, 16 229, 24 220).  More rows: what is
// resident - two workgroups a CU, one for gq of 128 dims (2048 x 8192 x 16 heads of 128, forward: 1 a CU 263 us, 2 211, 3 229; gq: 1 a
// CU 290, 2 317) - and twice that where the samples' lengths differ and some ranges have no keys (4 x 511 x 4100, 2733, 1366, 0, four
// heads of 64 to a key head, forward + gq with their joins: 2 a CU 127 us, 4 95, 6 100, 8 118; four lengths of 1025 .. 4100: 132, 113,
// 119, 128).  Too few row blocks for the CUs, and 16-bit gq of 96 and 128 dims with a mask or dropout (426 x 375 x 127, 8 heads, key mask: 128 rows,
// one a CU, 637 us; 64, two a CU, 554; 2 x 1000 x 4000, 8 heads of 72: 108 and 90; float32 loses, 347 and 416): 64 rows a workgroup, and - heads of up to 32 dims, of which more are resident - eight a CU
// (57 x 20 rows x 19 070, four heads of 24: 564 -> 442; heads of 128 lose, 150 -> 170).  A tile of float32 keys takes 3 - 7 us with 64 and
// 128 dims: up to 16 ranges of single tiles (300 x 300, 8 heads of 64, forward 16.6 -> 7.4 + 4.9 us for the join; 23 x 598 of 128: 34 -> 10 + 5).
// Key lengths: the samples of an unbalanced batch load the XCDs evenly (where_ragged in attention.h) - if there is more than one workgroup
// a CU to place, and no more samples than lanes to look them up.
static bool ragged(const di_attention &t, const Plan &p, int cus) {
  return t.key_lengths != nullptr && t.B <= 64 && (long long)t.B * t.kv_heads * p.blocks * p.splits > cus;
}

// Rows per workgroup, and key tiles per wavefront, of a call that fills the CUs without splitting (the reasons above and in
// attention_plan.h).
static int row_block(const di_attention &t, bool forward) {
  const int DP = padded(t.head_dim);
  const long long rows = (long long)(t.heads / t.kv_heads) * t.L;
  const bool full = t.key_mask != nullptr || t.allowed != nullptr || t.dropout_p > 0.f;
  if (rows <= 16) return 16;
  return rows <= 64 || (!forward && DP >= 96 && full && t.dtype != DI_F32) ? 64 : 64 * row_tiles(DP);
}
static int widest_key_tiles(const di_attention &t) {
  const int n = key_tiles(t.dtype, padded(t.head_dim));
  return (t.allowed != nullptr || t.dropout_p > 0.f) && n > most_masked_key_tiles ? most_masked_key_tiles : n;
}

static int plan_rows(const di_attention &t, bool forward, Plan &p) {
  const int cus = device_cus();
  if (cus <= 0) return DI_ERR_LAUNCH;
  const int DP = padded(t.head_dim), rows = t.heads / t.kv_heads * t.L, block = row_block(t, forward);
  const long long problems = (long long)t.B * t.kv_heads;
  if (block == 16) {
    p.big = 0;
    cut(p, problems, rows, 16, t.S, t.dtype != DI_F32 ? 128 : 64, 4, 1, 24ll * cus);
    p.ragged = ragged(t, p, cus);
    return DI_OK;
  }
  const bool wide = !forward && DP == 128;
  const long long want = 2ll * cus * (t.key_lengths != nullptr ? 2 : 1);
  const int some = t.dtype == DI_F32 && DP >= 64 ? 16 : 1;
  p.big = 2;
  cut(p, problems, rows, 64 * row_tiles(DP), t.S, 64, 4, some, wide ? want / 2 : want);
  if (block == 64 || problems * p.blocks * p.splits < cus) {
    p.big = 1;
    cut(p, problems, rows, 64, t.S, 64, 4, some, DP <= 32 ? 4 * want : want);
  }
  p.ragged = ragged(t, p, cus);
  return DI_OK;
}

static int plan_keys(const di_attention &t, Plan &p) {
  const int cus = device_cus();
  if (cus <= 0) return DI_ERR_LAUNCH;
  const int DP = padded(t.head_dim), rows = t.heads / t.kv_heads * t.L, least = least_key_tiles(DP);
  const int tile = tile_rows(t.dtype, DP);
  const long long problems = (long long)t.B * t.kv_heads;
  const int S = t.S > 0 ? t.S : 1;                              // without keys, one block still writes gq's zeros
  p.big = widest_key_tiles(t);
  for (; p.big > least; p.big /= 2) {   // the largest key block that the keys fill, and that leaves work for all
    if (32 * p.big >= t.S) continue;
    cut(p, problems, S, 64 * p.big, rows, tile, 1, 1, 2ll * cus);
    if (problems * p.blocks * p.splits >= cus) break;
  }
  if (p.big <= least) cut(p, problems, S, 64 * p.big, rows, tile, 1, 1, 2ll * cus);
  p.ragged = ragged(t, p, cus);
  return DI_OK;
}

// A launch has fewer than 2^32 work-items, 256 a workgroup.  Only calls of more workgroups than any plan splits for come near: the blocks
// of the two plans as they are without splits, and the join of narrow heads' gq over the key blocks.
static bool fits(const di_attention &t, bool forward) {
  const int DP = padded(t.head_dim);
  const long long problems = (long long)t.B * t.kv_heads, rows = (long long)(t.heads / t.kv_heads) * t.L, most = (1 << 24) - 1;
  const int per = row_block(t, forward);
  if ((forward || !one_launch(DP)) && problems * ((rows + per - 1) / per) > most) return false;
  if (forward) return true;
  int big = widest_key_tiles(t);
  while (big > least_key_tiles(DP) && 32 * big >= t.S) big /= 2;
  const long long blocks = t.S > 0 ? ((long long)t.S + 64 * big - 1) / (64 * big) : 1;
  if (problems * blocks > most) return false;
  return !one_launch(DP) || blocks == 1 || problems * join_shape(t.head_dim, (int)blocks, (int)rows).blocks <= most;
}

// floats of the backward's workspace: delta | the sums of gq | the sums of gk and gv.  Two launches: gq's are joined before the others
// are written.
struct Room {
  long long gq, gkv;
};
static Room room_of(const di_attention &t, const Plan &p, const Plan &k) {
  const long long rows = (long long)t.B * t.heads * t.L, keys = (long long)t.B * t.kv_heads * t.S;
  const int n = one_launch(padded(t.head_dim)) ? k.blocks : p.splits;
  Room r;
  r.gq = n > 1 ? n * rows * t.head_dim : 0;
  r.gkv = k.splits > 1 ? 2ll * k.splits * keys * t.head_dim : 0;
  return r;
}

static bool aligned(const void *p, long long bs, long long rs, int size) {
  // a tile's rows (128 at the most) are addressed with 32 bits from its first
  return ((uintptr_t)p & 15) == 0 && (bs * size) % 16 == 0 && (rs * size) % 16 == 0 && rs >= 0 && rs * size < (1ll << 24);
}

static int check(const di_attention *t, bool forward) {
  DI_REQUIRE(t != nullptr, "attention: null pointer");
  DI_REQUIRE(t->dtype == DI_F32 || t->dtype == DI_F16 || t->dtype == DI_BF16, "attention: unsupported dtype %d", t->dtype);
  DI_REQUIRE(t->B >= 0 && t->L >= 0 && t->S >= 0, "attention: negative size");
  DI_REQUIRE(t->heads > 0 && t->kv_heads > 0 && t->heads % t->kv_heads == 0, "attention: %d query heads, %d key heads", t->heads, t->kv_heads);
  DI_REQUIRE(t->head_dim > 0 && t->head_dim % 8 == 0 && t->head_dim <= 128, "attention: head_dim %d (a multiple of 8, at most 128)", t->head_dim);
  DI_REQUIRE(t->scale > 0.f && isfinite(t->scale), "attention: the scale must be positive and finite");
  DI_REQUIRE(t->dropout_p >= 0.f && t->dropout_p < 1.f, "attention: dropout probability %f", (double)t->dropout_p);
  const long long rows = (long long)(t->heads / t->kv_heads) * t->L;
  DI_REQUIRE(rows <= 0x3fffffff && t->S <= 0x3fffffff, "attention: more than 2^30 rows or keys");
  DI_REQUIRE(fits(*t, forward), "attention: too many rows or keys for one launch (2^24 workgroups)");
  const int sz = t->dtype == DI_F32 ? 4 : 2;
  // rows of the output - and of the keys' gradients - are addressed as those of the inputs
  DI_REQUIRE((long long)t->heads * t->head_dim * sz < (1ll << 24), "attention: %d heads of %d (rows of 16 MB and more)", t->heads, t->head_dim);
  if (t->B == 0) return DI_OK;
  DI_REQUIRE(t->L == 0 || (t->q != nullptr && aligned(t->q, t->q_bs, t->q_rs, sz)), "attention: q must start and step on 16 bytes, its rows less than 16 MB apart");
  DI_REQUIRE(t->S == 0 || (t->k != nullptr && t->v != nullptr && aligned(t->k, t->k_bs, t->k_rs, sz) && aligned(t->v, t->v_bs, t->v_rs, sz)),
             "attention: k and v must start and step on 16 bytes, their rows less than 16 MB apart");
  return DI_OK;
}

// The rows of grad_k or grad_v in memory (in elements): `nin` rows `in` apart, `nout` groups of them `out` apart.
struct Rows {
  long long low, in, nin, out, nout, E;                         // low: the first byte's address
  long long group() const { return (nin - 1) * in + E; }
  long long span() const { return (nout - 1) * out + group(); }
  // each row is written once (nested groups; other layouts without an overlap exist, and are refused with the rest)
  bool apart() const { return (nin == 1 || in >= E) && (nout == 1 || out >= group()); }
};
static Rows rows_of(const di_attention &t, const void *p, long long bs, long long rs, int sz) {
  const long long step = bs < 0 ? -bs : bs;
  Rows r = {(long long)(uintptr_t)p + (bs < 0 ? (t.B - 1) * bs * sz : 0), rs, t.S, step, t.B, (long long)t.kv_heads * t.head_dim};
  if (t.S > 1 && t.B > 1 && step < rs) r = {r.low, step, t.B, rs, t.S, r.E};
  return r;
}
// ... and not by the other gradient: one behind the other, or one's rows, or groups, between the other's of the same strides
static bool clear_of(const Rows &a, const Rows &b, int sz) {
  const Rows &lo = a.low <= b.low ? a : b, &hi = a.low <= b.low ? b : a;
  const long long by = hi.low - lo.low;
  if (by >= lo.span() * sz) return true;
  const bool same = (a.nin == 1 || a.in == b.in) && (a.nout == 1 || a.out == b.out) && a.nin == b.nin;
  const bool rows = by >= a.E * sz && (a.nin == 1 || by + a.E * sz <= a.in * sz) && (a.nout == 1 || by + a.group() * sz <= a.out * sz);
  const bool groups = by >= a.group() * sz && (a.nout == 1 || by + a.group() * sz <= a.out * sz);
  return same && (rows || groups);
}

static Args args_of(const di_attention *t, const unsigned long long *seed_word) {
  Args a = {};
  const int sz = t->dtype == DI_F32 ? 4 : 2;
  a.q = (const char *)t->q; a.k = (const char *)t->k; a.v = (const char *)t->v;
  a.q_bs = t->q_bs * sz; a.q_rs = t->q_rs * sz;
  a.k_bs = t->k_bs * sz; a.k_rs = t->k_rs * sz;
  a.v_bs = t->v_bs * sz; a.v_rs = t->v_rs * sz;
  a.klen = t->key_lengths;
  if (t->S > 0) {                                              // no keys: nothing that a mask could exclude
    a.kmask = t->key_mask; a.kmask_bs = t->key_mask_bs;
    a.allowed = t->allowed; a.allowed_bs = t->allowed_bs; a.allowed_rs = t->allowed_rs;
  }
  a.B = t->B; a.L = t->L; a.S = t->S; a.Hk = t->kv_heads; a.G = t->heads / t->kv_heads; a.D = t->head_dim;
  a.scale = t->scale;
  a.scale2 = t->scale * kLog2e;
  a.drop = (unsigned)(t->dropout_p * 65536.f + 0.5f);
  if (a.drop > 65535u) a.drop = 65535u;
  a.keep_scale = 65536.f / (float)(65536u - a.drop);
  a.seed = t->seed;
  a.seed_ptr = seed_word;
  return a;
}

}  // namespace at
}  // namespace di

extern "C" {

long long di_attention_fwd_workspace_floats(const di_attention *t) {
  using namespace di::at;
  if (check(t, true) != DI_OK) return -1;
  Plan p;
  if (plan_rows(*t, true, p) != DI_OK) return -1;
  return p.splits == 1 ? 0 : (long long)p.splits * t->B * t->heads * t->L * (t->head_dim + 2);
}

long long di_attention_bwd_workspace_floats(const di_attention *t) {
  using namespace di::at;
  if (check(t, false) != DI_OK) return -1;
  Plan p, k;
  if (plan_rows(*t, false, p) != DI_OK || plan_keys(*t, k) != DI_OK) return -1;
  const Room r = room_of(*t, p, k);
  return ((long long)t->B * t->heads * t->L + 3) / 4 * 4 + r.gq + r.gkv;
}

int di_attention_fwd(const di_attention *t, void *out, float *lse, float *workspace, void *stream) {
  return di_attention_fwd_seeded(t, di::i2p_seed_ptr(), out, lse, workspace, stream);
}

int di_attention_fwd_seeded(const di_attention *t, const unsigned long long *seed_word, void *out, float *lse, float *workspace, void *stream) {
  using namespace di::at;
  if (int rc = check(t, true)) return rc;
  if (t->B == 0 || t->L == 0) return DI_OK;
  DI_REQUIRE(out != nullptr && ((uintptr_t)out & 15) == 0, "attention: the output must start on 16 bytes");
  Plan p;
  if (int rc = plan_rows(*t, true, p)) return rc;
  Args a = args_of(t, seed_word);
  a.o = (char *)out;
  a.lse = lse;
  if (p.splits > 1) {
    DI_REQUIRE(workspace != nullptr && ((uintptr_t)workspace & 15) == 0, "attention: workspace");
    a.part = workspace;
    a.part_ml = workspace + (long long)p.splits * t->B * t->heads * t->L * t->head_dim;
  }
  hipStream_t s = (hipStream_t)stream;
  return t->dtype == DI_F32 ? launch_fwd<DI_F32>(a, p, s) : t->dtype == DI_F16 ? launch_fwd<DI_F16>(a, p, s) : launch_fwd<DI_BF16>(a, p, s);
}

int di_attention_bwd(const di_attention *t, const void *out, const float *lse, const void *grad_out, long long go_bs, long long go_rs,
                     void *gq, void *gk, long long gk_bs, long long gk_rs, void *gv, long long gv_bs, long long gv_rs, float *workspace,
                     void *stream) {
  return di_attention_bwd_seeded(t, di::i2p_seed_ptr(), out, lse, grad_out, go_bs, go_rs, gq, gk, gk_bs, gk_rs, gv, gv_bs, gv_rs, workspace, stream);
}

int di_attention_bwd_seeded(const di_attention *t, const unsigned long long *seed_word, const void *out, const float *lse, const void *grad_out,
                            long long go_bs, long long go_rs, void *gq, void *gk, long long gk_bs, long long gk_rs, void *gv, long long gv_bs,
                            long long gv_rs, float *workspace, void *stream) {
  using namespace di::at;
  if (int rc = check(t, false)) return rc;
  if (t->B == 0 || (t->L == 0 && t->S == 0)) return DI_OK;
  const int sz = t->dtype == DI_F32 ? 4 : 2;
  DI_REQUIRE(t->L == 0 || (out && lse && grad_out && gq && ((uintptr_t)out & 15) == 0 && ((uintptr_t)gq & 15) == 0 && aligned(grad_out, go_bs, go_rs, sz)),
             "attention: out, grad_out and grad_q must start (and grad_out step) on 16 bytes");
  DI_REQUIRE(t->S == 0 || (gk && gv && aligned(gk, gk_bs, gk_rs, sz) && aligned(gv, gv_bs, gv_rs, sz)),
             "attention: grad_k and grad_v must start and step on 16 bytes");
  const Rows rk = rows_of(*t, gk, gk_bs, gk_rs, sz), rv = rows_of(*t, gv, gv_bs, gv_rs, sz);
  DI_REQUIRE(t->S == 0 || (rk.apart() && rv.apart()), "attention: rows of grad_k or grad_v overlap");
  DI_REQUIRE((workspace != nullptr || t->L == 0) && ((uintptr_t)workspace & 15) == 0, "attention: workspace");   // no rows: one range, no sums
  DI_REQUIRE(t->S == 0 || clear_of(rk, rv, sz), "attention: grad_k and grad_v overlap");
  Plan p, k;
  if (int rc = plan_rows(*t, false, p)) return rc;
  if (int rc = plan_keys(*t, k)) return rc;
  Args a = args_of(t, seed_word);
  a.o = (char *)const_cast<void *>(out);
  a.lse = const_cast<float *>(lse);
  a.go = (const char *)grad_out;
  a.go_bs = go_bs * sz; a.go_rs = go_rs * sz;
  a.gq = (char *)gq; a.gk = (char *)gk; a.gv = (char *)gv;
  a.gk_bs = gk_bs * sz; a.gk_rs = gk_rs * sz; a.gv_bs = gv_bs * sz; a.gv_rs = gv_rs * sz;
  a.delta = workspace;
  a.part = workspace + ((long long)t->B * t->heads * t->L + 3) / 4 * 4;
  a.part_k = a.part + room_of(*t, p, k).gq;
  a.part_v = a.part_k + (long long)k.splits * t->B * t->kv_heads * t->S * t->head_dim;
  hipStream_t s = (hipStream_t)stream;
  return t->dtype == DI_F32   ? launch_bwd<DI_F32>(a, p, k, s)
         : t->dtype == DI_F16 ? launch_bwd<DI_F16>(a, p, k, s)
                              : launch_bwd<DI_BF16>(a, p, k, s);
}

}  // extern "C"
