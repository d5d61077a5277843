// bx_ops.hip -- entry points of the dense operators over keypoints (bx_linear, bx_qk_norm_rope, bx_attention): argument checks on the
// host, then the launch.  Nothing here reads device memory or keeps state.
#include "bx_ops.h"
#include <cmath>

namespace {

constexpr long long LEN_MAX = 1LL << 30, EXTENT_MAX = 1LL << 44;

#define OP_REFUSE(cond, ...)                                     \
    do {                                                         \
        if (cond) { bx_set_error(__VA_ARGS__); return BX_ERR_ARG; } \
    } while (0)

int elem_bytes(int dtype) { return dtype == BX_TYPE_F32 ? 4 : 2; }
bool misaligned(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) != 0; }
// a stride that no memory can hold n of (this keeps every offset below inside 64 bits)
bool bad_stride(long long s, long long n) { return s < 0 || (n > 1 && s > EXTENT_MAX / (n - 1)); }

// the bytes that an operand's elements lie in, [lo, hi)
struct Bytes { uintptr_t lo, hi; };
Bytes span(const void* p, int e, long long n0, long long s0, long long n1 = 1, long long s1 = 0, long long n2 = 1, long long s2 = 0, long long n3 = 1)
{
    if (!p || n0 <= 0 || n1 <= 0 || n2 <= 0 || n3 <= 0) return {0, 0};
    const uintptr_t lo = (uintptr_t)p;
    return {lo, lo + (uintptr_t)e * (uintptr_t)((n0 - 1) * s0 + (n1 - 1) * s1 + (n2 - 1) * s2 + n3)};
}
bool meet(Bytes a, Bytes b) { return a.lo < b.hi && b.lo < a.hi; }

// whether rows of n3 elements at strides s0, s1, s2 (sizes n0, n1, n2) share an element: dimensions are visited from the smallest stride
// up, each has to clear what lies below it
bool self_overlap(long long n0, long long s0, long long n1, long long s1, long long n2, long long s2, long long n3)
{
    long long n[3] = {n0, n1, n2}, s[3] = {s0, s1, s2}, below = n3;
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (s[j] < s[i]) { const long long t = s[i]; s[i] = s[j]; s[j] = t; const long long u = n[i]; n[i] = n[j]; n[j] = u; }
    for (int i = 0; i < 3; ++i) {
        if (n[i] <= 1) continue;
        if (s[i] < below) return true;
        below += (n[i] - 1) * s[i];
    }
    return false;
}

// a head tensor [T][H][D] and another one: do they share an element?  Rows of one buffer (a projection that holds q and k side by side)
// interleave without sharing any: their token strides are equal and the heads' stretches miss each other within it.
struct Heads { const void* p; long long T, H, D, st, sh; };
bool heads_meet(const Heads& a, const Heads& b, int e)
{
    if (!meet(span(a.p, e, a.T, a.st, a.H, a.sh, a.D > 0 ? 1 : 0, 0, a.D), span(b.p, e, b.T, b.st, b.H, b.sh, b.D > 0 ? 1 : 0, 0, b.D))) return false;
    if (a.st != b.st) return true;
    const long long ea = ((a.H - 1) * a.sh + a.D) * e, eb = ((b.H - 1) * b.sh + b.D) * e, st = a.st * e;
    if (st < ea || st < eb) return true;
    const long long d = (long long)((intptr_t)a.p - (intptr_t)b.p);
    const long long delta = ((d % st) + st) % st;
    return !(delta >= eb && delta + ea <= st);
}
bool same_heads(const Heads& a, const Heads& b)
{
    return a.p == b.p && (a.T <= 1 || a.st == b.st) && (a.H <= 1 || a.sh == b.sh);
}

int check_linear(const bx_linear_args* a)
{
    OP_REFUSE(!a, "bx_linear: null argument");
    OP_REFUSE(a->dtype < BX_TYPE_F32 || a->dtype > BX_TYPE_BF16, "bx_linear: unknown type %d", a->dtype);
    OP_REFUSE(a->act < BX_ACT_NONE || a->act > BX_ACT_SILU, "bx_linear: unknown activation %d", a->act);
    OP_REFUSE(a->M < 0 || a->N < 0 || a->K < 0 || a->M > LEN_MAX || a->N > LEN_MAX || a->K > LEN_MAX,
              "bx_linear: sizes %lld x %lld x %lld out of range", (long long)a->M, (long long)a->N, (long long)a->K);
    if (a->M == 0 || a->N == 0) return BX_OK;
    const int e = elem_bytes(a->dtype);
    OP_REFUSE(!a->y || (a->K > 0 && (!a->x || !a->w)), "bx_linear: null argument");
    OP_REFUSE(bad_stride(a->ldx, a->M) || bad_stride(a->ldw, a->N) || bad_stride(a->ldy, a->M) || (a->residual && bad_stride(a->ldr, a->M)),
              "bx_linear: bad row stride");
    OP_REFUSE(a->M > 1 && a->ldy < a->N, "bx_linear: rows of y overlap (stride %lld, %lld columns)", (long long)a->ldy, (long long)a->N);
    OP_REFUSE(misaligned(a->x, e) || misaligned(a->w, e) || misaligned(a->bias, e) || misaligned(a->residual, e) || misaligned(a->y, e) ||
              misaligned(a->m_dev, 4), "bx_linear: a pointer is not aligned to its elements");
    const Bytes y = span(a->y, e, a->M, a->ldy, 1, 0, 1, 0, a->N);
    OP_REFUSE(meet(y, span(a->x, e, a->M, a->ldx, 1, 0, 1, 0, a->K)) || meet(y, span(a->w, e, a->N, a->ldw, 1, 0, 1, 0, a->K)) ||
              meet(y, span(a->bias, e, 1, 0, 1, 0, 1, 0, a->N)) || meet(y, span(a->m_dev, 4, 1, 0)), "bx_linear: y overlaps an input");
    OP_REFUSE(a->residual && !(a->residual == a->y && (a->M <= 1 || a->ldr == a->ldy)) && meet(y, span(a->residual, e, a->M, a->ldr, 1, 0, 1, 0, a->N)),
              "bx_linear: y overlaps the residual without being it");
    return BX_OK;
}

int check_rope(const bx_qk_norm_rope_args* a)
{
    OP_REFUSE(!a, "bx_qk_norm_rope: null argument");
    OP_REFUSE(a->dtype < BX_TYPE_F32 || a->dtype > BX_TYPE_BF16, "bx_qk_norm_rope: unknown type %d", a->dtype);
    OP_REFUSE(a->norm < BX_NORM_NONE || a->norm > BX_NORM_L2, "bx_qk_norm_rope: unknown norm %d", a->norm);
    OP_REFUSE(a->pairs != BX_PAIRS_HALF && a->pairs != BX_PAIRS_INTERLEAVED, "bx_qk_norm_rope: unknown order of pairs %d", a->pairs);
    OP_REFUSE(a->pos_dtype != BX_POS_F32 && a->pos_dtype != BX_POS_I32, "bx_qk_norm_rope: unknown type of positions %d", a->pos_dtype);
    OP_REFUSE(a->reserved != 0, "bx_qk_norm_rope: reserved must be 0");
    OP_REFUSE(a->D < 1 || a->D > 256, "bx_qk_norm_rope: D=%d outside [1, 256]", a->D);
    OP_REFUSE(a->axes < 1 || a->axes > 4, "bx_qk_norm_rope: axes=%d outside [1, 4]", a->axes);
    long long pairs = 0;
    for (int i = 0; i < a->axes; ++i) {
        OP_REFUSE(a->sections[i] < 0, "bx_qk_norm_rope: negative section");
        pairs += a->sections[i];
    }
    OP_REFUSE(2 * pairs > a->D, "bx_qk_norm_rope: %lld rotation pairs do not fit D=%d", pairs, a->D);
    OP_REFUSE(!(a->eps >= 0.0f) || std::isinf(a->eps), "bx_qk_norm_rope: eps must be finite and not negative");
    OP_REFUSE(a->T < 0 || a->T > LEN_MAX || a->Hq < 0 || a->Hk < 0 || a->Hq > (1 << 20) || a->Hk > (1 << 20), "bx_qk_norm_rope: sizes out of range");
    const bool has_q = a->Hq > 0 && a->q, has_k = a->Hk > 0 && a->k;
    if (a->T == 0 || (!has_q && !has_k)) return BX_OK;
    const int e = elem_bytes(a->dtype);
    OP_REFUSE((has_q && !a->q_out) || (has_k && !a->k_out) || (pairs > 0 && (!a->pos || !a->freqs)), "bx_qk_norm_rope: null argument");
    const long long st[9] = {a->q_stride_t, a->q_stride_h, a->k_stride_t, a->k_stride_h, a->q_out_stride_t, a->q_out_stride_h,
                             a->k_out_stride_t, a->k_out_stride_h, a->pos_stride_t};
    const long long sn[9] = {a->T, a->Hq, a->T, a->Hk, a->T, a->Hq, a->T, a->Hk, a->T};
    for (int i = 0; i < 9; ++i) OP_REFUSE(bad_stride(st[i], sn[i]), "bx_qk_norm_rope: bad stride");
    OP_REFUSE(misaligned(a->q, e) || misaligned(a->k, e) || misaligned(a->q_out, e) || misaligned(a->k_out, e) || misaligned(a->q_weight, e) ||
              misaligned(a->k_weight, e) || misaligned(a->pos, 4) || misaligned(a->freqs, 8) || misaligned(a->m_dev, 4),
              "bx_qk_norm_rope: a pointer is not aligned to its elements");
    const Heads in[2] = {{has_q ? a->q : nullptr, a->T, a->Hq, a->D, a->q_stride_t, a->q_stride_h}, {has_k ? a->k : nullptr, a->T, a->Hk, a->D, a->k_stride_t, a->k_stride_h}};
    const Heads out[2] = {{has_q ? a->q_out : nullptr, a->T, a->Hq, a->D, a->q_out_stride_t, a->q_out_stride_h},
                          {has_k ? a->k_out : nullptr, a->T, a->Hk, a->D, a->k_out_stride_t, a->k_out_stride_h}};
    for (int i = 0; i < 2; ++i) {
        if (!out[i].p) continue;
        OP_REFUSE(self_overlap(out[i].T, out[i].st, out[i].H, out[i].sh, 1, 0, out[i].D), "bx_qk_norm_rope: rows of an output overlap");
        const Bytes o = span(out[i].p, e, out[i].T, out[i].st, out[i].H, out[i].sh, 1, 0, a->D);
        OP_REFUSE(meet(o, span(a->q_weight, e, 1, 0, 1, 0, 1, 0, a->D)) || meet(o, span(a->k_weight, e, 1, 0, 1, 0, 1, 0, a->D)) ||
                  meet(o, span(a->pos, 4, a->T, a->pos_stride_t, 1, 0, 1, 0, a->axes)) || meet(o, span(a->freqs, 8, 1, 0, 1, 0, 1, 0, pairs)) ||
                  meet(o, span(a->m_dev, 4, 1, 0)), "bx_qk_norm_rope: an output overlaps an input");
        for (int j = 0; j < 2; ++j) {
            if (in[j].p && !(i == j && same_heads(out[i], in[j])))
                OP_REFUSE(heads_meet(out[i], in[j], e), "bx_qk_norm_rope: an output overlaps an input without being it");
            if (j > i && out[j].p) OP_REFUSE(heads_meet(out[i], out[j], e), "bx_qk_norm_rope: the outputs overlap");
        }
    }
    return BX_OK;
}

int check_attention(const bx_attention_args* a)
{
    OP_REFUSE(!a, "bx_attention: null argument");
    OP_REFUSE(a->dtype < BX_TYPE_F32 || a->dtype > BX_TYPE_BF16, "bx_attention: unknown type %d", a->dtype);
    OP_REFUSE(a->reserved != 0, "bx_attention: reserved must be 0");
    OP_REFUSE(a->D < 1 || a->D > 128, "bx_attention: D=%d outside [1, 128]", a->D);
    OP_REFUSE(a->Hq < 1 || a->Hk < 1 || a->Hq % a->Hk != 0, "bx_attention: %d query heads cannot share %d key heads", a->Hq, a->Hk);
    OP_REFUSE(a->B < 0 || a->Lq < 0 || a->Lk < 0 || a->Lk >= LEN_MAX || (long long)a->Lq * a->Hq >= LEN_MAX ||
              (long long)a->B * a->Lq * a->Hq >= LEN_MAX, "bx_attention: sizes out of range");
    OP_REFUSE(a->sinks < 0, "bx_attention: negative count of first keys");
    OP_REFUSE(!(a->scale >= 0x1p-100f && a->scale <= 0x1p100f), "bx_attention: scale must lie in [2^-100, 2^100]");
    if (a->B == 0 || a->Lq == 0) return BX_OK;
    const int e = elem_bytes(a->dtype);
    OP_REFUSE(!a->q || !a->o || (a->Lk > 0 && (!a->k || !a->v)), "bx_attention: null argument");
    const long long st[12] = {a->q_stride_b, a->q_stride_t, a->q_stride_h, a->k_stride_b, a->k_stride_t, a->k_stride_h,
                              a->v_stride_b, a->v_stride_t, a->v_stride_h, a->o_stride_b, a->o_stride_t, a->o_stride_h};
    const long long sn[12] = {a->B, a->Lq, a->Hq, a->B, a->Lk, a->Hk, a->B, a->Lk, a->Hk, a->B, a->Lq, a->Hq};
    for (int i = 0; i < 12; ++i) OP_REFUSE(bad_stride(st[i], sn[i]), "bx_attention: bad stride");
    OP_REFUSE(misaligned(a->q, e) || misaligned(a->k, e) || misaligned(a->v, e) || misaligned(a->o, e) || misaligned(a->q_lens, 4) ||
              misaligned(a->k_lens, 4) || misaligned(a->workspace, 16), "bx_attention: a pointer is not aligned to its elements (workspace: 16 bytes)");
    OP_REFUSE(self_overlap(a->B, a->o_stride_b, a->Lq, a->o_stride_t, a->Hq, a->o_stride_h, a->D), "bx_attention: rows of o overlap");
    const Bytes o = span(a->o, e, a->B, a->o_stride_b, a->Lq, a->o_stride_t, a->Hq, a->o_stride_h, a->D);
    const Bytes ws = span(a->workspace, 1, 1, 0, 1, 0, 1, 0, a->workspace_bytes);
    const Bytes in[5] = {span(a->q, e, a->B, a->q_stride_b, a->Lq, a->q_stride_t, a->Hq, a->q_stride_h, a->D),
                         span(a->k, e, a->B, a->k_stride_b, a->Lk, a->k_stride_t, a->Hk, a->k_stride_h, a->D),
                         span(a->v, e, a->B, a->v_stride_b, a->Lk, a->v_stride_t, a->Hk, a->v_stride_h, a->D),
                         span(a->q_lens, 4, a->B, 1), span(a->k_lens, 4, a->B, 1)};
    OP_REFUSE(meet(o, ws), "bx_attention: o overlaps the workspace");
    for (int i = 0; i < 5; ++i) OP_REFUSE(meet(o, in[i]) || meet(ws, in[i]), "bx_attention: o or the workspace overlaps an input");
    return BX_OK;
}

// bounds beyond every length mean what "as far as there are keys" means; this keeps the kernels' index sums inside 32 bits
bx_attention_args clamped(const bx_attention_args& a)
{
    bx_attention_args c = a;
    const int big = (int)(LEN_MAX - 1);
    c.left = a.left < 0 ? -1 : a.left > big ? big : a.left;
    c.right = a.right < 0 ? -1 : a.right > big ? big : a.right;
    c.sinks = a.sinks > big ? big : a.sinks;
    return c;
}

}  // namespace

extern "C" {

int bx_linear(bx_ctx* c, void* stream, const bx_linear_args* a)
{
    const int rc = check_linear(a);
    if (rc != BX_OK) return rc;
    OP_REFUSE(!c, "null context");
    BxDevScope ds(c->device);
    return bxk_linear((hipStream_t)stream, c->n_cu, *a);
}

int bx_qk_norm_rope(bx_ctx* c, void* stream, const bx_qk_norm_rope_args* a)
{
    const int rc = check_rope(a);
    if (rc != BX_OK) return rc;
    OP_REFUSE(!c, "null context");
    BxDevScope ds(c->device);
    return bxk_qk_norm_rope((hipStream_t)stream, c->n_cu, *a);
}

int64_t bx_attention_workspace(bx_ctx* c, const bx_attention_args* a)
{
    if (!c) { bx_set_error("null context"); return -1; }
    if (!a || a->B < 0 || a->Lq < 0 || a->Lk < 0 || a->Lk >= LEN_MAX || a->Hk < 1 || a->Hq < 1 || a->Hq % a->Hk != 0 || a->D < 1 || a->D > 128 ||
        a->sinks < 0 || (long long)a->B * a->Lq * a->Hq >= LEN_MAX || (long long)a->Lq * a->Hq >= LEN_MAX) {
        bx_set_error("bx_attention_workspace: bad argument");
        return -1;
    }
    return bxk_attention_workspace(c->n_cu, clamped(*a));
}

int bx_attention(bx_ctx* c, void* stream, const bx_attention_args* a)
{
    const int rc = check_attention(a);
    if (rc != BX_OK) return rc;
    OP_REFUSE(!c, "null context");
    BxDevScope ds(c->device);
    return bxk_attention((hipStream_t)stream, c->n_cu, clamped(*a));
}

}  // extern "C"
