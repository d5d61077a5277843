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

// an operand's elements: rows of `row` elements of `e` bytes at strides s (in elements) along up to three dimensions of sizes n
struct Rows { const void* p; int e; long long row, n[3], s[3]; };
Rows rows_of(const void* p, int e, long long row, long long n0 = 1, long long s0 = 0, long long n1 = 1, long long s1 = 0, long long n2 = 1, long long s2 = 0)
{
    return {p, e, row, {n0, n1, n2}, {s0, s1, s2}};
}

long long gcd(long long a, long long b) { while (b) { const long long t = a % b; a = b; b = t; } return a; }

// Whether two operands may share memory.  They do not where the stretches that they lie in miss each other; nor where their rows are interleaved, as the
// parts of one buffer are: with g the greatest common divisor of the strides along some dimensions of both, all rows of an operand lie at the same
// place modulo g but for what the other dimensions add, and the two places have to miss each other.  Every choice of dimensions is tried.
bool meet(const Rows& a, const Rows& b)
{
    const Rows* x[2] = {&a, &b};
    long long extent[2];
    for (int k = 0; k < 2; ++k) {
        if (!x[k]->p || x[k]->row <= 0) return false;
        extent[k] = x[k]->row;
        for (int i = 0; i < 3; ++i) {
            if (x[k]->n[i] <= 0) return false;
            extent[k] += (x[k]->n[i] - 1) * x[k]->s[i];
        }
        extent[k] *= x[k]->e;
    }
    const uintptr_t pa = (uintptr_t)a.p, pb = (uintptr_t)b.p;
    if (pa + (uintptr_t)extent[0] <= pb || pb + (uintptr_t)extent[1] <= pa) return false;
    for (int mask = 1; mask < 64; ++mask) {
        long long g = 0, in[2] = {a.row * a.e, b.row * b.e};
        for (int k = 0; k < 2; ++k)
            for (int i = 0; i < 3; ++i) {
                if (x[k]->n[i] <= 1) continue;
                const long long s = x[k]->s[i] * x[k]->e;
                if (mask >> (3 * k + i) & 1) g = gcd(g, s);
                else in[k] += (x[k]->n[i] - 1) * s;
            }
        if (g == 0 || in[0] > g || in[1] > g) continue;
        const long long d = (long long)((pa > pb ? pa - pb : pb - pa) % (uintptr_t)g), at = pa >= pb || d == 0 ? d : g - d;      // a's place behind b's
        if (at >= in[1] && at + in[0] <= g) return false;
    }
    return true;
}

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
    const Rows y = rows_of(a->y, e, a->N, a->M, a->ldy);
    OP_REFUSE(meet(y, rows_of(a->x, e, a->K, a->M, a->ldx)) || meet(y, rows_of(a->w, e, a->K, a->N, a->ldw)) || meet(y, rows_of(a->bias, e, a->N)) ||
              meet(y, rows_of(a->m_dev, 4, 1)), "bx_linear: y overlaps an input");
    OP_REFUSE(a->residual && !(a->residual == a->y && (a->M <= 1 || a->ldr == a->ldy)) && meet(y, rows_of(a->residual, e, a->N, a->M, a->ldr)),
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
    const Rows in[2] = {rows_of(has_q ? a->q : nullptr, e, a->D, a->T, a->q_stride_t, a->Hq, a->q_stride_h),
                        rows_of(has_k ? a->k : nullptr, e, a->D, a->T, a->k_stride_t, a->Hk, a->k_stride_h)};
    const Rows out[2] = {rows_of(has_q ? a->q_out : nullptr, e, a->D, a->T, a->q_out_stride_t, a->Hq, a->q_out_stride_h),
                         rows_of(has_k ? a->k_out : nullptr, e, a->D, a->T, a->k_out_stride_t, a->Hk, a->k_out_stride_h)};
    const auto same = [](const Rows& x, const Rows& y) { return x.p == y.p && (x.n[0] <= 1 || x.s[0] == y.s[0]) && (x.n[1] <= 1 || x.s[1] == y.s[1]); };
    for (int i = 0; i < 2; ++i) {
        const Rows& o = out[i];
        if (!o.p) continue;
        OP_REFUSE(self_overlap(o.n[0], o.s[0], o.n[1], o.s[1], 1, 0, o.row), "bx_qk_norm_rope: rows of an output overlap");
        OP_REFUSE(meet(o, rows_of(a->q_weight, e, a->D)) || meet(o, rows_of(a->k_weight, e, a->D)) || meet(o, rows_of(a->pos, 4, a->axes, a->T, a->pos_stride_t)) ||
                  meet(o, rows_of(a->freqs, 8, pairs)) || meet(o, rows_of(a->m_dev, 4, 1)), "bx_qk_norm_rope: an output overlaps an input");
        for (int j = 0; j < 2; ++j) {
            OP_REFUSE(!(i == j && same(o, in[j])) && meet(o, in[j]), "bx_qk_norm_rope: an output overlaps an input without being it");
            OP_REFUSE(j > i && meet(o, out[j]), "bx_qk_norm_rope: the outputs overlap");
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
    const Rows o = rows_of(a->o, e, a->D, a->B, a->o_stride_b, a->Lq, a->o_stride_t, a->Hq, a->o_stride_h);
    const Rows ws = rows_of(a->workspace, 1, a->workspace_bytes);
    const Rows in[5] = {rows_of(a->q, e, a->D, a->B, a->q_stride_b, a->Lq, a->q_stride_t, a->Hq, a->q_stride_h),
                        rows_of(a->k, e, a->D, a->B, a->k_stride_b, a->Lk, a->k_stride_t, a->Hk, a->k_stride_h),
                        rows_of(a->v, e, a->D, a->B, a->v_stride_b, a->Lk, a->v_stride_t, a->Hk, a->v_stride_h),
                        rows_of(a->q_lens, 4, a->B), rows_of(a->k_lens, 4, a->B)};
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
    if (!a || a->dtype < BX_TYPE_F32 || a->dtype > BX_TYPE_BF16 || a->B < 0 || a->Lq < 0 || a->Lk < 0 || a->Lk >= LEN_MAX || a->Hk < 1 || a->Hq < 1 || a->Hq % a->Hk != 0 || a->D < 1 || a->D > 128 ||
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
