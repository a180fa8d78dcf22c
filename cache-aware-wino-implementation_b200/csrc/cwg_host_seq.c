/*
 * cwg_host_seq.c -- host side of the sequence layers and the 8-bit matrix
 * product, in C: argument checking only.  Everything that can be known without
 * reading device memory is checked here, before any CUDA call; indices that live
 * in device memory are checked by the kernels.
 */
#include <stdint.h>

#include "../../include/cwg.h"
#include "cwg_internal.h"

/* Most rows, sequences and channels: indices, their tiles' ends and the middle of two of them
 * stay inside int. */
enum { kMaxRows = 1 << 30 };

/* Rows of `width` elements, `ld` apart, aligned to the element. */
static int rows_ok(const void *p, long long ld, long long rows, long long width, size_t esz) {
  if (!p || ((uintptr_t)p % esz)) return 0;
  /* one row has no next row: its ld says nothing */
  return rows <= 1 ? 1 : ld >= width && ld <= (1LL << 40);
}

/* Addresses and row distances of checked operands reach 2^72, beyond 64 bits. */
typedef __int128 wide;

/* Whether two row operands share bytes.  Two column ranges of one matrix have the
 * same row distance and lie apart within it. */
static int overlaps(const void *a, long long lda, long long wa, const void *b, long long ldb,
                    long long wb, long long rows, size_t esz) {
  if (!a || !b || rows <= 0) return 0;
  if (rows == 1) lda = wa, ldb = wb;
  const wide e = (wide)esz, a0 = (uintptr_t)a, b0 = (uintptr_t)b;
  if (a0 + ((wide)(rows - 1) * lda + wa) * e <= b0 || b0 + ((wide)(rows - 1) * ldb + wb) * e <= a0)
    return 0;
  if (lda != ldb || rows == 1) return 1;
  const wide step = lda * e;
  wide off = (b0 - a0) % step; /* b's columns behind a's, in one row */
  if (off < 0) off += step;
  return !(off >= wa * e && off + wb * e <= step);
}

/* Whether the byte ranges of two row operands meet. */
static int ranges_meet(const void *a, long long arow, const void *b, long long brow,
                       long long arows, long long brows, long long abytes, long long bbytes) {
  const wide a0 = (uintptr_t)a, b0 = (uintptr_t)b;
  return a0 < b0 + (brows > 1 ? (wide)(brows - 1) * brow : 0) + bbytes &&
         b0 < a0 + (arows > 1 ? (wide)(arows - 1) * arow : 0) + abytes;
}

/* A dense operand: neighbouring bytes. */
typedef struct block {
  const void *p;
  wide bytes;
} block;

static int blocks_meet(block a, block b) {
  const wide a0 = (uintptr_t)a.p, b0 = (uintptr_t)b.p;
  return a.p && b.p && a.bytes > 0 && b.bytes > 0 && a0 < b0 + b.bytes && b0 < a0 + a.bytes;
}

/* Whether a dense operand shares bytes with `rows` rows of `width` elements. */
static int meets_rows(block a, const void *p, long long ld, long long rows, long long width,
                      size_t esz) {
  if (!a.p || !p || a.bytes <= 0 || rows <= 0 || width <= 0) return 0;
  const wide step = (wide)ld * (wide)esz, row = (wide)width * (wide)esz;
  const wide off = (wide)(uintptr_t)a.p - (wide)(uintptr_t)p; /* of the block's first byte */
  if (off + a.bytes <= 0 || off >= (rows > 1 ? (rows - 1) * step : 0) + row) return 0;
  if (off < row) return 1;
  const wide first = (off - row) / step + 1; /* first row that ends behind the block's start */
  return first < rows && first * step < off + a.bytes;
}

/* Whether one of n dense inputs shares bytes with the rows of y or with the cache lines. */
static int outputs_meet(const block *in, int n, const void *y, long long ldy, long long rows,
                        long long width, size_t esz, block lines) {
  for (int i = 0; i < n; ++i)
    if (meets_rows(in[i], y, ldy, rows, width, esz) || blocks_meet(in[i], lines)) return 1;
  return 0;
}

static int act_of(unsigned flags, unsigned allowed) {
  const unsigned act = flags & (CWG_RELU | CWG_SILU);
  if (flags & ~(allowed | CWG_BF16 | CWG_NO_PDL)) return -1;
  if (act == (CWG_RELU | CWG_SILU)) return -1;
  return act == CWG_RELU ? CWGK_ACT_RELU : act == CWG_SILU ? CWGK_ACT_SILU : CWGK_ACT_NONE;
}

/* The cache lines: enough of them when sequence b takes line b. */
static int lines_ok(const void *state, const int *slots, int n_seq, int n_slots, size_t esz) {
  if (!state) return 1;
  if (((uintptr_t)state % esz) || ((uintptr_t)slots & 3) || n_slots < 0) return 0;
  return slots || n_slots >= n_seq;
}

static int conv1d_check(const cwgk_conv1d *p, int rows, unsigned flags) {
  const size_t esz = (flags & CWG_BF16) ? 2 : 4;
  if (rows < 0 || rows > kMaxRows || p->n_seq < 0 || p->n_seq > kMaxRows || p->channels <= 0 ||
      p->channels > kMaxRows)
    return CWG_EINVAL;
  if (p->width < 2) return CWG_EINVAL;
  if (p->width > 4) return CWG_EUNSUPPORTED;
  if (!p->w || ((uintptr_t)p->w & 3) || ((uintptr_t)p->bias & 3)) return CWG_EINVAL;
  if (!lines_ok(p->state, p->slots, p->n_seq, p->n_slots, esz)) return CWG_EINVAL;
  const block lines = {p->state, (wide)p->n_slots * (p->width - 1) * p->channels * (wide)esz};
  if (rows > 0) {
    if (!rows_ok(p->x, p->ldx, rows, p->channels, esz) ||
        !rows_ok(p->y, p->ldy, rows, p->channels, esz))
      return CWG_EINVAL;
    if (overlaps(p->x, p->ldx, p->channels, p->y, p->ldy, p->channels, rows, esz) ||
        meets_rows(lines, p->x, p->ldx, rows, p->channels, esz) ||
        meets_rows(lines, p->y, p->ldy, rows, p->channels, esz))
      return CWG_EINVAL;
  }
  const block in[] = {{p->w, (wide)p->channels * p->width * 4},
                      {p->bias, (wide)p->channels * 4},
                      {p->starts, ((wide)p->n_seq + 1) * 4},
                      {p->slots, (wide)p->n_seq * 4},
                      {p->resume, p->n_seq}};
  if (outputs_meet(in, 5, p->y, p->ldy, rows, p->channels, esz, lines)) return CWG_EINVAL;
  return CWG_OK;
}

int cwg_conv1d_causal(const void *x, long long ldx, const float *w, const float *bias, void *y,
                      long long ldy, void *state, const int *starts, const int *slots,
                      const unsigned char *resume, int tokens, int n_seq, int n_slots,
                      int channels, int width, unsigned flags, void *stream) {
  const int act = act_of(flags, CWG_RELU | CWG_SILU);
  if (act < 0) return CWG_EINVAL;
  const cwgk_conv1d op = {x,      ldx,    w,      bias,  y,       ldy,      state, starts,
                          slots,  resume, tokens, n_seq, n_slots, channels, width, act,
                          (flags & CWG_BF16) != 0, !(flags & CWG_NO_PDL)};
  const int rc = conv1d_check(&op, tokens, flags);
  if (rc) return rc;
  if (n_seq == 0) return CWG_OK;
  if (!starts || ((uintptr_t)starts & 3)) return CWG_EINVAL;
  if (tokens == 0 && !state) return CWG_OK;
  return cwgk_conv1d_prompt(&op, stream);
}

int cwg_conv1d_causal_step(const void *x, long long ldx, const float *w, const float *bias,
                           void *y, long long ldy, void *state, const int *slots, int n,
                           int n_slots, int channels, int width, unsigned flags, void *stream) {
  const int act = act_of(flags, CWG_RELU | CWG_SILU);
  if (act < 0) return CWG_EINVAL;
  const cwgk_conv1d op = {x,    ldx, w, bias, y,       ldy,      state, 0,  slots,
                          0,    n,   n, n_slots, channels, width, act, (flags & CWG_BF16) != 0,
                          !(flags & CWG_NO_PDL)};
  const int rc = conv1d_check(&op, n, flags);
  if (rc) return rc;
  if (n == 0) return CWG_OK;
  if (!state) return CWG_EINVAL; /* a step without a past is not a step */
  return cwgk_conv1d_step(&op, stream);
}

/* The call's dense inputs; a step looks at neither offsets nor `resume`. */
enum { kSsmDense = 6 };
static void ssm_dense(const cwg_ssm *p, int n_seq, int step, block *in) {
  const wide c = p->channels;
  in[0] = (block){p->A, c * p->states * 4};
  in[1] = (block){p->D, c * 4};
  in[2] = (block){p->dt_bias, c * 4};
  in[3] = (block){p->slots, (wide)n_seq * 4};
  in[4] = (block){step ? 0 : p->starts, ((wide)n_seq + 1) * 4};
  in[5] = (block){step ? 0 : p->resume, n_seq};
}
static block ssm_lines(const cwg_ssm *p) {
  return (block){p->state, (wide)p->n_slots * p->channels * p->states * 4};
}
/* Whether a dense operand shares bytes with the call's rows, inputs' or outputs'. */
static int meets_ssm_rows(block b, const cwg_ssm *p) {
  const size_t esz = (p->flags & CWG_BF16) ? 2 : 4;
  const long long rows = p->tokens, c = p->channels, gn = (long long)p->groups * p->states;
  return meets_rows(b, p->u, p->ldu, rows, c, esz) || meets_rows(b, p->dt, p->lddt, rows, c, esz) ||
         meets_rows(b, p->z, p->ldz, rows, c, esz) || meets_rows(b, p->B, p->ldb, rows, gn, esz) ||
         meets_rows(b, p->C, p->ldc, rows, gn, esz) || meets_rows(b, p->y, p->ldy, rows, c, esz);
}

static int ssm_check(const cwg_ssm *p, int n_seq, int step) {
  if (!p) return CWG_EINVAL;
  if (p->flags & ~(CWG_BF16 | CWG_SOFTPLUS | CWG_NO_PDL)) return CWG_EINVAL;
  const size_t esz = (p->flags & CWG_BF16) ? 2 : 4;
  if (p->tokens < 0 || p->tokens > kMaxRows || n_seq < 0 || n_seq > kMaxRows ||
      p->channels <= 0 || p->channels > kMaxRows || p->groups <= 0 || p->states <= 0)
    return CWG_EINVAL;
  if (p->channels % p->groups) return CWG_EINVAL;
  if (p->states > 64) return CWG_EUNSUPPORTED;
  if ((long long)p->groups * p->states > 0x7fffffffLL) return CWG_EINVAL;
  if (!p->A || ((uintptr_t)p->A & 3) || ((uintptr_t)p->D & 3) || ((uintptr_t)p->dt_bias & 3))
    return CWG_EINVAL;
  if (!lines_ok(p->state, p->slots, n_seq, p->n_slots, 4)) return CWG_EINVAL;
  if (p->tokens > 0) {
    const long long rows = p->tokens, c = p->channels, gn = (long long)p->groups * p->states;
    if (!rows_ok(p->u, p->ldu, rows, c, esz) || !rows_ok(p->dt, p->lddt, rows, c, esz) ||
        !rows_ok(p->B, p->ldb, rows, gn, esz) || !rows_ok(p->C, p->ldc, rows, gn, esz) ||
        !rows_ok(p->y, p->ldy, rows, c, esz) || (p->z && !rows_ok(p->z, p->ldz, rows, c, esz)))
      return CWG_EINVAL;
    if (overlaps(p->u, p->ldu, c, p->y, p->ldy, c, rows, esz) ||
        overlaps(p->dt, p->lddt, c, p->y, p->ldy, c, rows, esz) ||
        overlaps(p->z, p->ldz, c, p->y, p->ldy, c, rows, esz) ||
        overlaps(p->B, p->ldb, gn, p->y, p->ldy, c, rows, esz) ||
        overlaps(p->C, p->ldc, gn, p->y, p->ldy, c, rows, esz))
      return CWG_EINVAL;
    if (meets_ssm_rows(ssm_lines(p), p)) return CWG_EINVAL;
  }
  block in[kSsmDense];
  ssm_dense(p, n_seq, step, in);
  if (outputs_meet(in, kSsmDense, p->y, p->ldy, p->tokens, p->channels, esz, ssm_lines(p)))
    return CWG_EINVAL;
  return CWG_OK;
}

size_t cwg_ssm_workspace_bytes(int tokens, int n_seq, int channels, int states) {
  if (tokens < 0 || tokens > kMaxRows || n_seq < 0 || n_seq > kMaxRows || channels <= 0 ||
      channels > kMaxRows || states <= 0 || states > 64)
    return 0;
  return cwgk_ssm_workspace_bytes(tokens, n_seq, channels, states);
}

int cwg_ssm_scan(const cwg_ssm *op, void *workspace, size_t workspace_bytes, void *stream) {
  const int rc = ssm_check(op, op ? op->n_seq : 0, 0);
  if (rc) return rc;
  if (op->n_seq == 0) return CWG_OK;
  if (!op->starts || ((uintptr_t)op->starts & 3)) return CWG_EINVAL;
  if (workspace) {
    if ((uintptr_t)workspace & 255) return CWG_EINVAL;
    const size_t need = cwgk_ssm_call_bytes(op);
    if (workspace_bytes < need) return CWG_EINVAL;
    const block ws = {workspace, (wide)need};
    block in[kSsmDense];
    ssm_dense(op, op->n_seq, 0, in);
    int meet = meets_ssm_rows(ws, op) || blocks_meet(ws, ssm_lines(op));
    for (int i = 0; i < kSsmDense; ++i) meet |= blocks_meet(ws, in[i]);
    if (meet) return CWG_EINVAL;
  }
  if (op->tokens == 0 && !op->state) return CWG_OK;
  return cwgk_ssm_scan(op, workspace, stream);
}

int cwg_ssm_step(const cwg_ssm *op, void *stream) {
  const int rc = ssm_check(op, op ? op->tokens : 0, 1);
  if (rc) return rc;
  if (op->tokens == 0) return CWG_OK;
  if (!op->state) return CWG_EINVAL;
  return cwgk_ssm_step(op, stream);
}

int cwg_fp8_quantize(const void *x, long long ldx, void *q, long long ldq, float *scale,
                     long long lds, int rows, int cols, int block_rows, unsigned flags,
                     void *stream) {
  if (flags & ~(CWG_BF16 | CWG_NO_PDL)) return CWG_EINVAL;
  if (rows < 0 || rows > kMaxRows || cols <= 0 || cols > kMaxRows ||
      (block_rows != 1 && block_rows != 128))
    return CWG_EINVAL;
  if (rows == 0) return CWG_OK;
  const size_t esz = (flags & CWG_BF16) ? 2 : 4;
  const long long kb = ((long long)cols + 127) / 128;
  const long long rb = block_rows == 1 ? rows : ((long long)rows + 127) / 128;
  if (!rows_ok(x, ldx, rows, cols, esz) || !rows_ok(q, ldq, rows, cols, 1) ||
      !rows_ok(scale, lds, rb, kb, 4))
    return CWG_EINVAL;
  const long long e = (long long)esz;
  if (ranges_meet(x, ldx * e, q, ldq, rows, rows, cols * e, cols) ||
      ranges_meet(x, ldx * e, scale, lds * 4, rows, rb, cols * e, kb * 4) ||
      ranges_meet(q, ldq, scale, lds * 4, rows, rb, cols, kb * 4))
    return CWG_EINVAL;
  return cwgk_fp8_quantize(x, ldx, q, ldq, scale, lds, rows, cols, block_rows,
                           (flags & CWG_BF16) != 0, !(flags & CWG_NO_PDL), stream);
}

int cwg_fp8_matmul(const void *a, long long lda, const float *a_scale, long long lda_scale,
                   const void *w, long long ldw, const float *w_scale, long long ldw_scale,
                   const float *bias, void *y, long long ldy, int m, int n, int k,
                   unsigned flags, void *stream) {
  if (flags & ~(CWG_BF16 | CWG_RELU | CWG_NO_PDL)) return CWG_EINVAL;
  if (m < 0 || n <= 0 || k <= 0 || m > kMaxRows || n > kMaxRows || k > kMaxRows)
    return CWG_EINVAL;
  if (m == 0) return CWG_OK;
  const size_t esz = (flags & CWG_BF16) ? 2 : 4;
  const long long kb = ((long long)k + 127) / 128, nb = ((long long)n + 127) / 128;
  if (!rows_ok(a, lda, m, k, 16) || !rows_ok(w, ldw, n, k, 16) ||
      !rows_ok(a_scale, lda_scale, m, kb, 4) || !rows_ok(w_scale, ldw_scale, nb, kb, 4) ||
      !rows_ok(y, ldy, m, n, esz) || ((uintptr_t)bias & 3))
    return CWG_EINVAL;
  if ((m > 1 && (lda & 15)) || (n > 1 && (ldw & 15))) return CWG_EINVAL;
  const long long e = (long long)esz;
  if (ranges_meet(a, lda, y, ldy * e, m, m, k, n * e) ||
      ranges_meet(w, ldw, y, ldy * e, n, m, k, n * e) ||
      ranges_meet(a_scale, lda_scale * 4, y, ldy * e, m, m, kb * 4, n * e) ||
      ranges_meet(w_scale, ldw_scale * 4, y, ldy * e, nb, m, kb * 4, n * e) ||
      (bias && ranges_meet(bias, 0, y, ldy * e, 1, m, n * 4LL, n * e)))
    return CWG_EINVAL;
  const cwgk_fp8 op = {a,       w,         lda,       ldw, a_scale, w_scale, bias,
                       lda_scale, ldw_scale, y,         ldy, m,       n,       k,
                       (flags & CWG_RELU) != 0, (flags & CWG_BF16) != 0,
                       !(flags & CWG_NO_PDL)};
  return cwgk_fp8_matmul(&op, stream);
}
