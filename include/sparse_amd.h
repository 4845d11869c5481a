/* sparse_amd.h -- C ABI of libsparse_amd.so, the MI355X-native implementation of
 * the diku-dk/sparse `mk_compressed` hot path.
 *
 * The reference is a Futhark library; the only thing a C caller can bind is the
 * API that `futhark c --library` (or `futhark hip --library`) generates from
 * `entry` definitions.  This header follows that generated-API convention
 * symbol for symbol (context / arrays / opaques / entries; outputs first as
 * pointer-to-pointer, scalars by value, 0 = success, error text through
 * futhark_context_get_error), so a harness written against the reference's
 * generated library links against this one unchanged.
 *
 *   S/ = lib/github.com/diku-dk/sparse/ in the reference tree.
 *
 * Three groups of entry points:
 *   (1) the reference's OWN entries -- S/compressed_test.fut, module
 *       `mk_compressed i32` -- under their generated names
 *       futhark_entry_test_*;
 *   (2) entries for f64 / f32 / i32 with opaque matrix handles.  The reference
 *       exports no such entries (its module is only reachable from Futhark
 *       source); integration/sparse_entry.fut is the entry file a maintainer adds
 *       to the reference to obtain exactly these symbols;
 *   (3) sparse_amd_* extensions with no counterpart in the generated API
 *       (stream hand-over, zero-copy wrapping, structure observation).
 *
 * Conventions that differ from textbook CSR (and are kept at this boundary):
 *   - row_off is the INCLUSIVE prefix sum of length n (S/compressed.fut:94,159);
 *   - all indices are int64_t (S/compressed.fut:66,94-95);
 *   - a CSC matrix of shape n x m IS the CSR matrix of its m x n transpose
 *     (S/compressed.fut:226); transpose moves no data (S/compressed.fut:185,220).
 *
 * All arrays and opaques are owned by the context and live in device memory.
 * futhark_new_* copies from the host; futhark_values_* copies to the host and
 * returns after the copy has completed.  Entries are asynchronous on the
 * context's HIP stream unless they must return a host scalar.
 */
#ifndef SPARSE_AMD_H
#define SPARSE_AMD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------ context */
struct futhark_context_config;
struct futhark_context;

struct futhark_context_config *futhark_context_config_new(void);
void futhark_context_config_free(struct futhark_context_config *cfg);
void futhark_context_config_set_debugging(struct futhark_context_config *cfg, int flag);
void futhark_context_config_set_profiling(struct futhark_context_config *cfg, int flag);
void futhark_context_config_set_logging(struct futhark_context_config *cfg, int flag);
/* Generated by `futhark multicore --library` (size of its worker pool; SURVEY 8b, BASELINE.md harness).
 * Accepted so that a harness written for the multicore reference library links and runs unchanged; a GPU
 * context has no worker pool and the value changes nothing. */
void futhark_context_config_set_num_threads(struct futhark_context_config *cfg, int n);
/* Device selection as in the generated GPU back ends: "#k" selects HIP device k. */
void futhark_context_config_set_device(struct futhark_context_config *cfg, const char *s);

struct futhark_context *futhark_context_new(struct futhark_context_config *cfg);
void futhark_context_free(struct futhark_context *ctx);
int futhark_context_sync(struct futhark_context *ctx);
/* Heap string owned by the caller (free()), or NULL if no error is pending. */
char *futhark_context_get_error(struct futhark_context *ctx);
int futhark_context_clear_caches(struct futhark_context *ctx);
char *futhark_context_report(struct futhark_context *ctx);

/* ------------------------------------------------------------------- arrays */
#define SPARSE_AMD_DECL_ARRAY_1D(NAME, CT)                                                        \
  struct futhark_##NAME##_1d;                                                                     \
  struct futhark_##NAME##_1d *futhark_new_##NAME##_1d(struct futhark_context *ctx,                \
                                                      const CT *data, int64_t dim0);              \
  /* data is a device pointer (hipDeviceptr_t); contents are copied */                            \
  struct futhark_##NAME##_1d *futhark_new_raw_##NAME##_1d(struct futhark_context *ctx,            \
                                                          const void *data, int64_t dim0);        \
  int futhark_free_##NAME##_1d(struct futhark_context *ctx, struct futhark_##NAME##_1d *arr);     \
  int futhark_values_##NAME##_1d(struct futhark_context *ctx, struct futhark_##NAME##_1d *arr,    \
                                 CT *data);                                                       \
  void *futhark_values_raw_##NAME##_1d(struct futhark_context *ctx,                               \
                                       struct futhark_##NAME##_1d *arr);                          \
  const int64_t *futhark_shape_##NAME##_1d(struct futhark_context *ctx,                           \
                                           struct futhark_##NAME##_1d *arr);                      \
  /* extension: alias caller-owned device memory without copying; free releases the handle only */\
  struct futhark_##NAME##_1d *sparse_amd_wrap_##NAME##_1d(struct futhark_context *ctx,            \
                                                          void *data, int64_t dim0);

#define SPARSE_AMD_DECL_ARRAY_2D(NAME, CT)                                                        \
  struct futhark_##NAME##_2d; /* row-major [dim0][dim1] */                                        \
  struct futhark_##NAME##_2d *futhark_new_##NAME##_2d(struct futhark_context *ctx,                \
                                                      const CT *data, int64_t dim0, int64_t dim1);\
  struct futhark_##NAME##_2d *futhark_new_raw_##NAME##_2d(                                        \
      struct futhark_context *ctx, const void *data, int64_t dim0, int64_t dim1);                 \
  int futhark_free_##NAME##_2d(struct futhark_context *ctx, struct futhark_##NAME##_2d *arr);     \
  int futhark_values_##NAME##_2d(struct futhark_context *ctx, struct futhark_##NAME##_2d *arr,    \
                                 CT *data);                                                       \
  void *futhark_values_raw_##NAME##_2d(struct futhark_context *ctx,                               \
                                       struct futhark_##NAME##_2d *arr);                          \
  const int64_t *futhark_shape_##NAME##_2d(struct futhark_context *ctx,                           \
                                           struct futhark_##NAME##_2d *arr);                      \
  struct futhark_##NAME##_2d *sparse_amd_wrap_##NAME##_2d(struct futhark_context *ctx,            \
                                                          void *data, int64_t dim0, int64_t dim1);

SPARSE_AMD_DECL_ARRAY_1D(i64, int64_t)
SPARSE_AMD_DECL_ARRAY_1D(i32, int32_t)
SPARSE_AMD_DECL_ARRAY_1D(f32, float)
SPARSE_AMD_DECL_ARRAY_1D(f64, double)
SPARSE_AMD_DECL_ARRAY_2D(i32, int32_t)
SPARSE_AMD_DECL_ARRAY_2D(f32, float)
SPARSE_AMD_DECL_ARRAY_2D(f64, double)

/* -------------------------------------------- (2) typed matrix entry points
 * TT in {f64, f32, i32}  <->  `module c = mk_compressed TT` (S/compressed.fut:61).
 * futhark_opaque_csr_TT is c.sr[n][m]; futhark_opaque_csc_TT is c.sc[n][m], whose
 * storage is the CSR record of the m x n transpose (S/compressed.fut:226).
 */
#define SPARSE_AMD_DECL_MATRIX(TT, CT)                                                            \
  struct futhark_opaque_csr_##TT;                                                                 \
  struct futhark_opaque_csc_##TT;                                                                 \
  int futhark_free_opaque_csr_##TT(struct futhark_context *ctx, struct futhark_opaque_csr_##TT *o);\
  int futhark_free_opaque_csc_##TT(struct futhark_context *ctx, struct futhark_opaque_csc_##TT *o);\
  /* Serialisers the compiler generates for every opaque type (here: the abstract sr / sc of    */\
  /* S/compressed.fut:24-54).  store: *n = size in bytes; p == NULL only asks for the size; *p   */\
  /* == NULL makes the library malloc() the buffer (caller frees), otherwise *p must hold *n     */\
  /* bytes.  restore: a new handle from such bytes, or NULL (error text pending).  The bytes hold */\
  /* n, m, row_off[n] (inclusive), col_idx[nnz] as i64 and vals[nnz] of the stored record; the    */\
  /* format is this library's own, as the generated format is the compiler's own.                */\
  int futhark_store_opaque_csr_##TT(struct futhark_context *ctx,                                  \
                                    const struct futhark_opaque_csr_##TT *obj, void **p, size_t *n);\
  int futhark_store_opaque_csc_##TT(struct futhark_context *ctx,                                  \
                                    const struct futhark_opaque_csc_##TT *obj, void **p, size_t *n);\
  struct futhark_opaque_csr_##TT *futhark_restore_opaque_csr_##TT(struct futhark_context *ctx,    \
                                                                  const void *p);                 \
  struct futhark_opaque_csc_##TT *futhark_restore_opaque_csc_##TT(struct futhark_context *ctx,    \
                                                                  const void *p);                 \
                                                                                                  \
  /* sr.sparse n m coo -- S/compressed.fut:154-160 (norm_coo :72-87).  Non-zero return on an   */ \
  /* out-of-range index (the assert at :156).                                                   */\
  int futhark_entry_csr_##TT##_sparse(struct futhark_context *ctx,                                \
                                      struct futhark_opaque_csr_##TT **out0, const int64_t n,     \
                                      const int64_t m, const struct futhark_i64_1d *rs,           \
                                      const struct futhark_i64_1d *cs,                            \
                                      const struct futhark_##TT##_1d *vs);                        \
  /* sc.sparse n m coo = sr.sparse m n (swap coo) -- S/compressed.fut:211-212 */                  \
  int futhark_entry_csc_##TT##_sparse(struct futhark_context *ctx,                                \
                                      struct futhark_opaque_csc_##TT **out0, const int64_t n,     \
                                      const int64_t m, const struct futhark_i64_1d *rs,           \
                                      const struct futhark_i64_1d *cs,                            \
                                      const struct futhark_##TT##_1d *vs);                        \
  /* sr.zero :98-103 / sc.zero :193-194 */                                                        \
  int futhark_entry_csr_##TT##_zero(struct futhark_context *ctx,                                  \
                                    struct futhark_opaque_csr_##TT **out0, const int64_t n,       \
                                    const int64_t m);                                             \
  int futhark_entry_csc_##TT##_zero(struct futhark_context *ctx,                                  \
                                    struct futhark_opaque_csc_##TT **out0, const int64_t n,       \
                                    const int64_t m);                                             \
  /* sr.eye :105-113 / sc.eye :199-200 */                                                         \
  int futhark_entry_csr_##TT##_eye(struct futhark_context *ctx,                                   \
                                   struct futhark_opaque_csr_##TT **out0, const int64_t n,        \
                                   const int64_t m);                                              \
  int futhark_entry_csc_##TT##_eye(struct futhark_context *ctx,                                   \
                                   struct futhark_opaque_csc_##TT **out0, const int64_t n,        \
                                   const int64_t m);                                              \
  /* sr.diag :115-120 / sc.diag :202-203 */                                                       \
  int futhark_entry_csr_##TT##_diag(struct futhark_context *ctx,                                  \
                                    struct futhark_opaque_csr_##TT **out0,                        \
                                    const struct futhark_##TT##_1d *v);                           \
  int futhark_entry_csc_##TT##_diag(struct futhark_context *ctx,                                  \
                                    struct futhark_opaque_csc_##TT **out0,                        \
                                    const struct futhark_##TT##_1d *v);                           \
  /* sr.dense :122-132 / sc.dense :214-215 (both return the matrix in its own n x m shape) */     \
  int futhark_entry_csr_##TT##_dense(struct futhark_context *ctx, struct futhark_##TT##_2d **out0,\
                                     const struct futhark_opaque_csr_##TT *a);                    \
  int futhark_entry_csc_##TT##_dense(struct futhark_context *ctx, struct futhark_##TT##_2d **out0,\
                                     const struct futhark_opaque_csc_##TT *a);                    \
  /* sr.scale :148-152 / sc.scale :196-197 */                                                     \
  int futhark_entry_csr_##TT##_scale(struct futhark_context *ctx,                                 \
                                     struct futhark_opaque_csr_##TT **out0, const CT v,           \
                                     const struct futhark_opaque_csr_##TT *a);                    \
  int futhark_entry_csc_##TT##_scale(struct futhark_context *ctx,                                 \
                                     struct futhark_opaque_csc_##TT **out0, const CT v,           \
                                     const struct futhark_opaque_csc_##TT *a);                    \
  /* sr.nnz :162-164 / sc.nnz :205-206 (counts stored values that are not zero) */                \
  int futhark_entry_csr_##TT##_nnz(struct futhark_context *ctx, int64_t *out0,                    \
                                   const struct futhark_opaque_csr_##TT *a);                      \
  int futhark_entry_csc_##TT##_nnz(struct futhark_context *ctx, int64_t *out0,                    \
                                   const struct futhark_opaque_csc_##TT *a);                      \
  /* sr.coo :166-177 / sc.coo :208-209 (unzip3: rows, cols, values in stored order) */            \
  int futhark_entry_csr_##TT##_coo(struct futhark_context *ctx, struct futhark_i64_1d **out0,     \
                                   struct futhark_i64_1d **out1, struct futhark_##TT##_1d **out2, \
                                   const struct futhark_opaque_csr_##TT *a);                      \
  int futhark_entry_csc_##TT##_coo(struct futhark_context *ctx, struct futhark_i64_1d **out0,     \
                                   struct futhark_i64_1d **out1, struct futhark_##TT##_1d **out2, \
                                   const struct futhark_opaque_csc_##TT *a);                      \
  /* sr.+ :179-180, sr.- :182-183 / sc.+ :217, sc.- :218 */                                       \
  int futhark_entry_csr_##TT##_add(struct futhark_context *ctx,                                   \
                                   struct futhark_opaque_csr_##TT **out0,                         \
                                   const struct futhark_opaque_csr_##TT *a,                       \
                                   const struct futhark_opaque_csr_##TT *b);                      \
  int futhark_entry_csr_##TT##_sub(struct futhark_context *ctx,                                   \
                                   struct futhark_opaque_csr_##TT **out0,                         \
                                   const struct futhark_opaque_csr_##TT *a,                       \
                                   const struct futhark_opaque_csr_##TT *b);                      \
  int futhark_entry_csc_##TT##_add(struct futhark_context *ctx,                                   \
                                   struct futhark_opaque_csc_##TT **out0,                         \
                                   const struct futhark_opaque_csc_##TT *a,                       \
                                   const struct futhark_opaque_csc_##TT *b);                      \
  int futhark_entry_csc_##TT##_sub(struct futhark_context *ctx,                                   \
                                   struct futhark_opaque_csc_##TT **out0,                         \
                                   const struct futhark_opaque_csc_##TT *a,                       \
                                   const struct futhark_opaque_csc_##TT *b);                      \
  /* sr.transpose :185-186 / sc.transpose :220-221: re-labels, moves no data (the new handle   */ \
  /* shares storage with its argument; free both).                                              */\
  int futhark_entry_csr_##TT##_transpose(struct futhark_context *ctx,                             \
                                         struct futhark_opaque_csc_##TT **out0,                   \
                                         const struct futhark_opaque_csr_##TT *a);                \
  int futhark_entry_csc_##TT##_transpose(struct futhark_context *ctx,                             \
                                         struct futhark_opaque_csr_##TT **out0,                   \
                                         const struct futhark_opaque_csc_##TT *a);                \
  /* sr.smvm :134-146:  y[n] = A[n][m] x[m] */                                                    \
  int futhark_entry_csr_##TT##_smvm(struct futhark_context *ctx, struct futhark_##TT##_1d **out0, \
                                    const struct futhark_opaque_csr_##TT *a,                      \
                                    const struct futhark_##TT##_1d *x);                           \
  /* sc.vsmm :223-224:  out[m] = a[n] B[n][m] = sr.smvm (transpose B) a */                        \
  int futhark_entry_csc_##TT##_vsmm(struct futhark_context *ctx, struct futhark_##TT##_1d **out0, \
                                    const struct futhark_##TT##_1d *a,                            \
                                    const struct futhark_opaque_csc_##TT *b);                     \
  /* sparse x dense panel.  Not a member of `compressed`; defined as the column-wise smvm      */ \
  /* C[:,j] = sr.smvm A B[:,j] (:134-146; precedent mono.sr.dmsmm, S/mono.fut:161-162).        */ \
  int futhark_entry_csr_##TT##_smm(struct futhark_context *ctx, struct futhark_##TT##_2d **out0,  \
                                   const struct futhark_opaque_csr_##TT *a,                       \
                                   const struct futhark_##TT##_2d *b);                            \
  /* physical CSR(A) -> CSC(A) = sc.sparse n m (sr.coo A)  (:166-177 then :211-212), and back   */\
  /* CSC(A) -> CSR(A) = sr.sparse n m (sc.coo A)  (:208-209 then :154-160).                     */\
  int futhark_entry_csr_##TT##_to_csc(struct futhark_context *ctx,                                \
                                      struct futhark_opaque_csc_##TT **out0,                      \
                                      const struct futhark_opaque_csr_##TT *a);                   \
  int futhark_entry_csc_##TT##_to_csr(struct futhark_context *ctx,                                \
                                      struct futhark_opaque_csr_##TT **out0,                      \
                                      const struct futhark_opaque_csc_##TT *a);                   \
  /* smsmm :268-331: sr[n][m] -> sc[m][k] -> sr[n][k] */                                          \
  int futhark_entry_smsmm_##TT(struct futhark_context *ctx, struct futhark_opaque_csr_##TT **out0,\
                               const struct futhark_opaque_csr_##TT *a,                           \
                               const struct futhark_opaque_csc_##TT *b);                          \
                                                                                                  \
  /* ---- (3) extensions: no counterpart in the generated API ------------------------------- */  \
  /* Stored shape and stored entry count of the underlying CSR record (for a csc handle: of   */  \
  /* the transposed record).                                                                   */ \
  int sparse_amd_csr_##TT##_dims(struct futhark_context *ctx,                                     \
                                 const struct futhark_opaque_csr_##TT *a, int64_t *n, int64_t *m, \
                                 int64_t *stored);                                                \
  int sparse_amd_csc_##TT##_dims(struct futhark_context *ctx,                                     \
                                 const struct futhark_opaque_csc_##TT *a, int64_t *n, int64_t *m, \
                                 int64_t *stored);                                                \
  /* The record fields in the reference's convention (S/compressed.fut:93-96): row_off[n]     */  \
  /* inclusive, col_idx[nnz] as i64, vals[nnz].  The module ascription hides them in the      */  \
  /* reference; parity tests need them to compare index arrays bit for bit.                   */  \
  int sparse_amd_csr_##TT##_fields(struct futhark_context *ctx, struct futhark_i64_1d **row_off,  \
                                   struct futhark_i64_1d **col_idx,                               \
                                   struct futhark_##TT##_1d **vals,                               \
                                   const struct futhark_opaque_csr_##TT *a);                      \
  int sparse_amd_csc_##TT##_fields(struct futhark_context *ctx, struct futhark_i64_1d **row_off,  \
                                   struct futhark_i64_1d **col_idx,                               \
                                   struct futhark_##TT##_1d **vals,                               \
                                   const struct futhark_opaque_csc_##TT *a);                      \
  /* Adopt an already-normalised record (row_off[n] inclusive, col_idx strictly increasing    */  \
  /* within each row): how a row-sharded rank builds its slice without re-sorting.  Checked:  */  \
  /* lengths, monotone row_off, 0 <= col < m.                                                  */ \
  int sparse_amd_csr_##TT##_from_fields(struct futhark_context *ctx,                              \
                                        struct futhark_opaque_csr_##TT **out0, const int64_t n,   \
                                        const int64_t m, const struct futhark_i64_1d *row_off,    \
                                        const struct futhark_i64_1d *col_idx,                     \
                                        const struct futhark_##TT##_1d *vals);               \
  /* sr.smvm (:134-146) into caller-owned storage, for loops that must not create an array per */ \
  /* product (the row-sharded multi-GPU step).  rows == NULL: y[i] = (A x)[i], y has A's n      */ \
  /* elements.  rows != NULL (n distinct indices into y): y[rows[i]] += (A x)[i] -- how a rank  */ \
  /* adds the part of its rows that multiplies x entries received from other ranks (small       */ \
  /* records: one launch, a row summed sub-wavefront-wise, i.e. in another order than smvm).    */ \
  int sparse_amd_csr_##TT##_smvm_into(struct futhark_context *ctx, struct futhark_##TT##_1d *y,   \
                                      const struct futhark_opaque_csr_##TT *a,                    \
                                      const struct futhark_##TT##_1d *x,                          \
                                      const struct futhark_i64_1d *rows);                         \
  /* No counterpart in the reference.  For callers that cannot allocate device memory (code     */\
  /* under HIP graph capture, tight serving loops, harnesses that forbid hipMalloc): y = A x    */\
  /* as smvm_into with rows == NULL, but the call allocates nothing -- no hipMalloc, no pool    */\
  /* request.  The per-tile partial sums of rows that cross tile ends go to a static device     */\
  /* array of 4 MiB instead of the record's own, so the record may hold at most                 */\
  /* 4 MiB / sizeof(element) * 1024 stored entries (f64: 5.4e8, f32 / i32: 1.07e9); larger      */\
  /* records are refused with an error.  It runs the one-pass streaming kernel on what the      */\
  /* record already holds (16-bit columns / row offsets only if an earlier ordinary product     */\
  /* built them).  It never waits for the stream either: on a record no ordinary product has    */\
  /* seen yet it does not read the plan's statistics back but zero-fills y and keeps the        */\
  /* fix-up launch, so the call is legal while the context's stream is being captured.          */\
  /* All calls on one GPU share that array: calls that overlap on one GPU (two                  */\
  /* contexts or streams) race; calls on one context are ordered by its stream.                 */\
  int sparse_amd_csr_##TT##_smvm_into_noalloc(struct futhark_context *ctx,                        \
                                              struct futhark_##TT##_1d *y,                        \
                                              const struct futhark_opaque_csr_##TT *a,            \
                                              const struct futhark_##TT##_1d *x);                 \
  /* No counterpart in the reference (its smvm, :134-146, keeps no state between calls).  How    */\
  /* many products the caller will run with this matrix.  A record's faster SpMV forms -- 16-bit */\
  /* tile-relative indices for banded / stencil records, the two-pass copy for gather-bound      */\
  /* ones -- are second copies that cost 10 to 30 products' worth of time to build.  Without a   */\
  /* hint a record is served by kernels that need nothing built until it has been multiplied 16  */\
  /* times, and builds then.  expected_products >= 16: decided and built now, inside this call,  */\
  /* so the first product already runs at its steady state; 1..15: nothing is ever built for     */\
  /* this record (until a later call says otherwise).  Results of the forms differ in summation  */\
  /* order only (within the f64 / f32 bars, equal for i32).  csc: the same for vsmm (:223-224).  */\
  int sparse_amd_csr_##TT##_prepare(struct futhark_context *ctx,                                  \
                                    const struct futhark_opaque_csr_##TT *a,                      \
                                    const int64_t expected_products);                             \
  int sparse_amd_csc_##TT##_prepare(struct futhark_context *ctx,                                  \
                                    const struct futhark_opaque_csc_##TT *a,                      \
                                    const int64_t expected_products);

SPARSE_AMD_DECL_MATRIX(f64, double)
SPARSE_AMD_DECL_MATRIX(f32, float)
SPARSE_AMD_DECL_MATRIX(i32, int32_t)

/* ----------------------- (1) the reference's own entries (mk_compressed i32)
 * Names and argument order are what `futhark c --library compressed_test.fut`
 * generates for the entry definitions cited on each line.
 */
/* S/compressed_test.fut:30-31 */
int futhark_entry_test_csr_eye(struct futhark_context *ctx, struct futhark_i32_2d **out0,
                               const int64_t in0, const int64_t in1);
/* S/compressed_test.fut:44-45 */
int futhark_entry_test_csr_sparse(struct futhark_context *ctx, struct futhark_i32_2d **out0,
                                  const int64_t in0, const int64_t in1,
                                  const struct futhark_i64_1d *in2, const struct futhark_i64_1d *in3,
                                  const struct futhark_i32_1d *in4);
/* S/compressed_test.fut:57-59 (in5 is consumed: `*[m]csr.t`) */
int futhark_entry_test_csr_smvm(struct futhark_context *ctx, struct futhark_i32_1d **out0,
                                const int64_t in0, const int64_t in1,
                                const struct futhark_i64_1d *in2, const struct futhark_i64_1d *in3,
                                const struct futhark_i32_1d *in4, const struct futhark_i32_1d *in5);
/* S/compressed_test.fut:68-69 */
int futhark_entry_test_csr_nnz(struct futhark_context *ctx, int64_t *out0, const int64_t in0,
                               const int64_t in1, const struct futhark_i64_1d *in2,
                               const struct futhark_i64_1d *in3, const struct futhark_i32_1d *in4);
/* S/compressed_test.fut:76-78 */
int futhark_entry_test_csr_coo(struct futhark_context *ctx, struct futhark_i64_1d **out0,
                               struct futhark_i64_1d **out1, struct futhark_i32_1d **out2,
                               const int64_t in0, const int64_t in1,
                               const struct futhark_i64_1d *in2, const struct futhark_i64_1d *in3,
                               const struct futhark_i32_1d *in4);
/* S/compressed_test.fut:104-105 */
int futhark_entry_test_csc_eye(struct futhark_context *ctx, struct futhark_i32_2d **out0,
                               const int64_t in0, const int64_t in1);
/* S/compressed_test.fut:118-119 */
int futhark_entry_test_csc_sparse(struct futhark_context *ctx, struct futhark_i32_2d **out0,
                                  const int64_t in0, const int64_t in1,
                                  const struct futhark_i64_1d *in2, const struct futhark_i64_1d *in3,
                                  const struct futhark_i32_1d *in4);
/* S/compressed_test.fut:128-129 */
int futhark_entry_test_csc_nnz(struct futhark_context *ctx, int64_t *out0, const int64_t in0,
                               const int64_t in1, const struct futhark_i64_1d *in2,
                               const struct futhark_i64_1d *in3, const struct futhark_i32_1d *in4);
/* S/compressed_test.fut:136-138 */
int futhark_entry_test_csc_coo(struct futhark_context *ctx, struct futhark_i64_1d **out0,
                               struct futhark_i64_1d **out1, struct futhark_i32_1d **out2,
                               const int64_t in0, const int64_t in1,
                               const struct futhark_i64_1d *in2, const struct futhark_i64_1d *in3,
                               const struct futhark_i32_1d *in4);
/* S/compressed_test.fut:145-147 */
int futhark_entry_test_csr_transpose(struct futhark_context *ctx, struct futhark_i32_2d **out0,
                                     const int64_t in0, const int64_t in1,
                                     const struct futhark_i64_1d *in2,
                                     const struct futhark_i64_1d *in3,
                                     const struct futhark_i32_1d *in4);
/* S/compressed_test.fut:154-156 */
int futhark_entry_test_csc_transpose(struct futhark_context *ctx, struct futhark_i32_2d **out0,
                                     const int64_t in0, const int64_t in1,
                                     const struct futhark_i64_1d *in2,
                                     const struct futhark_i64_1d *in3,
                                     const struct futhark_i32_1d *in4);
/* S/compressed_test.fut:172-178 */
int futhark_entry_test_smsmm(struct futhark_context *ctx, struct futhark_i32_2d **out0,
                             const int64_t in0, const int64_t in1, const int64_t in2,
                             const struct futhark_i64_1d *in3, const struct futhark_i64_1d *in4,
                             const struct futhark_i32_1d *in5, const struct futhark_i64_1d *in6,
                             const struct futhark_i64_1d *in7, const struct futhark_i32_1d *in8);

/* ---------------------------------------------------- (4) mono sparse matrices
 * TT in {f64, f32, i32}  <->  `module mo = mk_mono TT` (S/mono.fut:61): at most one stored
 * element per row (msr) or per column (msc).  futhark_opaque_msr_TT is mo.sr[n][m]
 * (record col_idx[n], vals[n], S/mono.fut:95); futhark_opaque_msc_TT is mo.sc[n][m], whose
 * storage is the msr record of the m x n transpose (S/mono.fut:203).  SURVEY.md 8(f) row 3.
 */
#define SPARSE_AMD_DECL_MONO(TT, CT)                                                              \
  struct futhark_opaque_msr_##TT;                                                                 \
  struct futhark_opaque_msc_##TT;                                                                 \
  int futhark_free_opaque_msr_##TT(struct futhark_context *ctx, struct futhark_opaque_msr_##TT *o);\
  int futhark_free_opaque_msc_##TT(struct futhark_context *ctx, struct futhark_opaque_msc_##TT *o);\
  /* sparse (S/mono.fut:119-129; sc: :188-189).  Non-zero return for an index out of range  */    \
  /* and for two elements in one row (one column for msc) -- the reference's two asserts.    */   \
  int futhark_entry_msr_##TT##_sparse(struct futhark_context *ctx,                                \
                                      struct futhark_opaque_msr_##TT **out0, const int64_t n,     \
                                      const int64_t m, const struct futhark_i64_1d *rs,           \
                                      const struct futhark_i64_1d *cs,                            \
                                      const struct futhark_##TT##_1d *vs);                        \
  int futhark_entry_msc_##TT##_sparse(struct futhark_context *ctx,                                \
                                      struct futhark_opaque_msc_##TT **out0, const int64_t n,     \
                                      const int64_t m, const struct futhark_i64_1d *rs,           \
                                      const struct futhark_i64_1d *cs,                            \
                                      const struct futhark_##TT##_1d *vs);                        \
  /* zero :97-100 / :170-171, eye :102-105 / :176-177, diag :107-110 / :179-180 */                \
  int futhark_entry_msr_##TT##_zero(struct futhark_context *ctx,                                  \
                                    struct futhark_opaque_msr_##TT **out0, const int64_t n,       \
                                    const int64_t m);                                             \
  int futhark_entry_msc_##TT##_zero(struct futhark_context *ctx,                                  \
                                    struct futhark_opaque_msc_##TT **out0, const int64_t n,       \
                                    const int64_t m);                                             \
  int futhark_entry_msr_##TT##_eye(struct futhark_context *ctx,                                   \
                                   struct futhark_opaque_msr_##TT **out0, const int64_t n,        \
                                   const int64_t m);                                              \
  int futhark_entry_msc_##TT##_eye(struct futhark_context *ctx,                                   \
                                   struct futhark_opaque_msc_##TT **out0, const int64_t n,        \
                                   const int64_t m);                                              \
  int futhark_entry_msr_##TT##_diag(struct futhark_context *ctx,                                  \
                                    struct futhark_opaque_msr_##TT **out0,                        \
                                    const struct futhark_##TT##_1d *v);                           \
  int futhark_entry_msc_##TT##_diag(struct futhark_context *ctx,                                  \
                                    struct futhark_opaque_msc_##TT **out0,                        \
                                    const struct futhark_##TT##_1d *v);                           \
  /* dense :112-114 / :191-192 */                                                                 \
  int futhark_entry_msr_##TT##_dense(struct futhark_context *ctx, struct futhark_##TT##_2d **out0,\
                                     const struct futhark_opaque_msr_##TT *a);                    \
  int futhark_entry_msc_##TT##_dense(struct futhark_context *ctx, struct futhark_##TT##_2d **out0,\
                                     const struct futhark_opaque_msc_##TT *a);                    \
  /* scale :116-117 / :173-174 */                                                                 \
  int futhark_entry_msr_##TT##_scale(struct futhark_context *ctx,                                 \
                                     struct futhark_opaque_msr_##TT **out0, const CT v,           \
                                     const struct futhark_opaque_msr_##TT *a);                    \
  int futhark_entry_msc_##TT##_scale(struct futhark_context *ctx,                                 \
                                     struct futhark_opaque_msc_##TT **out0, const CT v,           \
                                     const struct futhark_opaque_msc_##TT *a);                    \
  /* nnz :131-133 / :182-183 (stored values that are not zero) */                                 \
  int futhark_entry_msr_##TT##_nnz(struct futhark_context *ctx, int64_t *out0,                    \
                                   const struct futhark_opaque_msr_##TT *a);                      \
  int futhark_entry_msc_##TT##_nnz(struct futhark_context *ctx, int64_t *out0,                    \
                                   const struct futhark_opaque_msc_##TT *a);                      \
  /* coo :135-137 / :185-186 (zero values are filtered out, unlike compressed) */                 \
  int futhark_entry_msr_##TT##_coo(struct futhark_context *ctx, struct futhark_i64_1d **out0,     \
                                   struct futhark_i64_1d **out1, struct futhark_##TT##_1d **out2, \
                                   const struct futhark_opaque_msr_##TT *a);                      \
  int futhark_entry_msc_##TT##_coo(struct futhark_context *ctx, struct futhark_i64_1d **out0,     \
                                   struct futhark_i64_1d **out1, struct futhark_##TT##_1d **out2, \
                                   const struct futhark_opaque_msc_##TT *a);                      \
  /* + and - :139-149 / :194-195: non-zero return when the operands' col_idx differ */            \
  int futhark_entry_msr_##TT##_add(struct futhark_context *ctx,                                   \
                                   struct futhark_opaque_msr_##TT **out0,                         \
                                   const struct futhark_opaque_msr_##TT *a,                       \
                                   const struct futhark_opaque_msr_##TT *b);                      \
  int futhark_entry_msr_##TT##_sub(struct futhark_context *ctx,                                   \
                                   struct futhark_opaque_msr_##TT **out0,                         \
                                   const struct futhark_opaque_msr_##TT *a,                       \
                                   const struct futhark_opaque_msr_##TT *b);                      \
  int futhark_entry_msc_##TT##_add(struct futhark_context *ctx,                                   \
                                   struct futhark_opaque_msc_##TT **out0,                         \
                                   const struct futhark_opaque_msc_##TT *a,                       \
                                   const struct futhark_opaque_msc_##TT *b);                      \
  int futhark_entry_msc_##TT##_sub(struct futhark_context *ctx,                                   \
                                   struct futhark_opaque_msc_##TT **out0,                         \
                                   const struct futhark_opaque_msc_##TT *a,                       \
                                   const struct futhark_opaque_msc_##TT *b);                      \
  /* transpose :151-152 / :197-198: no data moves, the handle is re-labelled */                   \
  int futhark_entry_msr_##TT##_transpose(struct futhark_context *ctx,                             \
                                         struct futhark_opaque_msc_##TT **out0,                   \
                                         const struct futhark_opaque_msr_##TT *a);                \
  int futhark_entry_msc_##TT##_transpose(struct futhark_context *ctx,                             \
                                         struct futhark_opaque_msr_##TT **out0,                   \
                                         const struct futhark_opaque_msc_##TT *a);                \
  /* smvm :154-155 */                                                                             \
  int futhark_entry_msr_##TT##_smvm(struct futhark_context *ctx, struct futhark_##TT##_1d **out0, \
                                    const struct futhark_opaque_msr_##TT *a,                      \
                                    const struct futhark_##TT##_1d *v);                           \
  /* vsmm :157-159 (msr: scatter-add, summed per column in ascending row order) / :200-201 */     \
  int futhark_entry_msr_##TT##_vsmm(struct futhark_context *ctx, struct futhark_##TT##_1d **out0, \
                                    const struct futhark_##TT##_1d *v,                            \
                                    const struct futhark_opaque_msr_##TT *a);                     \
  int futhark_entry_msc_##TT##_vsmm(struct futhark_context *ctx, struct futhark_##TT##_1d **out0, \
                                    const struct futhark_##TT##_1d *a,                            \
                                    const struct futhark_opaque_msc_##TT *b);                     \
  /* dmsmm :161-162: dense [n][k] times msr[k][m] -> dense [n][m] */                              \
  int futhark_entry_msr_##TT##_dmsmm(struct futhark_context *ctx, struct futhark_##TT##_2d **out0,\
                                     const struct futhark_##TT##_2d *d,                           \
                                     const struct futhark_opaque_msr_##TT *s);                    \
  /* extension (no counterpart in the generated API): the record fields col_idx[n], vals[n] */    \
  /* (for an msc handle: of the transposed record), for bit-for-bit parity tests.           */    \
  int sparse_amd_msr_##TT##_fields(struct futhark_context *ctx, struct futhark_i64_1d **col_idx,  \
                                   struct futhark_##TT##_1d **vals,                               \
                                   const struct futhark_opaque_msr_##TT *a);                      \
  int sparse_amd_msc_##TT##_fields(struct futhark_context *ctx, struct futhark_i64_1d **col_idx,  \
                                   struct futhark_##TT##_1d **vals,                               \
                                   const struct futhark_opaque_msc_##TT *a);

SPARSE_AMD_DECL_MONO(f64, double)
SPARSE_AMD_DECL_MONO(f32, float)
SPARSE_AMD_DECL_MONO(i32, int32_t)

/* The reference's own entries for mono (mk_mono i32, S/mono_test.fut:5). */
#define SPARSE_AMD_COO_ARGS                                                                       \
  const int64_t in0, const int64_t in1, const struct futhark_i64_1d *in2,                         \
      const struct futhark_i64_1d *in3, const struct futhark_i32_1d *in4
/* S/mono_test.fut:30-31 */
int futhark_entry_test_msr_eye(struct futhark_context *ctx, struct futhark_i32_2d **out0,
                               const int64_t in0, const int64_t in1);
/* S/mono_test.fut:42-43 */
int futhark_entry_test_msr_sparse(struct futhark_context *ctx, struct futhark_i32_2d **out0,
                                  SPARSE_AMD_COO_ARGS);
/* S/mono_test.fut:55-57 (in5 is consumed) */
int futhark_entry_test_msr_smvm(struct futhark_context *ctx, struct futhark_i32_1d **out0,
                                SPARSE_AMD_COO_ARGS, const struct futhark_i32_1d *in5);
/* S/mono_test.fut:66-67 */
int futhark_entry_test_msr_nnz(struct futhark_context *ctx, int64_t *out0, SPARSE_AMD_COO_ARGS);
/* S/mono_test.fut:74-76 */
int futhark_entry_test_msr_coo(struct futhark_context *ctx, struct futhark_i64_1d **out0,
                               struct futhark_i64_1d **out1, struct futhark_i32_1d **out2,
                               SPARSE_AMD_COO_ARGS);
/* S/mono_test.fut:87-89: (n, m, v[n], xs, ys, vs) */
int futhark_entry_test_msr_vsmm(struct futhark_context *ctx, struct futhark_i32_1d **out0,
                                const int64_t in0, const int64_t in1,
                                const struct futhark_i32_1d *in2, const struct futhark_i64_1d *in3,
                                const struct futhark_i64_1d *in4, const struct futhark_i32_1d *in5);
/* S/mono_test.fut:114-115 */
int futhark_entry_test_msc_eye(struct futhark_context *ctx, struct futhark_i32_2d **out0,
                               const int64_t in0, const int64_t in1);
/* S/mono_test.fut:126-127 */
int futhark_entry_test_msc_sparse(struct futhark_context *ctx, struct futhark_i32_2d **out0,
                                  SPARSE_AMD_COO_ARGS);
/* S/mono_test.fut:136-137 */
int futhark_entry_test_msc_nnz(struct futhark_context *ctx, int64_t *out0, SPARSE_AMD_COO_ARGS);
/* S/mono_test.fut:144-146 */
int futhark_entry_test_msc_coo(struct futhark_context *ctx, struct futhark_i64_1d **out0,
                               struct futhark_i64_1d **out1, struct futhark_i32_1d **out2,
                               SPARSE_AMD_COO_ARGS);
/* S/mono_test.fut:153-155 */
int futhark_entry_test_msr_transpose(struct futhark_context *ctx, struct futhark_i32_2d **out0,
                                     SPARSE_AMD_COO_ARGS);
/* S/mono_test.fut:162-164 */
int futhark_entry_test_msc_transpose(struct futhark_context *ctx, struct futhark_i32_2d **out0,
                                     SPARSE_AMD_COO_ARGS);

/* ------------------------------------------- (5) Matrix Market loader (host side)
 * No counterpart in the reference, which has no file format: its inputs only arrive as entry-point
 * arrays.  SURVEY.md 8(f) row 4: the step in front of `sparse`.  Reads a `coordinate` file
 * (real | integer | pattern; general | symmetric | skew-symmetric) into 0-based i64 triples in file
 * order, symmetric files expanded; `threads` > 1 parses the body in parallel.  The three arrays are
 * malloc'ed: release each with sparse_amd_mtx_free.  On failure returns non-zero and, if `error` is
 * not NULL, a malloc'ed message the caller frees.  No GPU is touched. */
int sparse_amd_mtx_read(const char *path, int threads, int64_t *n, int64_t *m, int64_t *count,
                        int64_t **rows, int64_t **cols, double **vals, char **error);
/* Writes `coordinate real general` with 17 significant digits (every f64 round-trips). */
int sparse_amd_mtx_write(const char *path, int64_t n, int64_t m, int64_t count, const int64_t *rows,
                         const int64_t *cols, const double *vals, char **error);
void sparse_amd_mtx_free(void *p);

/* ------------------------------------- (6) one process, several devices (native multi-GPU)
 * No counterpart in the reference (Futhark targets one device; SURVEY.md 8b "Threading", 8e).  A group owns one
 * context per device; a distributed matrix holds contiguous row blocks of nearly equal triple counts, member k's
 * block being an ordinary futhark_opaque_csr_f64 of member k's context (global column numbers), and the members'
 * records are, bit for bit, the row blocks of the record one device would build (triples reach their owner in
 * input order).  y = A x: every member's slice of x goes to every member -- grouped ncclSend / ncclRecv over RCCL,
 * all pairs at once (transport "rccl": librccl is opened with dlopen, devices must be distinct), or direct peer
 * copies ordered by events (transport "peer"; also how several members rehearse on ONE device) -- then every member
 * runs sr.smvm (S/compressed.fut:134-146) on its rows.  transport == NULL: rccl when there are several distinct
 * devices and the library loads, else peer.  A group of ONE member named "rccl" opens librccl too and moves its slice
 * of x by a grouped ncclSend / ncclRecv to itself (the transport's code path on a one-GPU machine).  x is cut like the rows when n == m, else into equal slices.  Calls on one group
 * come from one host thread.  All functions return 0 or non-zero with the text in sparse_amd_group_get_error
 * (heap string, caller frees); sparse_amd_group_new always returns a group object to read that text from. */
struct sparse_amd_group;
struct sparse_amd_dcsr_f64;
struct sparse_amd_dvec_f64;
int sparse_amd_group_new(struct sparse_amd_group **out, int ndev, const int *devices /* NULL: 0..ndev-1 */,
                         const char *transport);
void sparse_amd_group_free(struct sparse_amd_group *g);
char *sparse_amd_group_get_error(struct sparse_amd_group *g);
int sparse_amd_group_size(struct sparse_amd_group *g);
const char *sparse_amd_group_transport(struct sparse_amd_group *g);   /* "rccl", "peer" or "none" (one member, no RCCL) */
struct futhark_context *sparse_amd_group_context(struct sparse_amd_group *g, int k);
int sparse_amd_group_sync(struct sparse_amd_group *g);
/* sr.sparse n m coo (S/compressed.fut:154-160) from host triples, rows dealt to the members. */
int sparse_amd_dcsr_f64_sparse(struct sparse_amd_group *g, struct sparse_amd_dcsr_f64 **out, int64_t n, int64_t m,
                               const int64_t *rs, const int64_t *cs, const double *vs, int64_t count);
int sparse_amd_dcsr_f64_free(struct sparse_amd_group *g, struct sparse_amd_dcsr_f64 *A);
/* ndev + 1 bounds each; either pointer may be NULL */
int sparse_amd_dcsr_f64_bounds(struct sparse_amd_group *g, const struct sparse_amd_dcsr_f64 *A, int64_t *row_bounds,
                               int64_t *col_bounds);
/* member k's row block (owned by A; use it with sparse_amd_group_context(g, k)) */
struct futhark_opaque_csr_f64 *sparse_amd_dcsr_f64_member(struct sparse_amd_group *g,
                                                          const struct sparse_amd_dcsr_f64 *A, int k);
/* a vector cut like A's columns (like_rows == 0) or rows (like_rows != 0); host may be NULL */
int sparse_amd_dvec_f64_new(struct sparse_amd_group *g, struct sparse_amd_dvec_f64 **out,
                            const struct sparse_amd_dcsr_f64 *A, int like_rows, const double *host);
int sparse_amd_dvec_f64_values(struct sparse_amd_group *g, const struct sparse_amd_dvec_f64 *v, double *host);
int sparse_amd_dvec_f64_free(struct sparse_amd_group *g, struct sparse_amd_dvec_f64 *v);
void *sparse_amd_dvec_f64_member_ptr(struct sparse_amd_group *g, const struct sparse_amd_dvec_f64 *v, int k,
                                     int64_t *len);
int sparse_amd_dcsr_f64_smvm(struct sparse_amd_group *g, struct sparse_amd_dvec_f64 *y,
                             const struct sparse_amd_dcsr_f64 *A, const struct sparse_amd_dvec_f64 *x);

/* ------------------------------- (7) token records: products of a language model's sparse matrices
 * No counterpart in the reference.  Neighbours of mono (S/mono.fut:95: one stored element per row, col_idx[n] and vals[n]) and of
 * smm for the records a language model makes anew at every step, given by their column indices alone:
 *   - a lookup is a mono record times a panel: n token ids (col_idx), optional values f[n], one scale s for all;
 *   - a routing is a record of K elements per row: each token's K chosen experts.  `route` gives every choice a place such
 *     that an expert's places lie side by side, in the order of the batch; dispatch and combine are the products with that
 *     permutation and with its weighted transpose, experts the product with the block-diagonal matrix of the experts' blocks.
 * Conventions of this group, where they differ from the rest of this header:
 *   - arguments are plain device pointers; a panel of rows has a row stride (`ld...`, in elements) and no alignment beyond its
 *     elements'.  The rows of a result lie apart (ld >= width); rows that are only read may have any stride, zero included;
 *   - every call names the HIP stream it runs on (NULL: the null stream) and touches neither the context's stream nor its
 *     memory: it allocates nothing, never waits, keeps nothing between calls, and may be captured into a graph.  What needs
 *     a workspace takes it as an argument (256-byte aligned, at least ..._workspace bytes that no other argument shares,
 *     free for other use when the stream has passed the call; contents do not matter).  The calling thread's current device is left as it was;
 *   - `type` is the element type of the panels: SPARSE_AMD_F32, SPARSE_AMD_F16, SPARSE_AMD_BF16 (experts...: the 16-bit ones).
 *     Sums are held in 32 bits and rounded once; values, weights and their gradients are 32-bit floats;
 *   - indices that come in have `id_bits` = 32 or 64 bits.  An id outside 0 .. V-1, or an expert outside 0 .. X-1, selects
 *     nothing: a row of zeros, no place (pos = -1), no gradient;
 *   - results are the same bits on every call with the same arguments.  A row of an experts' product may differ in its last
 *     bits where the other rows of the batch differ: they decide which workgroup adds it, and where it begins;
 *   - a result may not overlap another result or an argument, nor lie between its rows.
 * Errors: as everywhere in this header (non-zero, text in futhark_context_get_error); nothing is launched then. */
#define SPARSE_AMD_F32 0
#define SPARSE_AMD_F16 1
#define SPARSE_AMD_BF16 2
/* y[i] = scale vals[i] table[ids[i]], i < n; vals may be NULL (ones). */
int sparse_amd_tokens_lookup(struct futhark_context *ctx, void *stream, int type, void *y, int64_t ldy, const void *table,
                             int64_t V, int64_t D, int64_t ldt, const void *ids, int id_bits, int64_t n,
                             const float *vals, float scale);
/* dvals[i] = scale <dy[i], table[ids[i]]>: lookup's gradient by vals. */
int sparse_amd_tokens_lookup_dots(struct futhark_context *ctx, void *stream, int type, float *dvals, const void *dy,
                                  int64_t ldy, const void *table, int64_t V, int64_t D, int64_t ldt, const void *ids,
                                  int id_bits, int64_t n, float scale);
/* dtable[v] = sum over i with ids[i] = v of scale vals[i] dy[i], added in an order that the ids, their number, the type and the
 * width decide: lookup's gradient by the table.
 * accumulate = 0: every row of dtable is written (zeros where no id names it); else the sums are added to dtable, and rows
 * no id names are not touched.  out_type: type or SPARSE_AMD_F32.  V and n are at most 2^31 - 2. */
int sparse_amd_tokens_lookup_grad(struct futhark_context *ctx, void *stream, int type, int out_type, int accumulate,
                                  void *dtable, int64_t V, int64_t D, int64_t ldt, const void *dy, int64_t ldy,
                                  const void *ids, int id_bits, int64_t n, const float *vals, float scale, void *work,
                                  int64_t work_bytes);
int64_t sparse_amd_tokens_lookup_grad_workspace(int type, int64_t n, int64_t V, int64_t D);
/* chosen[n], n = tokens * K: the experts of all tokens, X <= 1024 experts.  pos[i] = place of choice i or -1; src[p] = the
 * choice at place p, -1 behind the last; offsets[X + 1]: expert e's places are offsets[e] .. offsets[e + 1] - 1.  The same
 * expert twice in a token is two choices. */
int sparse_amd_tokens_route(struct futhark_context *ctx, void *stream, const void *chosen, int id_bits, int64_t n, int64_t X,
                            int32_t *pos, int32_t *src, int32_t *offsets, void *work, int64_t work_bytes);
int64_t sparse_amd_tokens_route_workspace(int64_t n, int64_t X);
/* xs[pos[t, j]] = weights[t, j] x[t], t < n, j < K; weights may be NULL (ones).  Rows of xs without a choice are left as
 * they are.  Also the gradient of combine without weights. */
int sparse_amd_tokens_dispatch(struct futhark_context *ctx, void *stream, int type, void *xs, int64_t ldxs, int64_t slots,
                               const void *x, int64_t ldx, int64_t n, int64_t D, int64_t K, const int32_t *pos,
                               const float *weights);
/* y[t] = sum over j of weights[t, j] ys[pos[t, j]], in the order of j; weights may be NULL (ones).  A token without a place
 * has a row of zeros; rows of ys without a choice are not read.  Also the gradient of dispatch. */
int sparse_amd_tokens_combine(struct futhark_context *ctx, void *stream, int type, void *y, int64_t ldy, const void *ys,
                              int64_t ldys, int64_t slots, int64_t n, int64_t D, int64_t K, const int32_t *pos,
                              const float *weights);
/* combine's gradient: dys[pos[t, j]] = weights[t, j] dy[t] (rows without a choice are left as they are) and
 * dweights[t, j] = <dy[t], ys[pos[t, j]]> (0 where there is no place). */
int sparse_amd_tokens_combine_grad(struct futhark_context *ctx, void *stream, int type, void *dys, int64_t lddys,
                                   float *dweights, const void *dy, int64_t lddy, const void *ys, int64_t ldys,
                                   int64_t slots, int64_t n, int64_t D, int64_t K, const int32_t *pos,
                                   const float *weights);
/* ys[r] = w[e] xs[r] for the rows r = offsets[e] .. offsets[e + 1] - 1 of every expert e; w[e] is F x D with rows `ldw` apart, the
 * blocks `blockw` apart.  Rows from offsets[X] on are neither read nor written. */
int sparse_amd_tokens_experts(struct futhark_context *ctx, void *stream, int type, void *ys, int64_t ldy, const void *xs,
                              int64_t ldx, int64_t rows, const void *w, int64_t X, int64_t F, int64_t D, int64_t ldw,
                              int64_t blockw, const int32_t *offsets);
/* its gradients: dxs[r] = w[e]^T dys[r], and dw[e] = sum over e's rows of dys[r] xs[r]^T (accumulate, out_type: as in
 * lookup_grad; an expert without rows has a block of zeros, or is left as it is). */
int sparse_amd_tokens_experts_grad_x(struct futhark_context *ctx, void *stream, int type, void *dxs, int64_t ldx,
                                     const void *dys, int64_t ldy, int64_t rows, const void *w, int64_t X, int64_t F,
                                     int64_t D, int64_t ldw, int64_t blockw, const int32_t *offsets);
int sparse_amd_tokens_experts_grad_w(struct futhark_context *ctx, void *stream, int type, int out_type, int accumulate,
                                     void *dw, int64_t X, int64_t F, int64_t D, int64_t ldw, int64_t blockw,
                                     const void *dys, int64_t ldy, const void *xs, int64_t ldx, int64_t rows,
                                     const int32_t *offsets);

/* ------------------------------------------------- (3) context extensions
 * No counterpart in the generated API. */
/* Run all subsequent work on the caller's HIP stream (hipStream_t); the context
 * first drains its current stream.  NULL is the HIP null stream (what torch calls
 * its default stream), not "no stream". */
int sparse_amd_context_set_stream(struct futhark_context *ctx, void *hip_stream);
void *sparse_amd_context_get_stream(struct futhark_context *ctx);
/* Tuning / test overrides.  Keys: "spmv_algo" (0 auto, 1 nnz-split stream,
 * 2 wavefront-per-row, 3 sub-wavefront-per-row), "spmv_lanes" (sub-wavefront
 * width, power of two <= 64), "wide_col" (1: keep col_idx as i64 on device),
 * "spmm_algo" (0 streaming row panels with banded long-row tiles on the matrix cores,
 * 2 plain wavefront-per-row, 3 streaming row panels without the matrix cores), "sort_algo"
 * (assembly's radix sort: 0 one global histogram + look-back, 1 histogram pass per digit),
 * "spmv_reorder" (hot-column renumbering for gather-bound SpMV: 0 decided per record, 1 whenever the
 * record is large enough, -1 never), "spmv_cblk" (column-blocked copy for wide records with flat column
 * popularity: 0 decided per record, W > 0 always, with W columns per block, -1 never).  "spmv_pb" (two-pass SpMV with the
 * x and y slices in LDS: 0 large skewed records of 4-byte values, 1 also flat column popularity, 2 always,
 * -1 never; "spmv_pb_fold": its folded layout, a row's products inside one piece summed in the first pass, 0 and
 * 1 always, -1 never (the plain layout); "spmv_pb_deal": column lines sorted into the blocks by popularity (1), dealt round
 * them (-1), or decided per record (0)), "spmv_col16" (16-bit tile-relative columns for banded / stencil records: 0 decided per record,
 * -1 never), "spmv_eager" (1: every record decides and builds at its first product instead of its 16th; see
 * sparse_amd_csr_*_prepare).  Read-only: "spmv_last_path", "spmv_last_col_bytes" (what the last product ran),
 * "sort_last_msd", "sort_last_long_runs" (what the last assembly did).  The per-record choices are made when a
 * record has been multiplied 16 times, or at once by sparse_amd_csr_*_prepare or an explicit kernel request.
 * Returns non-zero for an unknown key. */
int sparse_amd_context_set_option(struct futhark_context *ctx, const char *key, int64_t value);
int64_t sparse_amd_context_get_option(struct futhark_context *ctx, const char *key);
const char *sparse_amd_version(void);
/* No counterpart in the reference.  What this card sustains for a streaming mix, measured now, on the context's
 * stream: `groups` workgroups each read read_bytes_per_group contiguous bytes (128-bit non-temporal loads, as the
 * SpMV / SpMM kernels stream a tile) and write write_bytes_per_group contiguous bytes (non-temporal stores); no
 * arithmetic.  Both are multiples of 16 (0 = none).  *gb_per_s = moved bytes / median launch time, *us = that time.
 * For quoting a kernel's achieved bandwidth against the measured ceiling of its own access mix next to the data
 * sheet's 8 TB/s (bench.py: roofline.peak_measured).  Allocates its buffers from the context's pool. */
int sparse_amd_context_measure_bandwidth(struct futhark_context *ctx, int64_t read_bytes_per_group,
                                         int64_t write_bytes_per_group, int64_t groups, double *gb_per_s, double *us);

#ifdef __cplusplus
}
#endif
#endif /* SPARSE_AMD_H */
