/*
 * exl3_hip.h -- C-ABI of the MI355X (gfx950) EXL3 packed-weight linear layer.
 *
 * Plain pointers and sizes; every pointer named "device" is HIP device memory
 * owned by the caller.  Work is enqueued on the given stream (0 = the null
 * stream) and the functions return without synchronising unless stated.
 * No function throws; every one returns an exl3_status.
 *
 * Reference interfaces replaced (paths are in the reference checkout):
 *   exl3_hip_mul_mat      <- ggml_exl3_mul_mat        src/exl3-ggml.cpp:51-92,
 *                            declared include/exl3-block.h:46, dispatched from
 *                            ggml_compute_forward_mul_mat (patches/llama-exl3.patch:44-51);
 *                            device twin op_exl3_matmul src/exl3-htp.c:159-232
 *   exl3_hip_mul_mat_nd   <- ggml_exl3_mul_mat with its row_offset addressing of
 *                            ggml views (src/exl3-ggml.cpp:11-17, 64, 88)
 *   exl3_hip_get_rows_nd  <- ggml_exl3_get_rows with its id and row addressing
 *                            (src/exl3-ggml.cpp:34-36)
 *   exl3_hip_iface_matmul <- exl3_iface_matmul src/hexagon/exl3_service.c:265-305
 *                            (IDL src/hexagon/exl3_iface.idl:13-15): the same layer on the
 *                            upstream tile layout with separate su / sv, fp32 in and out
 *   exl3_hip_decode       <- exl3::decode_inner(_slice) src/exl3_codec.cpp:123-145
 *                            (and exl3_iface_decode src/hexagon/exl3_iface.idl:5-7)
 *   exl3_hip_reconstruct  <- exl3::reconstruct(_slice)  src/exl3_codec.cpp:169-204
 *   exl3_hip_get_rows     <- ggml_exl3_get_rows        src/exl3-ggml.cpp:19-49,
 *                            declared include/exl3-block.h:47, dispatched from
 *                            ggml_compute_forward_get_rows (patches/llama-exl3.patch:114-121);
 *                            tied embedding exl3::Model::embedding src/exl3_model.cpp:168-187
 *   exl3_hip_codebook     <- exl3::decode_codebook      src/exl3_codec.cpp:68-86
 *   exl3_hip_hadamard128  <- exl3::hadamard128          src/exl3_codec.cpp:147-167
 *   exl3_hip_pack_records <- record assembly tests/test-exl3-graph.cpp:37-45,
 *                            tools/export_native_gguf.py:27-36
 *   exl3_hip_validate_records <- ggml_validate_row_data EXL3 case
 *                            patches/llama-exl3.patch:327-338
 *   exl3_hip_supports_mul_mat <- supports_op predicates patches/llama-exl3.patch:81-84,225-235
 *   exl3_hip_model_*      <- exl3::Model src/exl3_model.cpp:79-187 (include/exl3_model.h),
 *                            for C callers; the C++ class is include/exl3_model.h
 */
#ifndef EXL3_HIP_H
#define EXL3_HIP_H

#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

#define EXL3_HIP_VERSION 10100u /* major * 10000 + minor * 100 + patch */

typedef enum exl3_status {
    EXL3_OK = 0,
    EXL3_INVAL_PARAMS = 1,       /* shape / rate / codebook / stride rejected (HTP_STATUS_INVAL_PARAMS) */
    EXL3_NO_SUPPORT = 2,         /* valid request this build does not implement (HTP_STATUS_NO_SUPPORT) */
    EXL3_WORKSPACE_TOO_SMALL = 3,/* caller workspace below exl3_hip_mul_mat_workspace_bytes() */
    EXL3_HIP_ERROR = 4           /* a HIP runtime call failed (HTP_STATUS_INTERNAL_ERR) */
} exl3_status;

typedef enum exl3_dtype { EXL3_F32 = 0, EXL3_F16 = 1 } exl3_dtype;

/* codebook ids match exl3::Codebook (include/exl3_codec.h) */
typedef enum exl3_codebook { EXL3_CB_3INST = 0, EXL3_CB_MCG = 1, EXL3_CB_MUL1 = 2 } exl3_codebook;

typedef enum exl3_layout {
    EXL3_LAYOUT_UPSTREAM_TILES = 0, /* [k/16][n/16][16*bits] u16, the .trellis tensor */
    EXL3_LAYOUT_RECORDS = 1         /* 128x128 group records, include/exl3-block.h */
} exl3_layout;

unsigned exl3_hip_version(void);
const char *exl3_hip_status_string(exl3_status status);

/* Largest row count served by the register-decode GEMV kernel (32): a grouped
 * call (exl3_hip_mul_mat_group) of at most this many rows is one GEMV launch.
 * exl3_hip_mul_mat runs the GEMV up to 14 rows (16 when a GEMV workgroup's
 * share of k is short: at most 64 (record, row) blocks to prepare) and the
 * LDS-decode MFMA GEMM kernel above, where the GEMM is the faster of the two. */
size_t exl3_hip_gemv_max_rows(void);

/* 1 when exl3_hip_mul_mat accepts this problem: bits 1..8, codebook 0..2,
 * k and n nonzero multiples of 128, 1 <= rows <= 65536, dtypes F32/F16. */
int exl3_hip_supports_mul_mat(unsigned bits, unsigned codebook, size_t k, size_t n, size_t rows,
                              exl3_dtype xt, exl3_dtype yt);

/* ---- engine-side op predicates (ggml supports_op) ------------------------
 * The reference gates the ggml ops that touch an EXL3 tensor in its CPU
 * backend's supports_op (patches/llama-exl3.patch:81-97).  A HIP backend asks
 * exl3_hip_supports_op with the op's tensors described by plain values:
 *   MUL_MAT    src0 EXL3 (types 43/44/45): ne0 and ne1 multiples of 128, ne2 = ne3 = 1,
 *              src0 contiguous, src1 F32 or F16 (patch:81-84); here also dst F32
 *              and the dimensions exl3_hip_mul_mat accepts
 *   MUL_MAT_ID src0 EXL3: unsupported (patch:92-93)
 *   GET_ROWS   src0 EXL3: ne0 and ne1 multiples of 128, ne2 = ne3 = 1, src1 I32
 *              (patch:94-97); here also dst F32 or F16
 *   CPY        dst or src0 EXL3: only a copy between contiguous tensors of the
 *              same EXL3 type, i.e. a byte copy of group records (patch:71-72)
 *   SET_ROWS   dst or src0 EXL3: unsupported (patch:69-72)
 * Returns 1 (served), 0 (refused: keep the op off this backend) or -1 (no EXL3
 * tensor in the op: not this library's decision). */
typedef enum exl3_op {
    EXL3_OP_MUL_MAT = 0,
    EXL3_OP_MUL_MAT_ID = 1,
    EXL3_OP_GET_ROWS = 2,
    EXL3_OP_CPY = 3,
    EXL3_OP_SET_ROWS = 4
} exl3_op;

/* ggml type ids used by the predicates (ggml.h enum ggml_type of the reference's
 * llama.cpp revision; the EXL3 ids are include/exl3-block.h's 43/44/45) */
#define EXL3_GGML_TYPE_F32 0u
#define EXL3_GGML_TYPE_F16 1u
#define EXL3_GGML_TYPE_I32 26u

typedef struct exl3_tensor_info {
    unsigned type;     /* ggml type id */
    int64_t ne[4];     /* ggml ne[]: ne[0] is the row length */
    int contiguous;    /* ggml_is_contiguous() */
    size_t nb[4];      /* ggml nb[]: byte strides of the four dimensions */
} exl3_tensor_info;

/* dst and src0 are required; src1 is required for MUL_MAT, MUL_MAT_ID and GET_ROWS
 * (NULL there: 0).  Beyond the reference's rules, MUL_MAT and GET_ROWS are served
 * when exl3_hip_mul_mat_nd / exl3_hip_get_rows_nd can address every row of the
 * views as the reference's row_offset does (src/exl3-ggml.cpp:11-17):
 *   MUL_MAT   src1 nb[0] = its element size and nb[1..3] multiples of it;
 *             dst F32, ne = [src0 ne[1], src1 ne[1], src1 ne[2], src1 ne[3]],
 *             nb[0] = 4, nb[1..3] multiples of 4, no two dst rows overlapping
 *   GET_ROWS  src1 (ids) ne[3] = 1 and nb[0..2] multiples of 4; dst ne = [src0
 *             ne[0], src1 ne[0], src1 ne[1], src1 ne[2]], nb[0] = its element
 *             size, nb[1..3] multiples of it, no two dst rows overlapping
 * Anything else touching an EXL3 tensor is refused (0), so no view is ever
 * read or written at addresses other than ggml's. */
int exl3_hip_supports_op(exl3_op op, const exl3_tensor_info *dst, const exl3_tensor_info *src0,
                         const exl3_tensor_info *src1);

/* Device workspace bytes exl3_hip_mul_mat needs for (k, n) at any row count
 * 1..rows.  The workspace starts with the 16 MiB of split-K hand-off words,
 * which every call leaves zero, followed by per-call staging: zero-fill it once
 * before its first use (exl3_hip_workspace_init).  One workspace serves any
 * sequence of calls when it holds at least exl3_hip_mul_mat_workspace_bytes(k,
 * n, rows) of every one of them; calls that share one must not run concurrently
 * (order them on one stream; a call may be several launches, so threads that share one
 * make their calls one at a time.  The internal workspace, NULL, is held by a call until
 * its launches are enqueued).  A GEMV call whose split-K partials would not fit
 * the 16 MiB runs the GEMM path instead (k * n above about 134 M weights at 32
 * rows). */
size_t exl3_hip_mul_mat_workspace_bytes(size_t k, size_t n, size_t rows);
/* Zero-fills workspace_bytes of a caller workspace; NULL: the internal workspace
 * of the current device and this stream, if one exists. */
exl3_status exl3_hip_workspace_init(void *workspace, size_t workspace_bytes, hipStream_t stream);

/* Split-K failure flag of a workspace (NULL: the internal workspace of the current
 * device and this stream).  A GEMV workgroup that sums split partials waits for each
 * other split's words a bounded time (2^20 polls per wave, about a second); one
 * that never arrives gives NaN in the outputs that need it and sets a status word
 * in the workspace.  A partial may then still arrive after the exchange was
 * cleared, so while the word is set every GEMV call with that workspace writes NaN
 * for every output it sums, without waiting; exl3_hip_workspace_init clears it.
 * *faulted = 1 when the word is set, else 0.  Synchronises the stream.  No
 * counterpart in the reference, whose ops run on one thread pool per call. */
exl3_status exl3_hip_workspace_status(const void *workspace, size_t workspace_bytes, int *faulted,
                                      hipStream_t stream);

/* Test hook for the failure path above, never needed by an engine: spin_limit > 0
 * replaces the wait budget (polls per wave) and drop_split >= 0 makes the
 * workgroups of that k split skip storing their partial, so the summing
 * workgroup's own bounded wait runs out and every kernel still ends normally.
 * (0, -1) restores the defaults.  Process-wide; not for concurrent use. */
exl3_status exl3_hip_test_exchange_fault(int spin_limit, int drop_split);

/*
 * y[r][j] = sv[j] * H128( sum_i H128(x[r] * su)[i] * W_hat[i][j] )   (0 <= r < rows)
 * i.e. y = x . diag(su) H W_hat H diag(sv), the EXL3 linear layer, with su taken
 * from record (0, kb) and sv from record (nb, 0) as src/exl3-ggml.cpp:60-90 does.
 *   records      device, (n/128)*(k/128) records of exl3_group_bytes(bits), 16-byte aligned
 *   bits         1..8; codebook 0..2 (the reference's ggml op uses mul1 = 2)
 *   x            device, rows x k of xt, row stride x_row_stride elements (>= k)
 *   y            device, rows x n of yt, row stride y_row_stride elements (>= n)
 *   input range  the kernels hold xh = H128(x[r] * su) / sqrt(128) in fp16 (as a
 *                hi + lo pair up to 16 rows, hi only above), where the reference
 *                keeps fp32: every element of xh must stay below 65520 in
 *                magnitude (true whenever |x[r][i] * su[i]| <= 5790 for all i);
 *                beyond that the affected output rows are Inf or NaN
 *   workspace    device, >= exl3_hip_mul_mat_workspace_bytes(k, n, rows), zero-filled
 *                before first use; NULL -> an internal per-(device, stream)
 *                workspace is allocated on first use and kept (grown, never
 *                freed, when a larger call needs more).  While the stream is
 *                being captured into a HIP graph the internal workspace cannot
 *                grow: such a call returns EXL3_WORKSPACE_TOO_SMALL unless an
 *                uncaptured call of at least this size came first; callers that
 *                capture should pass their own workspace
 * Deterministic: the same inputs give the same bits on every call.
 */
exl3_status exl3_hip_mul_mat(const void *records, unsigned bits, unsigned codebook, size_t k, size_t n,
                             const void *x, exl3_dtype xt, size_t rows, size_t x_row_stride,
                             void *y, exl3_dtype yt, size_t y_row_stride,
                             void *workspace, size_t workspace_bytes, hipStream_t stream);

/* exl3_hip_mul_mat without a workspace and without any allocation: no
 * counterpart in the reference; for callers that cannot allocate (code under
 * HIP-graph capture, serving loops or harnesses that forbid hipMalloc).  The
 * workspace is a 64 MiB device array inside the library, one per GPU, held
 * until the process ends; a call whose exl3_hip_mul_mat_workspace_bytes(k, n,
 * rows) exceeds it returns EXL3_WORKSPACE_TOO_SMALL before anything is
 * enqueued.  Every call on a GPU shares
 * that GPU's array: calls that overlap on one GPU (different streams, or
 * threads without ordering) race and give wrong results; order them on one
 * stream.  Results equal exl3_hip_mul_mat's bit for bit.  A split-K wait that
 * gives up (see exl3_hip_workspace_status) marks the array like any workspace;
 * the array cannot be zero-filled again from outside, so every later call on
 * that GPU that sums split partials writes NaN until the process ends. */
exl3_status exl3_hip_mul_mat_noalloc(const void *records, unsigned bits, unsigned codebook, size_t k, size_t n,
                                     const void *x, exl3_dtype xt, size_t rows, size_t x_row_stride,
                                     void *y, exl3_dtype yt, size_t y_row_stride, hipStream_t stream);

/* y = residual + layer(x): the graph ADD(MUL_MAT(w, x), residual) of
 * tests/test-exl3-graph.cpp:53-55 in one call, the sum formed in fp32 and
 * rounded once to yt.  residual: device, rows x n of yt, row stride
 * residual_row_stride (>= n); it is either y itself with y's stride (an in-place
 * accumulate) or disjoint from y.  Otherwise as exl3_hip_mul_mat.  The
 * reference declines this fusion for its kernels (patches/llama-exl3.patch:161-162)
 * and runs the ADD as a separate graph node. */
exl3_status exl3_hip_mul_mat_add(const void *records, unsigned bits, unsigned codebook, size_t k, size_t n,
                                 const void *x, exl3_dtype xt, size_t rows, size_t x_row_stride,
                                 const void *residual, size_t residual_row_stride,
                                 void *y, exl3_dtype yt, size_t y_row_stride,
                                 void *workspace, size_t workspace_bytes, hipStream_t stream);

/* One matrix of an exl3_hip_mul_mat_group call. */
typedef struct exl3_matrix_desc {
    const void *records;   /* device, (n/128)*(k/128) group records, 16-byte aligned */
    size_t n;              /* output features, multiple of 128 */
    void *y;               /* device, rows x n of the call's yt */
    size_t y_row_stride;   /* elements, >= n */
} exl3_matrix_desc;

/* y_i = layer_i(x) for 1..4 matrices that share k, bits, codebook, x and rows
 * (the q/k/v or gate/up projections of one decoder layer): at rows <=
 * exl3_hip_gemv_max_rows() one GEMV launch serves all of them, so the launch and
 * its latency chain are paid once; larger row counts run one GEMM launch for all of
 * them, or, where the workspace only holds that, one exl3_hip_mul_mat per matrix (the
 * same bits).  Each y_i is the exl3_hip_mul_mat result within the layer tolerance (in
 * the GEMV the split of k follows the total width, so the summation order may differ
 * from a single call's).  workspace: >= exl3_hip_mul_mat_workspace_bytes(k, n, rows) of
 * every n_i and of their sum; exl3_hip_mul_mat_group_workspace_bytes also holds the one
 * GEMM launch; NULL for the internal one.  This entry point has no
 * counterpart in the reference, whose ggml op multiplies one matrix per call. */
exl3_status exl3_hip_mul_mat_group(const exl3_matrix_desc *mats, size_t count, unsigned bits, unsigned codebook,
                                   size_t k, const void *x, exl3_dtype xt, size_t rows, size_t x_row_stride,
                                   exl3_dtype yt, void *workspace, size_t workspace_bytes, hipStream_t stream);

/* Workspace bytes of an exl3_hip_mul_mat_group call: the most any row count
 * 1..rows needs to run as one GEMV or one GEMM over all matrices (each has its own
 * prepared activations and split partials there).  0 for invalid arguments.  Calls
 * also take less: as much as exl3_hip_mul_mat needs for the total width and for each
 * matrix. */
size_t exl3_hip_mul_mat_group_workspace_bytes(size_t k, const size_t *n, size_t count, size_t rows);

/* The ggml op on ggml views, replacing ggml_exl3_mul_mat (src/exl3-ggml.cpp:51-92)
 * with its row addressing: row r = i1 + ne[1] (i2 + ne[2] i3) of x starts at byte
 * i1 nb[1] + i2 nb[2] + i3 nb[3] of x, and its output row at the same indices of y
 * (row_offset, src/exl3-ggml.cpp:11-17, used at :64 and :88).
 *   x_info  type EXL3_GGML_TYPE_F32 or _F16, ne[0] = k, nb[0] = its element size,
 *           nb[1..3] multiples of it, in any order (permuted and sliced views)
 *   y_info  type F32 or F16, ne[0] = n, ne[1..3] = x's, nb[0] = its element size,
 *           nb[1..3] multiples of it, no two rows overlapping
 *   (the contiguous fields are not read)
 * The longest run of row dimensions that both views step through with one
 * stride is one exl3_hip_mul_mat call; the other dimensions loop over such calls.
 * workspace: >= exl3_hip_mul_mat_workspace_bytes(k, n, ne[1] ne[2] ne[3]), or NULL.
 * Each row is within exl3_hip_mul_mat's tolerance (which kernel serves a row
 * depends on how many rows share its call). */
exl3_status exl3_hip_mul_mat_nd(const void *records, unsigned bits, unsigned codebook, size_t k, size_t n,
                                const void *x, const exl3_tensor_info *x_info, void *y,
                                const exl3_tensor_info *y_info, void *workspace, size_t workspace_bytes,
                                hipStream_t stream);

/* Decode packed weights to row-major fp16 bits out[k][column_count] for
 * columns [first_column, first_column + column_count), bit-exact with
 * exl3::decode_inner_slice.  UPSTREAM_TILES: k, n, first and count multiples
 * of 16; RECORDS: multiples of 128.  out is device memory. */
exl3_status exl3_hip_decode(const void *src, exl3_layout layout, unsigned bits, unsigned codebook,
                            size_t k, size_t n, size_t first_column, size_t column_count,
                            uint16_t *out, hipStream_t stream);

/* One matrix of an exl3_hip_decode_batch call. */
typedef struct exl3_decode_desc {
    const void *src;   /* device, packed weights in the call's layout, 16-byte aligned */
    size_t k, n;       /* shape (multiples of 16 for UPSTREAM_TILES, of 128 for RECORDS) */
    uint16_t *out;     /* device, row-major fp16 bits out[k][n], 16-byte aligned */
    unsigned bits;     /* 1..8 */
} exl3_decode_desc;

/* exl3_hip_decode of whole matrices, many per launch: the matrices of one rate
 * share a launch (up to 32 each), so a model's weight set decodes in a few
 * launches instead of one per tensor; output bit-identical to exl3_hip_decode.
 * count 0 is a no-op.  This entry point has no counterpart in the reference,
 * which decodes one tensor per decode_inner call (src/exl3_codec.cpp:117-145). */
exl3_status exl3_hip_decode_batch(const exl3_decode_desc *descs, size_t count, exl3_layout layout,
                                  unsigned codebook, hipStream_t stream);

/* Original-basis weights diag(su) H W_hat H diag(sv) as fp16 bits out[k][column_count],
 * bit-exact with exl3::reconstruct_slice.  UPSTREAM_TILES takes su (k) and sv (n)
 * fp16 device vectors; RECORDS reads them from the records (su/sv may be NULL).
 * k, n, first_column, column_count multiples of 128. */
exl3_status exl3_hip_reconstruct(const void *src, exl3_layout layout, const uint16_t *su,
                                 const uint16_t *sv, unsigned bits, unsigned codebook, size_t k,
                                 size_t n, size_t first_column, size_t column_count, uint16_t *out,
                                 hipStream_t stream);

/* GET_ROWS: out[r][0..k) = column ids[r] of the original-basis weight
 * diag(su) H W_hat H diag(sv), i.e. for every kb the reconstruct of record
 * (ids[r] / 128, kb) as a 128x128 matrix (exl3::reconstruct, fp16-rounded),
 * column ids[r] % 128; bit-exact, widened to fp32 for ot = F32 (ggml's dst type).
 *   records        device, as exl3_hip_mul_mat; codebook: the reference uses mul1 = 2
 *   ids            device int32[count] (GGML_TYPE_I32 ids)
 *   out            device, count rows of ot, row stride out_row_stride (>= k) elements
 *   bad_ids        optional device int: set to 1 when some id is outside [0, n)
 *                  (its row is NaN); the reference asserts instead
 * count == 0 is a no-op. */
exl3_status exl3_hip_get_rows(const void *records, unsigned bits, unsigned codebook, size_t k, size_t n,
                              const int32_t *ids, size_t count, void *out, exl3_dtype ot, size_t out_row_stride,
                              int *bad_ids, hipStream_t stream);

/* GET_ROWS on ggml views (ggml_exl3_get_rows, src/exl3-ggml.cpp:19-49): id
 * r = i0 + ne[0] (i1 + ne[1] i2) is read at byte i0 nb[0] + i1 nb[1] + i2 nb[2] of
 * ids, and its row written at byte i0 nb[1] + i1 nb[2] + i2 nb[3] of out (:34-36).
 *   ids_info  type EXL3_GGML_TYPE_I32, ne[3] = 1, nb[0..2] multiples of 4
 *   out_info  type F32 or F16, ne = [k, ids ne[0], ids ne[1], ids ne[2]], nb[0] =
 *             its element size, nb[1..3] multiples of it, no two rows overlapping
 * Otherwise as exl3_hip_get_rows; no ids (a zero ne) is a no-op. */
exl3_status exl3_hip_get_rows_nd(const void *records, unsigned bits, unsigned codebook, size_t k, size_t n,
                                 const int32_t *ids, const exl3_tensor_info *ids_info, void *out,
                                 const exl3_tensor_info *out_info, int *bad_ids, hipStream_t stream);

/* out[i] = fp16 codebook value of states[i], bit-exact with exl3::decode_codebook. */
exl3_status exl3_hip_codebook(const uint16_t *states, size_t count, unsigned codebook, uint16_t *out,
                              hipStream_t stream);

/* In-place orthonormal H128 over each consecutive 128 fp32 values (count % 128 == 0),
 * bit-exact with exl3::hadamard128. */
exl3_status exl3_hip_hadamard128(float *values, size_t count, hipStream_t stream);

/* Upstream tiles [k/16][n/16][16*bits] + su[k] + sv[n] -> records. */
exl3_status exl3_hip_pack_records(const uint16_t *packed, const uint16_t *su, const uint16_t *sv,
                                  unsigned bits, size_t k, size_t n, void *records, hipStream_t stream);

/* The DSP service's layer exl3_iface_matmul (src/hexagon/exl3_service.c:265-305,
 * IDL src/hexagon/exl3_iface.idl:13-15): y = x . diag(su) H W_hat H diag(sv) on the
 * upstream tile layout with separate su / sv vectors, fp32 in and out.  Up to the row
 * counts of exl3_hip_mul_mat's GEMV the kernel reads the tiles and scales as they are;
 * above, one call packs them into group records inside the workspace
 * (exl3_hip_pack_records) and runs exl3_hip_mul_mat on them (the same bits either way).
 * Callers that reuse the weights at many rows pack once and call exl3_hip_mul_mat.
 *   packed      device, [k/16][n/16][16*bits] u16 = k*n*bits/8 bytes, 16-byte aligned
 *   suh, svh    device fp16 su[k] and sv[n], 16-byte aligned
 *   x, y        device fp32, batch x k and batch x n, dense rows (the service's layout)
 *   workspace   >= exl3_hip_iface_matmul_workspace_bytes(bits, k, n, batch), 256-byte
 *               aligned, zero-filled before first use; NULL -> an internal one
 * The service also caps batch at 8 and k*n at 64 Mi (its memory); here batch is any row
 * count exl3_hip_mul_mat accepts.  Rejections follow the service: bits 1..8, codebook
 * 0..2, k and n nonzero multiples of 128, batch >= 1 (EXL3_INVAL_PARAMS where the
 * service returns 2). */
size_t exl3_hip_iface_matmul_workspace_bytes(unsigned bits, size_t k, size_t n, size_t batch);
exl3_status exl3_hip_iface_matmul(unsigned bits, unsigned codebook, size_t k, size_t n, size_t batch,
                                  const uint16_t *packed, const uint16_t *suh, const uint16_t *svh, const float *x,
                                  float *y, void *workspace, size_t workspace_bytes, hipStream_t stream);

/* ---- the attention block between the q/k/v layers and the o layer --------
 * The reference leaves these operators to llama.cpp's graph; none of the entry
 * points below has a counterpart in it.  Together they take the rows that the q, k
 * and v layers wrote to the rows that the o layer reads:
 *   exl3_hip_qk_norm_rope      norms and positions of the queries and keys
 *   exl3_hip_attention_prompt  attention of packed prompts over their own keys
 *   exl3_hip_kv_cache_write    new keys and values into the quantised cache
 *   exl3_hip_attention_cached  attention of the next token(s) over that cache
 *   exl3_hip_kv_cache_read     cached rows back as F16/F32 (a prompt that continues them)
 * Heads are grouped: with g = q heads / kv heads (a whole number), q head h reads kv
 * head h / g. */

/* Rows of heads: element i of head h of token t is at data[t * token_stride + h *
 * head_stride + i] (strides in elements, the head's elements dense), so a slice of a
 * fused q/k/v buffer is a view.  Outputs: no two heads overlap.  A stride is at most 2^40
 * elements, and tokens and heads each span at most 2^48. */
typedef struct exl3_head_view {
    void *data;          /* device */
    size_t heads;
    size_t token_stride;
    size_t head_stride;
} exl3_head_view;

/* RMS norm of each head and rotation by position, of queries and keys in one launch:
 *   z = x / sqrt(mean(x^2) + eps) * weight              (weight NULL: z = x)
 *   (a, b) -> rope_scale (a cos t - b sin t, b cos t + a sin t),  t = positions[token] inv_freq[p]
 * for the pairs p < rot_dim / 2 of z's first rot_dim elements, (z[p], z[p + rot_dim /
 * 2]) or with `interleaved` (z[2p], z[2p + 1]); the other elements stay z.  The scaling
 * of long contexts is the caller's inv_freq and rope_scale.  Computed in fp32 and
 * rounded once; t is reduced to a turn with two fp32 words per frequency, so sin and cos
 * hold to about 1e-6 at any position (|position| < 2^24).
 *   q, k       xt rows; k and k_out may both be NULL; q_out / k_out have their heads and
 *              are the same view as q / k (xt = yt: in place) or disjoint from both
 *   head_dim   multiple of 8 up to 256
 *   q_weight, k_weight   device fp32[head_dim] or NULL
 *   positions  device int32[tokens]; inv_freq device fp32[rot_dim / 2]; either may be
 *              NULL when rot_dim is 0
 *   rot_dim    multiple of 16 up to head_dim, or 0
 * tokens = 0 is a no-op. */
exl3_status exl3_hip_qk_norm_rope(const exl3_head_view *q, const exl3_head_view *k, exl3_dtype xt, size_t tokens,
                                  size_t head_dim, const float *q_weight, const float *k_weight, float eps,
                                  const int32_t *positions, const float *inv_freq, size_t rot_dim, int interleaved,
                                  float rope_scale, const exl3_head_view *q_out, const exl3_head_view *k_out,
                                  exl3_dtype yt, hipStream_t stream);

/* The cache: page_count pages of page_tokens (P) tokens, each with every kv head's keys
 * and values at `bits` = 4 or 8.  Token slot s = page * P + offset.  32 consecutive
 * elements of a head form a group: the group is rotated by the orthonormal
 * Walsh-Hadamard matrix H32 (which spreads a large channel over the group), ext is its
 * element of largest magnitude (the negative one of two equal), scale = fp16(-ext /
 * 2^(bits-1)) with its magnitude rounded up to 12 - bits significant bits (a zero is +0), and code =
 * clamp(rint(y / scale), -2^(bits-1), 2^(bits-1) - 1): every scale * code has at most 11
 * significant bits, so attention reads the cache without a further rounding (a product
 * above 65,504, which H32 can make of an fp16 row, included).  A group with a non-finite
 * element, or whose scale is beyond fp16's range (an extreme of half a million at 4 bits,
 * 7.8 million at 8), reads back as NaN.
 * A page is, for each kv head, four runs:
 *   keys    [P][head_dim * bits / 8]          code + 2^(bits-1); 4 bits: the even element low
 *   values  [P/4][16][4][head_dim * bits / 128]  blocks of 4 tokens: 16 slices of a row, each
 *                                               with its 4 tokens next to each other
 *   key scales    fp16 [P][head_dim / 32]
 *   value scales  fp16 [P/4][head_dim / 32][4]
 * Bytes of a page; 0 unless bits is 4 or 8, head_dim 64, 128 or 256, page_tokens a
 * nonzero multiple of 16 up to 65536 and 1 <= kv_heads <= 1024. */
size_t exl3_hip_kv_page_bytes(unsigned bits, size_t kv_heads, size_t head_dim, size_t page_tokens);

/* Quantises `tokens` rows of keys and values (k->heads = v->heads = kv heads) into
 * their slots.  slots: device int64[tokens], no slot twice; a negative one is skipped (a
 * padded place of a batch), one beyond the cache is skipped and sets *bad_slots
 * (optional device int) to 1.  pages: 16-byte aligned, page_count *
 * exl3_hip_kv_page_bytes() bytes, its unwritten slots of any contents. */
exl3_status exl3_hip_kv_cache_write(void *pages, size_t page_count, unsigned bits, size_t page_tokens, size_t head_dim,
                                    const exl3_head_view *k, const exl3_head_view *v, exl3_dtype xt, size_t tokens,
                                    const int64_t *slots, int *bad_slots, hipStream_t stream);

/* The rows of some slots as the cache holds them, rotated back, rounded once to yt.  A
 * slot outside the cache gives NaN rows and sets *bad_slots (optional). */
exl3_status exl3_hip_kv_cache_read(const void *pages, size_t page_count, unsigned bits, size_t page_tokens,
                                   size_t head_dim, const int64_t *slots, size_t tokens, const exl3_head_view *k_out,
                                   const exl3_head_view *v_out, exl3_dtype yt, int *bad_slots, hipStream_t stream);

/* Attention of the last q_len tokens of each sequence over the cache:
 *   out[i] = sum_n softmax_n(scale q[i] . K[n]) V[n]
 * where row s * q_len + j of q (F16) is token j of sequence s's last q_len, and sees the
 * keys n < kv_lens[s] - (q_len - 1 - j); a row that sees none is zero.  Token n of
 * sequence s is at offset n % P of page page_table[s * table_stride + n / P].
 *   page_table  device int32[sequences * table_stride]; an entry outside the cache makes
 *               the rows of its sequence that read it NaN
 *   kv_lens     device int32[sequences], the cached tokens of each sequence with the
 *               q_len new ones (written before the call); beyond table_stride * P it
 *               counts as that, negative as 0
 *   out         F16, disjoint from q
 *   workspace   device, 256-byte aligned, >= exl3_hip_attention_cached_workspace_bytes(),
 *               zero-filled before first use (exl3_hip_workspace_init); it may be one
 *               that exl3_hip_mul_mat uses too.  NULL: the internal one of this stream
 * head_dim 64, 128 or 256; q heads a multiple of kv_heads, up to 64 of them per kv head;
 * q_len 1..65536; scale finite.  Scores, softmax statistics and sums in fp32; q as an fp16 pair (high
 * and low part; an eighth of a row with elements above 11,576, so every finite row is
 * held), weights rounded to fp16.  The same inputs give the same bits on every
 * call.  A workspace whose exchange gave up (exl3_hip_workspace_status) gives NaN rows until
 * it is initialised again.  EXL3_NO_SUPPORT where kv_heads * ceil(group * q_len / 16) is
 * above 65,535, or times the sequences above 2^22.  sequences = 0 is a no-op. */
exl3_status exl3_hip_attention_cached(const exl3_head_view *q, const exl3_head_view *out, size_t head_dim,
                                      const void *pages, size_t page_count, unsigned bits, size_t page_tokens,
                                      size_t kv_heads, const int32_t *page_table, size_t table_stride,
                                      const int32_t *kv_lens, size_t sequences, size_t q_len, float scale,
                                      void *workspace, size_t workspace_bytes, hipStream_t stream);
/* 0 for arguments that exl3_hip_attention_cached refuses */
size_t exl3_hip_attention_cached_workspace_bytes(size_t q_heads, size_t kv_heads, size_t head_dim, size_t sequences,
                                                 size_t q_len);

/* Attention of packed sequences: sequence s has the query rows q_starts[s] ..
 * q_starts[s + 1] - 1 and the key and value rows kv_starts[s] .. kv_starts[s + 1] - 1
 * (device int32[sequences + 1] each, ascending from 0).  With `causal` query i of nq
 * sees the first nk - (nq - 1 - i) of its nk keys (the sequences' ends aligned: keys
 * ahead of the queries are a prefix), else all; a row that sees none is zero.  q, k, v
 * and out are F16, out disjoint from the inputs; head_dim 64, 128 or 256; q heads a
 * multiple of kv heads; scale finite.  q_tokens and kv_tokens are the rows of the views (no row
 * outside them is read or written, whatever the starts hold; a query row that no
 * sequence has is not written).  Scores, softmax statistics and sums in fp32, weights
 * rounded to fp16.  The same inputs give the same bits on every call.
 *   workspace   device, 256-byte aligned, >= exl3_hip_attention_prompt_workspace_bytes() where that
 *               is not 0 (few query rows over many keys: parts of the walk are joined there); it may
 *               be one that other calls use too.  NULL: the internal one of this stream
 * EXL3_NO_SUPPORT where (q_tokens / 128 + sequences) * q heads reaches 2^23.  sequences = 0 or q_tokens = 0
 * is a no-op. */
exl3_status exl3_hip_attention_prompt(const exl3_head_view *q, const exl3_head_view *k, const exl3_head_view *v,
                                      const exl3_head_view *out, size_t head_dim, const int32_t *q_starts,
                                      const int32_t *kv_starts, size_t sequences, size_t q_tokens, size_t kv_tokens,
                                      float scale, int causal, void *workspace, size_t workspace_bytes,
                                      hipStream_t stream);
/* 0 where exl3_hip_attention_prompt takes no workspace (and for arguments that it refuses) */
size_t exl3_hip_attention_prompt_workspace_bytes(size_t q_heads, size_t head_dim, size_t sequences, size_t q_tokens,
                                                 size_t kv_tokens);

/* ---- the linear-attention block and the norms between blocks --------------
 * Beside the attention block: the operators of a hybrid model's linear-attention layer between
 * its projections and its output layer, and the norm ahead of a layer.  The reference leaves
 * these to llama.cpp's graph too.  In the order of a layer:
 *   exl3_hip_rms_norm    the block's input: residual addition and norm
 *   exl3_hip_short_conv  the projected rows through a causal depthwise convolution
 *   exl3_hip_delta_rule  the gated delta rule over the sequences
 *   exl3_hip_rms_norm    each head's norm, gated
 * Rows are packed sequences: sequence s has the rows starts[s] .. starts[s + 1] - 1 (device
 * int32[sequences + 1], ascending from 0); with starts NULL each has tokens / sequences rows
 * (a whole number).  No row outside the views is read or written, whatever the starts hold; a
 * row that no sequence has is not written.
 * A sequence goes on from a state that an earlier call left.  States lie in a pool of `slots`
 * of them: sequence s starts from state slots_in[s] (from zeros where that is negative or
 * slots_in is NULL) and leaves its state in slots_out[s] (nowhere where that is negative or
 * slots_out is NULL); both device int32[sequences].  A slot_in beyond the pool counts as a state
 * of NaN, a slot_out beyond the pool is not written.  A slot that a sequence leaves its state in is
 * no other sequence's in the call, in or out; it may be its own slot_in.  A sequence without rows leaves
 * the state that it starts from. */

/* Root-mean-square norm of rows of heads:
 *   h = x + residual                                   (residual NULL: h = x)
 *   out = h / sqrt(mean(h^2) + eps) * weight * silu(gate)   (weight NULL: 1; gate NULL: no factor)
 *   residual_out = h                                   (NULL: not kept; needs a residual)
 * with silu(z) = z / (1 + exp(-z)).  Computed in fp32 from h as summed, each output rounded once; the squares are fp32's
 * too (|h| beyond 1.8e19 / sqrt(width) makes their sum infinite and the row 0).
 *   x, gate    xt rows; all views have x's heads, each head `width` elements, 1 .. 65536
 *   residual, residual_out   rt rows
 *   weight     device fp32[width] or NULL, shared by the heads
 *   out        yt rows.  out may be x's view (xt = yt) and residual_out residual's; otherwise
 *              outputs are disjoint from the inputs and from each other
 * tokens = 0 is a no-op. */
exl3_status exl3_hip_rms_norm(const exl3_head_view *x, const exl3_head_view *gate, exl3_dtype xt,
                              const exl3_head_view *residual, const exl3_head_view *residual_out, exl3_dtype rt,
                              size_t tokens, size_t width, const float *weight, float eps, const exl3_head_view *out,
                              exl3_dtype yt, hipStream_t stream);

/* Causal depthwise convolution of packed sequences:
 *   y[t][c] = act(bias[c] + sum_j weight[c][j] x[t - (width - 1) + j][c]),  j < width
 * where rows ahead of a sequence's first come from its state, and act is silu or the identity.
 * The state it leaves is its last width - 1 rows (those of the old state counted where it is
 * shorter), in xt: [slots][width - 1][channels], the oldest first.  Sums in fp32, rounded once.
 *   x, y       rows of `channels` elements, row strides in elements (at least channels), disjoint
 *   channels   1 .. 2^20; width 2 .. 4
 *   weight     device fp32[channels][width]; bias device fp32[channels] or NULL
 *   states     device, 16-byte aligned, or NULL with both slot lists NULL
 * EXL3_NO_SUPPORT where (tokens / 32 + sequences) * ceil(channels / 256) reaches 2^23.
 * sequences = 0 is a no-op. */
exl3_status exl3_hip_short_conv(const void *x, exl3_dtype xt, size_t x_row_stride, size_t tokens, size_t channels,
                                const float *weight, size_t width, const float *bias, int silu, const int32_t *starts,
                                size_t sequences, void *states, size_t slots, const int32_t *slots_in,
                                const int32_t *slots_out, void *y, exl3_dtype yt, size_t y_row_stride,
                                hipStream_t stream);

/* The gated delta rule of packed sequences.  Value head h has a state S, fp32 [key_dim][value_dim],
 * and reads key head h / (v heads / k heads); for each row in turn
 *   S <- exp(g) S,   u = beta (v - S^T k),   S <- S + k u^T,   out = scale S^T q
 * with q and k divided by sqrt(sum(x^2) + qk_eps) first (qk_eps negative: as they are), and
 *   g = -exp(a_log) softplus(g_in + dt_bias),  beta = 1 / (1 + exp(-beta_in))
 * where a_log is given, else g_in (a log decay, at most 0 in earnest; -inf empties the state) and beta_in.
 *   q, k       F16, the same heads; v, out F16, v heads a multiple of k heads; out disjoint from all
 *   key_dim    64 or 128; value_dim a multiple of 16 up to 256
 *   g, beta    device fp32, row t of v heads at t * gate_stride (at least v heads) elements
 *   a_log, dt_bias   device fp32[v heads], both or neither
 *   states     device fp32 [slots][v heads][key_dim][value_dim], 16-byte aligned, or NULL with both
 *              slot lists NULL
 *   scale      finite
 *   workspace  device, 256-byte aligned, >= exl3_hip_delta_rule_workspace_bytes() where that is
 *              not 0; it may be one that other calls use too.  NULL: the internal one of this stream
 * States and sums in fp32.  Long sequences' rows are taken 64 at a time, their products as fp16 pairs (high
 * and low part, 22 bits).  The pairs end at 2^-40 of a bound on their column among the 64 rows, which adds up to
 * 2^-31 ||T|| (|beta v| + beta |k|_1 |S|) to a state's error, of the largest v of the 64 rows and S of the state ahead of
 * them, T the inverse of 1 + (beta_i e^(G_i - G_j) k_i . k_j, j < i).  That is far below the 22 bits of those, but a state
 * that gates empty within 64 rows leaves it behind: 1e-3 was measured where the old state was 3e6 and the new one 0.4,
 * 1e-7 where it was 300.  Row by row binary32's bits are kept.
 * An element that is not finite leaves other sequences, other heads and the rows ahead of its 64 as they are.  One of v
 * or of a state reaches its own column alone (v counts as 65,504 in the bits of the others), one of k, g or beta its
 * heads: infinite or NaN from its row on, and where rows are taken 64 at a time the rows ahead of it among them may be
 * NaN as well.  One of q makes NaN of its row's outputs, there perhaps of others of the 64 too, and reaches no state.
 * Long sequences are those of 16 rows and more (24 where sequences * v heads * value_dim / 16 reaches 512) where
 * starts is NULL, and of 8 and more where it is given, tokens is at least 16 and tokens / sequences at least 2 (a
 * sequence alone: where tokens is at least 16).  The same inputs give the same bits on every call.
 * EXL3_NO_SUPPORT where (tokens / 64 + sequences) * v heads * value_dim / 16 reaches 2^22.  sequences = 0 is a no-op. */
exl3_status exl3_hip_delta_rule(const exl3_head_view *q, const exl3_head_view *k, const exl3_head_view *v,
                                const float *g, const float *beta, size_t gate_stride, const float *a_log,
                                const float *dt_bias, const exl3_head_view *out, size_t key_dim, size_t value_dim,
                                const int32_t *starts, size_t sequences, size_t tokens, float *states, size_t slots,
                                const int32_t *slots_in, const int32_t *slots_out, float scale, float qk_eps,
                                void *workspace, size_t workspace_bytes, hipStream_t stream);
/* 0 where exl3_hip_delta_rule takes no workspace, with starts or without (and for arguments that it refuses); else
 * (tokens / 64 + sequences) * v heads * 75,008 bytes (50,432 for key_dim 64) and 16 MiB, as for as many key
 * heads as value heads: 16 heads of 128 take 19 KB a token, 1.2 GB for 65,536.  The internal workspace keeps its largest
 * size for its stream. */
size_t exl3_hip_delta_rule_workspace_bytes(size_t v_heads, size_t key_dim, size_t value_dim, size_t sequences,
                                           size_t tokens);

/* *result (device int) = 1 when every su/sv value of every record is finite,
 * 0 otherwise; EXL3_INVAL_PARAMS when nbytes is not a whole number of records. */
exl3_status exl3_hip_validate_records(const void *records, size_t nbytes, unsigned bits, int *result,
                                      hipStream_t stream);

/* ---- deployment model reader (exl3::Model, src/exl3_model.cpp:79-187) ----
 * A model directory holds model.safetensors and hexagon-exl3.json; it is
 * validated as the reference validates it.  Host memory maps the file; the
 * embedding and the record upload use the current HIP device. */
typedef struct exl3_model exl3_model;

/* NULL when the directory is missing or malformed; the reason is copied into
 * error (NUL-terminated, at most error_bytes - 1 characters) when given. */
exl3_model *exl3_hip_model_open(const char *directory, char *error, size_t error_bytes);
void exl3_hip_model_close(exl3_model *model);
size_t exl3_hip_model_tensor_count(const exl3_model *model);
size_t exl3_hip_model_payload_bytes(const exl3_model *model);
size_t exl3_hip_model_hidden_size(const exl3_model *model);
size_t exl3_hip_model_vocab_size(const exl3_model *model);
double exl3_hip_model_bits_per_weight(const exl3_model *model);
/* out (host) = hidden_size fp16 bits of token's tied embedding, bit-exact with
 * exl3::Model::embedding; EXL3_INVAL_PARAMS when token >= vocab_size. */
exl3_status exl3_hip_model_embedding(const exl3_model *model, uint32_t token, uint16_t *out);
/* EXL3 matrices of the model (every <prefix>.trellis with its .suh/.svh), in name order */
size_t exl3_hip_model_matrix_count(const exl3_model *model);
exl3_status exl3_hip_model_matrix(const exl3_model *model, size_t index, char *name, size_t name_bytes,
                                  unsigned *bits, unsigned *codebook, size_t *k, size_t *n);
/* device bytes of matrix index's group records (0 for a bad index) */
size_t exl3_hip_model_record_bytes(const exl3_model *model, size_t index);
/* Row-coded EXL3 embedding tables of the model: every <prefix>.trellis of rank 2
 * (I16 [rows, groups * words]) that has a <prefix>.signs (F16 [groups, 256]),
 * validated as the reference's model audit validates them
 * (tools/inspect_model.py:78-90): words = 16 * bits + 1 per group, bits 1..8.
 * Their decode is not implemented (the reference's runtime has none either).
 * EXL3_OK with *count, or EXL3_INVAL_PARAMS with the audit's reason copied into
 * error ("Invalid EXL3 embedding: <name>", "... groups: ...", "... bitrate: ..."). */
exl3_status exl3_hip_model_embedding_tables(const exl3_model *model, size_t *count, char *error, size_t error_bytes);
/* table index (name order): its prefix, rows, groups, bits and padded width
 * (groups * 256) */
exl3_status exl3_hip_model_embedding_table(const exl3_model *model, size_t index, char *name, size_t name_bytes,
                                           size_t *rows, size_t *groups, unsigned *bits, size_t *width_padded);
/* packs matrix index into group records at device pointer records (16-byte
 * aligned, exl3_hip_model_record_bytes long), ready for exl3_hip_mul_mat;
 * returns when they are complete.  k and n must be multiples of 128. */
exl3_status exl3_hip_model_upload_records(const exl3_model *model, size_t index, void *records, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* EXL3_HIP_H */
