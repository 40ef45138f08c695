/*
 * deep8_hip.h -- C ABI of libdeep8_hip.so: the MI355X (gfx950) kernels behind Deep8's
 * MatrixMultiply / Conv2d / DeConv2d GPU entry points.
 *
 * Plain pointers and integers only.  Every function returns 0 on success or a non-zero code
 * (a hipError_t value, or D8_ERR_* below); d8_last_error() gives the text.  Nothing throws
 * across this boundary; the C++ host layer turns a non-zero code into the same
 * std::runtime_error Deep8's CUDA_CHECK raises (deep8/include/basic/GPUException.h:15-24).
 *
 * All matrices are row-major (deep8/src/model/Shape.cpp:86-96).  Device pointers unless said
 * otherwise.  `stream` is a hipStream_t passed as void* (NULL = the default stream, which is
 * what Deep8 uses everywhere).  All launches are asynchronous.
 */
#ifndef DEEP8_HIP_H
#define DEEP8_HIP_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element types: the ids of Deep8's DType (deep8/include/model/ElementType.h:8-22) */
#define D8_FLOAT16 10
#define D8_FLOAT32 11
#define D8_FLOAT64 12 /* the contraction path only: d8_fill, d8_gemm, the four gather maps, d8_matmul*, d8_conv2d*, d8_deconv2d* */

#define D8_ERR_ARGUMENT 10001 /* bad shape / leading dimension / null pointer */
#define D8_ERR_DTYPE    10002 /* element type not supported by this build     */
#define D8_ERR_ARCH     10003 /* the device is not gfx950                      */

const char *d8_last_error(void);

/* ---- device plumbing -------------------------------------------------------------------
 * Replaces what GPUDevice / GPUMemoryAllocator do through the CUDA runtime
 * (deep8/src/model/GPUDevice.cu:10-12, deep8/src/model/GPUMemoryAllocator.cu:17-56).      */
int d8_device_init(int device_id);                /* hipSetDevice + arch check (gfx950)    */
int d8_device_count(int *count);
int d8_device_info(int *cu_count, int *clock_khz, size_t *hbm_bytes, char *name, int name_len);
int d8_mem_info(size_t *free_bytes, size_t *total_bytes); /* device memory free / in all (no counterpart in
                                                     the reference; lets a caller see that a call allocated nothing) */
int d8_malloc(void **ptr, size_t bytes);          /* cudaMalloc      GPUMemoryAllocator.cu:17 */
int d8_free(void *ptr);                           /* cudaFree        GPUMemoryAllocator.cu:27 */
int d8_host_malloc(void **ptr, size_t bytes);     /* pinned host memory                    */
int d8_host_free(void *ptr);
int d8_memset(void *ptr, int value, size_t bytes, void *stream);   /* cudaMemset  :34      */
int d8_memcpy_h2d(void *dst, const void *src, size_t bytes);       /* cudaMemcpy  :46      */
int d8_memcpy_d2h(void *dst, const void *src, size_t bytes);       /* cudaMemcpy  :50      */
int d8_memcpy_d2d(void *dst, const void *src, size_t bytes, void *stream);  /* :40,:54     */
/* value[i] = scalar for n elements.  Replaces ConstantKernel (deep8/src/math/Constant.cu:10-44),
 * which Variable::zeroGradient / oneGradient use (deep8/src/nodes/Variable.cpp:119-130).   */
int d8_fill(int dtype, void *ptr, size_t n, float scalar, void *stream);
int d8_stream_create(void **stream);
int d8_stream_destroy(void *stream);
int d8_stream_sync(void *stream);
/* Every entry point of this header only launches kernels on the stream it is given (no allocation, no
 * synchronisation, no memset node), so a sequence of calls can be captured once and replayed: for products
 * so small that the launches cost more than the arithmetic.  d8_graph_begin starts capturing on `stream`
 * (not the default stream); the calls that follow, given the same stream, are recorded instead of run;
 * d8_graph_end returns the instantiated graph; d8_graph_launch replays it on a stream.  No counterpart in
 * the reference (hipStreamBeginCapture / hipStreamEndCapture / hipGraphInstantiate / hipGraphLaunch). */
int d8_graph_begin(void *stream);
int d8_graph_end(void *stream, void **graph);
int d8_graph_launch(void *graph, void *stream);
int d8_graph_destroy(void *graph);
int d8_event_create(void **event);
int d8_event_destroy(void *event);
int d8_event_record(void *event, void *stream);
int d8_event_elapsed_ms(void *start, void *stop, float *ms);  /* synchronises on `stop` */

/* ---- GEMM ------------------------------------------------------------------------------
 * C_b = op(A_b) * op(B_b) + beta * C_b,   b = 0 .. batch-1,  beta in {0, 1}
 *
 * op(A) is M x K, op(B) is K x N.  transA != 0: A is stored K x M (lda >= M); otherwise M x K
 * (lda >= K).  transB != 0: B is stored N x K (ldb >= K); otherwise K x N (ldb >= N).
 * transA and transB both set is rejected (Deep8 never issues it).  Strides are in elements;
 * strideA/strideB 0 broadcasts that operand over the batch.  strideC == 0 with batch > 1
 * sums all batch products into the one C (Deep8's gradient of a batch-1 operand).
 * fp16 operands accumulate in fp32 and are rounded once; beta = 1 adds the old C in fp32.
 * D8_FLOAT64 operands accumulate in fp64 (the cublasDgemm twins of the call sites below); a split
 * reduction keeps its partial sums in fp64 too.
 *
 * Sizes: any batch and any M (a batch of more than 448 independent products and a matrix of more than
 * 8 388 480 rows are run as several launches on slices); Float64 takes at most 4 194 240 columns.
 *
 * `workspace` (may be NULL) lets the kernel split the reduction (long K / summed batch, small
 * M x N) over more workgroups; d8_gemm_workspace_bytes says how much it can use.  It must be
 * 16-byte aligned (a misaligned workspace is ignored).
 *
 * Replaces the 27 cublas{S,H}gemm call sites in deep8/src/math/MatrixMultiply.cu:36-55,
 * 75-94,115-134 (forward), :211-230,253-272,296-315 (GradX), :399-418,441-460,484-503
 * (GradY) and the 18 in deep8/src/math/Conv2d.cu:195,473,801 / DeConv2d.cu:109,428,699
 * (+ their half twins).                                                                    */
size_t d8_gemm_workspace_bytes(int dtype, int transA, int transB, int M, int N, int K,
                               int batch, long strideC);
int d8_gemm(int dtype, int transA, int transB, int M, int N, int K,
            const void *A, int lda, long strideA,
            const void *B, int ldb, long strideB,
            float beta, void *C, int ldc, long strideC, int batch,
            void *workspace, size_t workspace_bytes, void *stream);

/* ---- Conv2d gather / scatter -------------------------------------------------------------
 * Geometry is explicit; padTop/padLeft >= 0 count the zero rows/columns before the image
 * (Deep8 passes the same numbers negated, deep8/src/math/Conv2d.cu:335-336).
 *
 * d8_im2col:  col[(b,oy,ox)][(fy,fx,c)] = im[b, oy*sy + fy*dy - padTop, ox*sx + fx*dx - padLeft, c]
 *             or +0 outside.  col is [B*OH*OW, FH*FW*C].   Replaces Conv2dIm2ColKernel
 *             (deep8/src/math/Conv2d.cu:10-61, launched :170,:776).
 * d8_col2im:  im += transpose of that map applied to col; taps added in (fy,fx) ascending
 *             order.  Replaces Conv2dCol2ImKernel (Conv2d.cu:64-118, launched :475).       */
int d8_im2col(int dtype, const void *im, void *col,
              int B, int IH, int IW, int C, int OH, int OW, int FH, int FW,
              int sy, int sx, int dy, int dx, int padTop, int padLeft, void *stream);
int d8_col2im(int dtype, const void *col, void *im,
              int B, int IH, int IW, int C, int OH, int OW, int FH, int FW,
              int sy, int sx, int dy, int dx, int padTop, int padLeft, void *stream);

/* ---- DeConv2d gather maps ------------------------------------------------------------------
 * zmat / dzmat are [B*IH*IW, OC*FH*FW] with column index oc*FH*FW + fy*FW + fx.
 *
 * d8_deconv_col2im: z[b,oy,ox,oc] = sum over taps (fy,fx) with iy*sy == oy - padTop + fy,
 *             ix*sx == ox - padLeft + fx inside the input, of zmat[(b,iy,ix)][oc,fy,fx];
 *             overwrites z.  Replaces DeConv2dCol2ImKernel (deep8/src/math/DeConv2d.cu:11-58,
 *             launched :115).
 * d8_deconv_im2col: dzmat[(b,iy,ix)][oc,fy,fx] = dz[b, iy*sy + padTop - fy, ix*sx + padLeft - fx, oc]
 *             or +0 outside.  Replaces DeConv2dIm2ColKernel (DeConv2d.cu:310-351, launched
 *             :405,:675).                                                                   */
int d8_deconv_col2im(int dtype, const void *zmat, void *z,
                     int B, int IH, int IW, int OH, int OW, int OC, int FH, int FW,
                     int sy, int sx, int padTop, int padLeft, void *stream);
int d8_deconv_im2col(int dtype, const void *dz, void *dzmat,
                     int B, int IH, int IW, int OH, int OW, int OC, int FH, int FW,
                     int sy, int sx, int padTop, int padLeft, void *stream);

/* ---- whole-operator entry points -----------------------------------------------------------
 * What Math::*GPU call (deep8/include/math/MatrixMultiply.h:17,26,35, Conv2d.h:23,33,45,
 * DeConv2d.h:18,28,38): shape cases, pad formulas, scratch use and accumulate-vs-overwrite
 * semantics are Deep8's.  A matrix operand is (batch, rows, cols) with cols = 1 for a 1-D
 * tensor.  `scratch` is the interim buffer the node allocates (size from the *_scratch_bytes
 * function, which already includes any split-reduction workspace and, for Float16 products whose
 * rows do not start at multiples of 16 bytes, room for copies that do where they pay).  Where that function
 * returns 0 the operator stages nothing (its patch matrix is read by the GEMM's tile loader)
 * and `scratch` may be NULL; a scratch smaller than asked for is an error only when the
 * operator has to stage.  The size functions assume tensors that are 16-byte aligned (every
 * allocation of d8_malloc and of Deep8's pools is): a Conv2d / DeConv2d tensor at an address that
 * is not can only take the staged route, whose interim matrix is sizeof(T)*B*OH*OW*FH*FW*IC
 * (Conv2d) or sizeof(T)*B*IH*IW*OC*FH*FW (DeConv2d) bytes plus d8_gemm_workspace_bytes; with
 * less the call fails with D8_ERR_ARGUMENT and says so.                                       */
size_t d8_matmul_scratch_bytes(int dtype, int which /*0 fwd, 1 gradX, 2 gradY, 3 both gradients from one call*/,
                               int xb, int xr, int xc, int yb, int yr, int yc);
int d8_matmul(int dtype, const void *x, int xb, int xr, int xc,
              const void *y, int yb, int yr, int yc, void *z,
              void *scratch, size_t scratch_bytes, void *stream);
int d8_matmul_grad_x(int dtype, void *dx, int xb, int xr, int xc,
                     const void *y, int yb, int yr, int yc, const void *dz,
                     void *scratch, size_t scratch_bytes, void *stream);
int d8_matmul_grad_y(int dtype, const void *x, int xb, int xr, int xc,
                     void *dy, int yb, int yr, int yc, const void *dz,
                     void *scratch, size_t scratch_bytes, void *stream);
/* The same two products written over their destination instead of added to it: what the pair
 * "zero the gradient, then accumulate" (deep8/src/model/EagerExecutor.cpp:51-65 followed by
 * Math::MatrixMultiplyGradX/YGPU) leaves behind, without the fill and without reading the zeros
 * back.  For callers that know the destination holds zeros (or nothing yet).                    */
int d8_matmul_grad_x_overwrite(int dtype, void *dx, int xb, int xr, int xc,
                               const void *y, int yb, int yr, int yc, const void *dz,
                               void *scratch, size_t scratch_bytes, void *stream);
int d8_matmul_grad_y_overwrite(int dtype, const void *x, int xb, int xr, int xc,
                               void *dy, int yb, int yr, int yc, const void *dz,
                               void *scratch, size_t scratch_bytes, void *stream);
/* Both gradients of one MatrixMultiply from one call: what Function::backward leaves after it has run for
 * index 0 and for index 1 (deep8/src/nodes/MatrixMultiply.cpp:31-52 -> Math::MatrixMultiplyGradX, then
 * Math::MatrixMultiplyGradY; deep8/src/math/MatrixMultiply.cu:193-363,381-551).  The two products are independent
 * of each other, so large Float16 ones run as ONE launch in which a workgroup goes from a tile of dx straight on
 * to a tile of dy; everything else is d8_matmul_grad_x followed by d8_matmul_grad_y.  The results are bit for bit
 * those of the two calls.  overwrite: bit 0 -- dx is written instead of added to, bit 1 -- dy likewise (the
 * _overwrite forms above).  scratch: d8_matmul_scratch_bytes(which = 3), room for both gradients' scratch side by
 * side and, in Float16, for copies of the operands whose rows do not start at multiples of 16 bytes, where copies
 * pay; with less, but at least the larger of which = 1 and which = 2, the call still works (mid-size products
 * then run as two launches, and such operands are read as they lie, which takes longer).  Two small products share a launch as
 * well (each at most four 128 x 128 tiles over a reduction of at most 512, or reductions of at most 512 -- in Float16 1024 --
 * and no more 32 x 32 tiles than run at once), and so do two mid-size ones.                                             */
int d8_matmul_grad_xy(int dtype, const void *x, void *dx, int xb, int xr, int xc,
                      const void *y, void *dy, int yb, int yr, int yc, const void *dz, int overwrite,
                      void *scratch, size_t scratch_bytes, void *stream);

/* d8_matmul_grad_y for callers that cannot allocate and have no scratch to pass.  No counterpart in the
 * reference: it is for code under HIP graph capture, tight serving loops and harnesses that forbid
 * hipMalloc.  Same arguments, checks and result (bit for bit) as d8_matmul_grad_y given a scratch of
 * d8_matmul_scratch_bytes(dtype, 2, ...) bytes, but the split reduction's partial sums go to a device
 * array of D8_STATIC_SCRATCH_BYTES that lives in the library (each GPU the library runs on holds one
 * until the process ends).  A shape that would need more is refused with D8_ERR_ARGUMENT.  The call
 * allocates and frees nothing.  All calls on one GPU share that GPU's array: calls that overlap in time
 * on one GPU (different streams or host threads) race.                                                  */
#define D8_STATIC_SCRATCH_BYTES (32u << 20)
int d8_matmul_grad_y_static(int dtype, const void *x, int xb, int xr, int xc,
                            void *dy, int yb, int yr, int yc, const void *dz, void *stream);

/* out[0..3] = OH, OW, padTop, padLeft (deep8/src/math/Conv2d.cpp:20-32, Conv2d.cu:332-336;
 * deep8/src/math/DeConv2d.cpp:23-29, DeConv2d.cu:99-100) */
int d8_conv2d_geometry(int IH, int IW, int FH, int FW, int covered,
                       int sy, int sx, int dy, int dx, int *out);
int d8_deconv2d_geometry(int IH, int IW, int FH, int FW, int covered, int sy, int sx, int *out);

/* which: 0 forward, 1 gradient of x, 2 gradient of the filter, 3 both gradients from one call (the _grad_xy entry
 * points; the same for the DeConv2d queries) */
size_t d8_conv2d_scratch_bytes(int dtype, int which, int B, int IH, int IW, int IC,
                               int OC, int FH, int FW, int covered, int sy, int sx, int dy, int dx);
int d8_conv2d(int dtype, const void *x, int B, int IH, int IW, int IC,
              const void *w, int OC, int FH, int FW, void *z,
              int covered, int sy, int sx, int dy, int dx,
              void *scratch, size_t scratch_bytes, void *stream);
int d8_conv2d_grad_x(int dtype, void *gx, int B, int IH, int IW, int IC,
                     const void *w, int OC, int FH, int FW, const void *gz,
                     int covered, int sy, int sx, int dy, int dx,
                     void *scratch, size_t scratch_bytes, void *stream);
int d8_conv2d_grad_y(int dtype, const void *x, int B, int IH, int IW, int IC,
                     void *gw, int OC, int FH, int FW, const void *gz,
                     int covered, int sy, int sx, int dy, int dx,
                     void *scratch, size_t scratch_bytes, void *stream);

size_t d8_deconv2d_scratch_bytes(int dtype, int which, int B, int IH, int IW, int IC,
                                 int OC, int FH, int FW, int covered, int sy, int sx);
int d8_deconv2d(int dtype, const void *x, int B, int IH, int IW, int IC,
                const void *w, int OC, int FH, int FW, void *z,
                int covered, int sy, int sx,
                void *scratch, size_t scratch_bytes, void *stream);
int d8_deconv2d_grad_x(int dtype, void *gx, int B, int IH, int IW, int IC,
                       const void *w, int OC, int FH, int FW, const void *gz,
                       int covered, int sy, int sx,
                       void *scratch, size_t scratch_bytes, void *stream);
int d8_deconv2d_grad_y(int dtype, const void *x, int B, int IH, int IW, int IC,
                       void *gw, int OC, int FH, int FW, const void *gz,
                       int covered, int sy, int sx,
                       void *scratch, size_t scratch_bytes, void *stream);

/* DeConv2d with the geometry given outright instead of derived from `covered`: the output is OH x OW and
 * z[b,oy,ox,:] sums the taps (fy,fx) with iy*sy == oy - padTop + fy, ix*sx == ox - padLeft + fx inside the input
 * (padTop, padLeft >= 0: the pads of the stride-1 correlation over the zero-inflated input, as returned by
 * d8_deconv2d_geometry).  Math::DeConv2d admits only two output sizes per input (deep8/src/nodes/DeConv2d.cpp:36-52,
 * pads deep8/src/math/DeConv2d.cpp:295-301); these entry points run the same kernels on any other, e.g. PyTorch's
 * ConvTranspose2d(k, s, p) = OH (IH-1)*s + k - 2p, padTop = k - 1 - p.  The gradients accumulate unless
 * overwrite != 0.  scratch from d8_deconv2d_scratch_bytes_ex.                                                  */
size_t d8_deconv2d_scratch_bytes_ex(int dtype, int which, int B, int IH, int IW, int IC,
                                    int OC, int FH, int FW, int OH, int OW, int padTop, int padLeft, int sy, int sx);
int d8_deconv2d_ex(int dtype, const void *x, int B, int IH, int IW, int IC,
                   const void *w, int OC, int FH, int FW, void *z,
                   int OH, int OW, int padTop, int padLeft, int sy, int sx,
                   void *scratch, size_t scratch_bytes, void *stream);
int d8_deconv2d_grad_x_ex(int dtype, void *gx, int B, int IH, int IW, int IC,
                          const void *w, int OC, int FH, int FW, const void *gz,
                          int OH, int OW, int padTop, int padLeft, int sy, int sx, int overwrite,
                          void *scratch, size_t scratch_bytes, void *stream);
int d8_deconv2d_grad_y_ex(int dtype, const void *x, int B, int IH, int IW, int IC,
                          void *gw, int OC, int FH, int FW, const void *gz,
                          int OH, int OW, int padTop, int padLeft, int sy, int sx, int overwrite,
                          void *scratch, size_t scratch_bytes, void *stream);

/* Overwrite forms of the four convolution gradients: the destination's old contents are ignored
 * (what "zero the gradient, then accumulate" leaves, without the fill and the read-back).      */
int d8_conv2d_grad_x_overwrite(int dtype, void *gx, int B, int IH, int IW, int IC,
                               const void *w, int OC, int FH, int FW, const void *gz,
                               int covered, int sy, int sx, int dy, int dx,
                               void *scratch, size_t scratch_bytes, void *stream);
int d8_conv2d_grad_y_overwrite(int dtype, const void *x, int B, int IH, int IW, int IC,
                               void *gw, int OC, int FH, int FW, const void *gz,
                               int covered, int sy, int sx, int dy, int dx,
                               void *scratch, size_t scratch_bytes, void *stream);
int d8_deconv2d_grad_x_overwrite(int dtype, void *gx, int B, int IH, int IW, int IC,
                                 const void *w, int OC, int FH, int FW, const void *gz,
                                 int covered, int sy, int sx,
                                 void *scratch, size_t scratch_bytes, void *stream);
int d8_deconv2d_grad_y_overwrite(int dtype, const void *x, int B, int IH, int IW, int IC,
                                 void *gw, int OC, int FH, int FW, const void *gz,
                                 int covered, int sy, int sx,
                                 void *scratch, size_t scratch_bytes, void *stream);

/* Both gradients of a convolution from one call: what the _grad_x call followed by the _grad_y call of the same
 * operator leave (Conv2d::backward / DeConv2d::backward run once per input, deep8/src/nodes/Conv2d.cpp:85-151,
 * deep8/src/nodes/DeConv2d.cpp:74-126, each a cublasSgemm / cublasHgemm sequence of its own:
 * deep8/src/math/Conv2d.cu:440-492 and :750-802, deep8/src/math/DeConv2d.cu:371-429 and :642-700).  The two are
 * independent of each other; on a layer whose products each leave compute units idle they run as ONE launch, the
 * workgroups of both side by side.  gw is bit for bit what the _grad_y call leaves; so is gx, except on small half
 * layers where the product behind gx, cut into pieces when it runs alone, runs whole beside the other's workgroups:
 * the same sums added in another order (equal within half rounding).  overwrite: bit 0 -- gx is
 * written instead of added to, bit 1 -- gw likewise.  scratch: the scratch query with which = 3 (room for both
 * gradients' scratch side by side); with less, but at least the larger of which = 1 and which = 2, the call still
 * works and large layers run as two launches.                                                                     */
int d8_conv2d_grad_xy(int dtype, const void *x, void *gx, int B, int IH, int IW, int IC,
                      const void *w, void *gw, int OC, int FH, int FW, const void *gz,
                      int covered, int sy, int sx, int dy, int dx, int overwrite,
                      void *scratch, size_t scratch_bytes, void *stream);
int d8_deconv2d_grad_xy(int dtype, const void *x, void *gx, int B, int IH, int IW, int IC,
                        const void *w, void *gw, int OC, int FH, int FW, const void *gz,
                        int covered, int sy, int sx, int overwrite,
                        void *scratch, size_t scratch_bytes, void *stream);
int d8_deconv2d_grad_xy_ex(int dtype, const void *x, void *gx, int B, int IH, int IW, int IC,
                           const void *w, void *gw, int OC, int FH, int FW, const void *gz,
                           int OH, int OW, int padTop, int padLeft, int sy, int sx, int overwrite,
                           void *scratch, size_t scratch_bytes, void *stream);

/* Test and measurement aid: how many of the _grad_xy calls above have run as one launch since the library was
 * loaded (no counterpart in the reference): those whose gradient of x runs whole, or with its remainder band, and
 * those whose two products are tiled and cut as they would be alone.  A call counts in one of the three at most.   */
unsigned long d8_conv_grad_pair_launches(void);
unsigned long d8_conv_grad_kept_pair_launches(void);
unsigned long d8_conv_grad_crowded_pair_launches(void);  /* likewise, Float32: 128 x 128 tiles in both, or more workgroups than run at once */
unsigned long d8_matmul_grad_pair_launches(void);  /* ... and of the d8_matmul_grad_xy calls: whole K steps, and no more workgroups than run at once; */
unsigned long d8_matmul_grad_kept_pair_launches(void);  /* the others: a K step (64 in Float16, 32 in Float32) that is cut short, or more workgroups */
unsigned long d8_matmul_grad_copied_calls(void);   /* d8_matmul_grad_xy calls that ran on copies of their odd operands */
unsigned long d8_matmul_copied_calls(void);        /* ... and d8_matmul and d8_matmul_bias_relu calls */
/* How many Conv2d / DeConv2d calls have run (each gradient is one; both gradients from one call are two), by route: 0 on an
 * interim matrix in scratch, 1 with the patches read by the GEMM's loader, 2 on the kernels for images of few channels. */
unsigned long d8_conv_route_calls(int route);

/* ---- Add (broadcasting) and ReLu -----------------------------------------------------------
 * The element-wise steps that follow MatrixMultiply / Conv2d in a network (bias, activation).
 * Shapes are Deep8's 5-entry enlarged form [batch, d0, d1, d2, d3]: dims right-aligned, padded
 * with 1 (deep8/include/utils/ShapeUtils.h:41-56); an operand axis equals z's or is 1.
 *
 * d8_add       z = x + y with broadcasting.  Replaces Math::AddGPU (deep8/include/math/Add.h:20,
 *              deep8/src/math/Add.cu:21-52).
 * d8_add_grad  g += dz summed over the axes where g has extent 1 and dz does not; this one map
 *              is both Math::AddGradXGPU and Math::AddGradYGPU (Add.h:31,42; Add.cu:64-133:
 *              the gradient op returns dz).  `scratch` (may be NULL; size from
 *              d8_add_grad_scratch_bytes, 16-byte aligned) lets the reduction run in two passes.
 * d8_relu      y = x > 0 ? x : 0.   Replaces Math::ReLuGPU (deep8/include/math/ReLu.h:19,
 *              deep8/src/math/ReLu.cu:20-59).
 * d8_relu_grad dx += x > 0 ? dy : 0.  Replaces Math::ReLuGradGPU (ReLu.h:30, ReLu.cu:61-116).     */
int d8_add(int dtype, const void *x, const int *xdims, const void *y, const int *ydims,
           void *z, const int *zdims, void *stream);
size_t d8_add_grad_scratch_bytes(int dtype, const int *gdims, const int *zdims);
int d8_add_grad(int dtype, void *g, const int *gdims, const void *dz, const int *zdims,
                void *scratch, size_t scratch_bytes, void *stream);
int d8_relu(int dtype, const void *x, void *y, long n, void *stream);
int d8_relu_grad(int dtype, const void *x, void *dx, const void *dy, long n, void *stream);
/* Overwrite forms of the two gradients: the destination's old contents are not read (what "zero the
 * gradient, then accumulate" leaves, deep8/src/model/EagerExecutor.cpp:51-65, without the fill and
 * the read-back).                                                                                   */
int d8_add_grad_overwrite(int dtype, void *g, const int *gdims, const void *dz, const int *zdims,
                          void *scratch, size_t scratch_bytes, void *stream);
int d8_relu_grad_overwrite(int dtype, const void *x, void *dx, const void *dy, long n, void *stream);

/* ---- bias and activation folded into the contraction --------------------------------------------------
 * In a network Add (a per-channel bias broadcast over the rows) and ReLu follow every MatrixMultiply / Conv2d as
 * passes of their own over the result (Math::AddGPU, deep8/src/math/Add.cu:21-52; Math::ReLuGPU,
 * deep8/src/math/ReLu.cu:20-59).  These entry points give the result of the three-call sequence from one call:
 *
 * d8_matmul_bias_relu   z = relu?(x * y + bias): d8_matmul, then bias[n] added along z's last axis (bias: that many
 *                       elements of the tensors' type, or NULL), then ReLu when relu != 0.  z's last axis has yc
 *                       elements when yc > 1; when y is a vector or a batch of vectors (yc == 1) z is [batch][xr]
 *                       (deep8/src/nodes/MatrixMultiply.cpp:23-27) and the bias has xr elements.
 * d8_conv2d_bias_relu   the same after d8_conv2d (bias: OC elements).
 *     Both apply bias and ReLu in the store of the product's kernel (before the one rounding to the element type)
 *     wherever that kernel is one of the tiled ones, and otherwise run the product followed by ONE in-place pass.
 *     Float32: bit for bit the result of d8_matmul / d8_conv2d, d8_add, d8_relu.  Float16: the fused store rounds
 *     once instead of three times.  scratch as for d8_matmul / d8_conv2d.  Float64 is rejected.
 * d8_bias_relu_grad     the way back in one pass over the [rows][cols] gradient of z: dpre = z > 0 ? dz : 0 is
 *                       written (dpre may be dz), and dbias (cols elements) receives its column sums, added to
 *                       what it holds when accumulate_bias != 0, else written.  z is the layer's output (it is
 *                       positive exactly where the pre-activation was).  Replaces Math::ReLuGradGPU
 *                       (ReLu.cu:61-116) + Math::AddGradYGPU (Add.cu:99-133); the sums are bit for bit those of
 *                       d8_add_grad on dpre.  scratch (may be NULL): d8_bias_relu_grad_scratch_bytes, 16-byte aligned.
 *                       dpre then feeds d8_matmul_grad_* / d8_conv2d_grad_* as dz.                                  */
int d8_matmul_bias_relu(int dtype, const void *x, int xb, int xr, int xc,
                        const void *y, int yb, int yr, int yc, const void *bias, int relu, void *z,
                        void *scratch, size_t scratch_bytes, void *stream);
int d8_conv2d_bias_relu(int dtype, const void *x, int B, int IH, int IW, int IC,
                        const void *w, int OC, int FH, int FW, const void *bias, int relu, void *z,
                        int covered, int sy, int sx, int dy, int dx,
                        void *scratch, size_t scratch_bytes, void *stream);
size_t d8_bias_relu_grad_scratch_bytes(int dtype, long rows, int cols);
int d8_bias_relu_grad(int dtype, const void *z, const void *dz, void *dpre, void *dbias, long rows, int cols,
                      int accumulate_bias, void *scratch, size_t scratch_bytes, void *stream);

/* ---- Minus, L1Norm / L2Norm, ReduceMean, AXPBY ------------------------------------------------
 * What a loss and a trainer step need on top of the operators above.  Shapes as for d8_add.
 * Reductions take an optional two-pass `scratch` (16-byte aligned; size from
 * d8_add_grad_scratch_bytes(dtype, shape of the reduced tensor, shape of the full tensor)).
 *
 * d8_minus            z = x - y with broadcasting.  Math::MinusGPU (deep8/include/math/Minus.h:16,
 *                     deep8/src/math/Minus.cu:21-52).  Math::MinusGradXGPU (Minus.h:27) is d8_add_grad.
 * d8_minus_grad_y     g -= dz summed over the axes where g has extent 1.  Math::MinusGradYGPU
 *                     (Minus.h:38, Minus.cu:103-147).
 * d8_l1norm           y[b] = sum_i |x[b][i]|.  Math::L1NormGPU (deep8/include/math/L1Norm.h,
 *                     deep8/src/math/L1Norm.cu:27-75).
 * d8_l1norm_grad      dx[b][i] += dy[b] * sign(x[b][i]) (sign(0) = 0).  Math::L1NormGradGPU
 *                     (L1Norm.cu:77-136).
 * d8_l2norm           y[b] = sqrt(sum_i x[b][i]^2).  Math::L2NormGPU (deep8/src/math/L2Norm.cu).
 * d8_l2norm_grad      dx[b][i] += dy[b] / y[b] * x[b][i].  Math::L2NormGradGPU.
 * d8_reduce_mean      y = mean of x over the axes where ydims is 1 and xdims is not (ydims is the
 *                     keepDims form of the output shape; dropping the axes does not move data).
 *                     Math::ReduceMeanGPU (deep8/include/math/ReduceMean.h, deep8/src/math/ReduceMean.cu:30-110).
 * d8_reduce_mean_grad dx += dy / count, dy broadcast over the reduced axes.  Math::ReduceMeanGradGPU
 *                     (ReduceMean.cu:112-203).
 * d8_axpby            z = alpha * x + beta * y (z may be x or y).  Math::AXPBYGPU
 *                     (deep8/include/math/AXPBY.h, deep8/src/math/AXPBY.cu:9-47): the SGD update.       */
int d8_minus(int dtype, const void *x, const int *xdims, const void *y, const int *ydims,
             void *z, const int *zdims, void *stream);
int d8_minus_grad_y(int dtype, void *g, const int *gdims, const void *dz, const int *zdims,
                    void *scratch, size_t scratch_bytes, void *stream);
int d8_l1norm(int dtype, const void *x, void *y, int batch, long size,
              void *scratch, size_t scratch_bytes, void *stream);
int d8_l1norm_grad(int dtype, const void *x, void *dx, const void *dy, int batch, long size, void *stream);
int d8_l2norm(int dtype, const void *x, void *y, int batch, long size,
              void *scratch, size_t scratch_bytes, void *stream);
int d8_l2norm_grad(int dtype, const void *x, void *dx, const void *y, const void *dy, int batch, long size,
                   void *stream);
int d8_reduce_mean(int dtype, const void *x, const int *xdims, void *y, const int *ydims,
                   void *scratch, size_t scratch_bytes, void *stream);
int d8_reduce_mean_grad(int dtype, void *dx, const int *xdims, const void *dy, const int *ydims, void *stream);
int d8_axpby(int dtype, const void *x, float alpha, const void *y, float beta, void *z, long n, void *stream);
/* d8_adam_update: gradient += weight_decay * value; m = beta1 m + (1 - beta1) gradient;
 * v = beta2 v + (1 - beta2) gradient^2; value -= ratio * m / (sqrt(v) + epsilon) with
 * ratio = learning_rate * sqrt(1 - beta2^steps) / (1 - beta1^steps), steps < 1 taken as 1.
 * Math::AdamUpdateGPU (deep8/include/math/AdamUpdate.h, deep8/src/math/AdamUpdate.cu:9-47).      */
int d8_adam_update(int dtype, void *value, void *gradient, void *m, void *v, float beta1, float beta2,
                   float epsilon, float learning_rate, float weight_decay, long steps, long n, void *stream);

/* ---- MaxPooling2d / AvgPooling2d --------------------------------------------------------------
 * x [B][IH][IW][C], y [B][OH][OW][C]; (OH, OW, padTop, padLeft) = d8_conv2d_geometry(IH, IW, FH, FW,
 * covered, sy, sx, 1, 1).  Semantics are those of Deep8's CPU path: the forward window is cut from
 * the zero-padded image (zeros take part in the maximum and in the mean, which divides by FH * FW);
 * the max gradient goes to the first maximum of the window clipped to the image; gradients are
 * added into dx.
 * d8_maxpool2d / _grad  Math::MaxPooling2dGPU / MaxPooling2dGradGPU (deep8/include/math/MaxPooling2d.h,
 *                       deep8/src/math/MaxPooling2d.cu:41-147 -- a cuDNN call there; checks and CPU
 *                       semantics deep8/src/math/MaxPooling2d.cpp:6-251)
 * d8_avgpool2d / _grad  Math::AvgPooling2dGPU / AvgPooling2dGradGPU (deep8/include/math/AvgPooling2d.h,
 *                       deep8/src/math/AvgPooling2d.cu; CPU semantics AvgPooling2d.cpp:99-245)          */
int d8_maxpool2d(int dtype, const void *x, void *y, int B, int IH, int IW, int C,
                 int FH, int FW, int covered, int sy, int sx, void *stream);
int d8_maxpool2d_grad(int dtype, const void *x, void *dx, const void *dy, int B, int IH, int IW, int C,
                      int FH, int FW, int covered, int sy, int sx, void *stream);
int d8_avgpool2d(int dtype, const void *x, void *y, int B, int IH, int IW, int C,
                 int FH, int FW, int covered, int sy, int sx, void *stream);
int d8_avgpool2d_grad(int dtype, void *dx, const void *dy, int B, int IH, int IW, int C,
                      int FH, int FW, int covered, int sy, int sx, void *stream);
/* The two pooling gradients written over dx instead of added to it (see d8_relu_grad_overwrite). */
int d8_maxpool2d_grad_overwrite(int dtype, const void *x, void *dx, const void *dy, int B, int IH, int IW, int C,
                                int FH, int FW, int covered, int sy, int sx, void *stream);
int d8_avgpool2d_grad_overwrite(int dtype, void *dx, const void *dy, int B, int IH, int IW, int C,
                                int FH, int FW, int covered, int sy, int sx, void *stream);

/* ---- a transformer layer --------------------------------------------------------------------------
 * Three operators of such a layer, to stand beside MatrixMultiply and Add; no counterpart in the reference.  Float16 and Float32.  Rows
 * (tokens) of several heads lie `ld` elements apart, the heads of a row next to each other, so that queries, keys and values
 * may be parts of one product's rows.  Gradients are added to what their destination holds unless their bit of `overwrite` is set.
 * Sums, statistics of norms and softmax are fp32; results are rounded once.  Between two products Float16 calls hold halves: d8_attention its
 * probabilities, d8_attention_grad these and the scores' gradients, d8_matmul_gated_grad the gradients of g and u.  Each adds about as much
 * error as the result's rounding (2.6 to 3 10^-4 of a result's norm in all, where the rounding alone is 2.1).
 *
 * d8_rotary_table        table[p][i] = (cos, sin)(p f_i) in fp32, i < rotary / 2, positions p < positions, f_i = base^(-2 i / rotary);
 *                        angles in fp64.  For contexts longer than a model was trained on, factor > 1 slows the rotation down:
 *                        every f_i is divided by it when slow_above is 0; else those with a wave length (2 pi / f_i positions)
 *                        of at least slow_above, those of at most keep_below stay, and between the two the share that stays
 *                        goes linearly with 1 / wave length.
 * d8_head_norm_rotary    each head x of `dim` elements of queries and keys becomes n = x / sqrt(mean(x^2) + epsilon) * weight (norm != 0;
 *                        weight: dim elements or NULL for ones), and the first `rotary` elements of n are turned by the angles of
 *                        the token's position: the pairs (i, i + rotary / 2), or with interleaved != 0 the pairs (2 i, 2 i + 1).
 *                        positions[tokens] (NULL: a token's row); a position outside the table counts as its nearest.
 *                        Outputs may be the inputs.  q_heads or k_heads may be 0.  dim <= 2048.
 * d8_head_norm_rotary_grad  from q, k and the gradients of the outputs (dq_out, dk_out) those of q, k (bit 0 of overwrite) and of
 *                        the weights (bit 1; NULL: not wanted).  dq may be dq_out, dk may be dk_out.
 * d8_attention           sequence s has queries q_starts[s] .. q_starts[s + 1] - 1 and keys k_starts[s] .. k_starts[s + 1] - 1 (rows of
 *                        q and k; arrays of sequences + 1 on the device; what reaches beyond the tensors is cut, and a start that lies before
 *                        an earlier one counts as that one, so sequences never overlap).  A query sees its
 *                        sequence's keys, causal != 0: query t of nq sees the keys up to t + nk - nq, so the last query sees them
 *                        all.  o = softmax(scale q k^T) v, head i with the keys and values of head i / (heads / kv_heads).
 *                        lse[heads][q_tokens] (may be NULL): the logarithm of the sum of exp(score).  A query that sees nothing
 *                        gets o = 0 and lse = -infinity.  Rows of no sequence are left alone.  dim <= 256.  The same
 *                        call serves training (q_starts = k_starts), a prompt's next part and a step of decoding (one query a sequence).
 *                        A cache with free places after each sequence's keys: count every gap as a sequence of keys without a query
 *                        (q_starts 0, 1, 1, 2; k_starts 0, length 0, capacity, capacity + length 1).  NaN and infinities outside a
 *                        query's sequence never reach it.  Inside it a hidden key's weight is 0, as if written out: NaN or infinity
 *                        in that key's row of v (gradients: of k, v, and of the query's q, dout) can still make 0 times it, NaN.
 * d8_attention_grad      the gradients of q (bit 0 of overwrite), k (bit 1) and v (bit 2) from those of o (dout), with o and lse as the
 *                        forward call left them.  The same bits every time.  Float16: a score's gradient is held relative to the largest that it can be,
 *                        in a row of dq by that row and its keys, in a key's dk by the rows (same sequence, heads that share the key) and keys of
 *                        its workgroup.  A term keeps its bits down to 2^-28 of that and is lost below 2^-39.
 *     scratch: d8_attention_scratch_bytes, which = 0 forward, 1 gradients; 16-byte aligned.
 * d8_matmul_gated        h = act(g) * u with (g | u) = x w: w is [inner][2 * cols], its first `cols` columns the gate's.  act: D8_GATE_*.
 *                        pre (may be NULL): [rows][2 * cols], receives g and u for the gradients.  Refused: 128 rows of x (all, if they
 *                        are fewer) or 32 rows of w (Float16, more than 64 rows of x: 64) of more than 2 GiB.
 * d8_matmul_gated_grad   dx (bit 0 of overwrite) and dw (bit 1) from dh, with pre as the forward call left it.
 *     scratch: d8_matmul_gated_scratch_bytes, which = 0 forward with x and w at multiples of 16 bytes, 2 forward wherever they lie
 *     (room for a copy of each, rows padded to 16 bytes, unless which = 0 has it), 1 gradients; 16-byte aligned. */
#define D8_GATE_SILU    0 /* a sigmoid(a)                 */
#define D8_GATE_GELU    1 /* a (1 + erf(a / sqrt 2)) / 2  */
#define D8_GATE_RELU    2
#define D8_GATE_SIGMOID 3
int d8_rotary_table(float *table, int positions, int rotary, double base, double factor, double keep_below, double slow_above,
                    void *stream);
int d8_head_norm_rotary(int dtype, const void *q, long ldq, int q_heads, const void *q_weight, void *q_out, long ldq_out,
                        const void *k, long ldk, int k_heads, const void *k_weight, void *k_out, long ldk_out,
                        int tokens, int dim, int norm, float epsilon, const int *positions, const float *table,
                        int table_positions, int rotary, int interleaved, void *stream);
size_t d8_head_norm_rotary_grad_scratch_bytes(int dtype, int tokens, int q_heads, int k_heads, int dim);
int d8_head_norm_rotary_grad(int dtype, const void *q, long ldq, int q_heads, const void *q_weight, const void *dq_out, long lddq_out,
                             void *dq, long lddq, void *dq_weight, const void *k, long ldk, int k_heads, const void *k_weight,
                             const void *dk_out, long lddk_out, void *dk, long lddk, void *dk_weight, int tokens, int dim, int norm,
                             float epsilon, const int *positions, const float *table, int table_positions, int rotary,
                             int interleaved, int overwrite, void *scratch, size_t scratch_bytes, void *stream);
size_t d8_attention_scratch_bytes(int dtype, int which, int sequences, int q_tokens, int k_tokens, int heads, int kv_heads, int dim,
                                  int causal);
int d8_attention(int dtype, const void *q, long ldq, const void *k, long ldk, const void *v, long ldv, void *o, long ldo, float *lse,
                 const int *q_starts, const int *k_starts, int sequences, int q_tokens, int k_tokens, int heads, int kv_heads, int dim,
                 float scale, int causal, void *scratch, size_t scratch_bytes, void *stream);
int d8_attention_grad(int dtype, const void *q, long ldq, const void *k, long ldk, const void *v, long ldv, const void *o, long ldo,
                      const float *lse, const void *dout, long lddo, void *dq, long lddq, void *dk, long lddk, void *dv, long lddv,
                      const int *q_starts, const int *k_starts, int sequences, int q_tokens, int k_tokens, int heads, int kv_heads,
                      int dim, float scale, int causal, int overwrite, void *scratch, size_t scratch_bytes, void *stream);
size_t d8_matmul_gated_scratch_bytes(int dtype, int which, int rows, int inner, int cols);
int d8_matmul_gated(int dtype, const void *x, int rows, int inner, const void *w, int cols, int act, void *pre, void *h,
                    void *scratch, size_t scratch_bytes, void *stream);
int d8_matmul_gated_grad(int dtype, const void *x, void *dx, int rows, int inner, const void *w, void *dw, int cols, int act,
                         const void *pre, const void *dh, int overwrite, void *scratch, size_t scratch_bytes, void *stream);

/* ---- a transformer layer: the norm of its rows, and what it takes to serve it in 8 bits ---------------------
 * No counterpart in the reference.  Float16 and Float32 (of x, q, k, v and results; sums, statistics and scales are fp32).
 *
 * d8_layer_norm          each row x of `cols` elements becomes (x - m) / sqrt(mean((x - m)^2) + epsilon) * weight + bias, m = mean(x) (weight, bias:
 *                        cols elements, or NULL for ones and zeros).  Rows lie ldx and ldy elements apart; y may be x (ldy = ldx then).
 *                        (The sum of a row's squares has to be one that fp32 holds: elements of less than 10^17 or so.)
 * d8_layer_norm_grad     from x and the gradient of y (dy) those of x (bit 0 of overwrite; NULL: not wanted) and of weight and bias (bit 1; NULL: not
 *                        wanted); gradients are added to what their destination holds unless their bit of `overwrite` is set.  dx may be dy or x (its rows then lie
 *                        where theirs do).  The same bits every time.  scratch: d8_layer_norm_grad_scratch_bytes, 16-byte aligned; none if neither weight's nor bias'
 *                        gradient is wanted.
 *
 * Products in 8-bit integers.  A matrix of codes has its reduction axis along memory: a row of x, or a column of w, takes d8_int8_pitch(inner) bytes
 * (`inner` rounded up to 128), codes of -128 to 127 and behind them zeros, which take part in the sums.  16-byte aligned.  inner <= 131071.
 * d8_quantize_rows       each row of x (cols elements, ldx apart): scale = max |x| / 127 (in fp32; at least 2^-100), codes x / scale rounded to the nearest
 *                        whole number, halves to the even one, from the exact quotient.  A row with NaN or an infinity: scale NaN, codes 0.
 * d8_quantize_columns    the same for each column of w [rows][cols] (rows ldw apart), whose codes become a row: for weights, laid out once.
 * d8_matmul_int8         z[i][j] = x_scales[i] w_scales[j] sum over k of x[i][k] w[j][k], rows of z ldz apart: x (rows) and w (cols) as above, sums exact,
 *                        multiplied by one scale and then the other in fp32, rounded once to the element type.
 *     scratch: d8_matmul_int8_scratch_bytes, 16-byte aligned.
 *
 * A cache of keys and values in 8-bit integers, in pages of D8_CACHE_PAGE tokens with a scale for each page and key head.  With pitch = dim rounded up to 16:
 * k_codes [pages][kv_heads][token][pitch], v_codes [pages][kv_heads][pitch][token], both 16-byte aligned, k_scales and v_scales [pages][kv_heads]; a code
 * stands for code * scale.  Which pages a sequence has: table[sequences][table_pages], on the device; entry p is the page of its tokens 64 p ..
 * 64 p + 63, one outside 0 .. pages - 1 is no page.  lengths[sequences], on the device: how many tokens a sequence has in the cache, those
 * that the call brings among them; rows starts[s] .. starts[s + 1] - 1 of a call (starts as d8_attention's) are its last ones.  dim <= 256.
 * d8_cache_append        rows of k and v (kv_heads heads each) into their places.  A page's scale is a power of two, at least 2^-100: the least of which 127
 *                        reach the largest element since the page's first token was written.  Codes are exact quotients rounded to the nearest, halves
 *                        to the even one; where new tokens raise the scale, codes that are there are rounded again in the same way.  NaN or an infinity makes
 *                        its page and head's scale NaN, and so everything that is read from it, until its first token is written anew.  A token whose
 *                        place is before the first or has no page is left out.  Two sequences must not bring tokens to one page in one
 *                        call, nor one sequence to a page that stands twice in its table; full pages may be in any number of tables.
 * d8_cache_read          the values of those places into rows of k and v, zeros for a token whose place is before the first or has no page.  Where codes stand
 *                        for more than the type holds (65504 as half is 64 steps of 1024), its largest number, here and in attention's results.
 * d8_attention_cache     o = softmax(scale q k^T) v over the values that such a cache holds, head i with the keys and values of head i / (heads / kv_heads);
 *                        scales may be any numbers.  causal != 0: query t of a sequence's n sees the keys of its places up to t + length - n, so the
 *                        last one sees them all; 0: every key.  Keys without a page are not seen.  lse[heads][q_tokens] (may be NULL) as
 *                        d8_attention's; a query that sees nothing gets o = 0 and lse = -infinity; rows of no sequence are left alone.  The same call
 *                        serves a prompt's next part, a step of decoding and attention to another sequence's states.  The same bits every time.
 *     scratch: d8_attention_cache_scratch_bytes, 16-byte aligned.
 */
#define D8_CACHE_PAGE 64
int d8_layer_norm(int dtype, const void *x, long ldx, const void *weight, const void *bias, void *y, long ldy, int rows, int cols, float epsilon,
                  void *stream);
size_t d8_layer_norm_grad_scratch_bytes(int dtype, int rows, int cols);
int d8_layer_norm_grad(int dtype, const void *x, long ldx, const void *weight, const void *dy, long lddy, void *dx, long lddx, void *dweight,
                       void *dbias, int rows, int cols, float epsilon, int overwrite, void *scratch, size_t scratch_bytes, void *stream);

int d8_int8_pitch(int inner);
int d8_quantize_rows(int dtype, const void *x, long ldx, int rows, int cols, signed char *codes, float *scales, void *stream);
int d8_quantize_columns(int dtype, const void *w, long ldw, int rows, int cols, signed char *codes, float *scales, void *stream);
size_t d8_matmul_int8_scratch_bytes(int rows, int inner, int cols);
int d8_matmul_int8(int dtype, const signed char *x, const float *x_scales, int rows, int inner, const signed char *w, const float *w_scales, int cols,
                   void *z, long ldz, void *scratch, size_t scratch_bytes, void *stream);

int d8_cache_append(int dtype, const void *k, long ldk, const void *v, long ldv, signed char *k_codes, float *k_scales, signed char *v_codes,
                    float *v_scales, const int *starts, const int *lengths, const int *table, int sequences, int tokens, int table_pages, int pages,
                    int kv_heads, int dim, void *stream);
int d8_cache_read(int dtype, void *k, long ldk, void *v, long ldv, const signed char *k_codes, const float *k_scales, const signed char *v_codes,
                  const float *v_scales, const int *starts, const int *lengths, const int *table, int sequences, int tokens, int table_pages, int pages,
                  int kv_heads, int dim, void *stream);

size_t d8_attention_cache_scratch_bytes(int dtype, int sequences, int q_tokens, int table_pages, int heads, int kv_heads, int dim);
int d8_attention_cache(int dtype, const void *q, long ldq, const signed char *k_codes, const float *k_scales, const signed char *v_codes,
                       const float *v_scales, void *o, long ldo, float *lse, const int *starts, const int *lengths, const int *table, int sequences,
                       int q_tokens, int table_pages, int pages, int heads, int kv_heads, int dim, float scale, int causal, void *scratch,
                       size_t scratch_bytes, void *stream);

/* ---- measurement aid (no counterpart in the reference) ---------------------------------------
 * d8_mfma_stream issues the GEMM kernels' MFMA instruction for `dtype` (D8_FLOAT16, D8_FLOAT32 or
 * D8_FLOAT64) back to back on operands taken from `operands` (any device buffer; 16-byte aligned)
 * and held in registers, on every CU, no LDS or global traffic in the loop.  Timing one launch gives the rate the matrix
 * pipe sustains on those operand bits, i.e. the ceiling a GEMM has on that data.  `out` takes
 * d8_mfma_stream_out_bytes() bytes; *flops receives the flops one launch performs.             */
/* A second aid needs no entry point: with D8_GEMM_STAMPS set in the environment before the first launch, a
 * d8_gemm call that runs the large-output fp16 kernel and is given an 8-byte aligned workspace of at least
 * 48 bytes per 256 x 256 tile of C leaves there, per tile, six 64-bit values: the chip's 100 MHz wall
 * clock when its workgroup turned to the tile, when its K loop began and ended and when its epilogue was through
 * (its stores acknowledged, for the workgroup's last tile), and the shader clock before and after the loop.
 * d8_matmul_grad_xy does the same with its scratch when the two products run as one launch (the first product's
 * tiles, then the second's).                                                                            */
/* A third one, for the tiled kernels (fp16 / fp32 products and the convolutions they carry): after
 * d8_gemm_phase_record(records, bytes) every tiled launch whose records fit leaves 64 bytes per workgroup in
 * `records` (a device buffer, 8-byte aligned; index = workgroup id x + grid size x * id z): the same four wall
 * clock values and two shader clock values, then (XCC_ID << 32 | HW_ID) of the wave that wrote them and 1 if the
 * workgroup worked on a remainder band.  Each launch writes from index 0, so read the buffer between launches.
 * records = null switches the records off again.  Process-wide and not thread-safe: a tool for one measuring thread. */
int d8_gemm_phase_record(void *records, size_t bytes);
size_t d8_mfma_stream_out_bytes(void);
int d8_mfma_stream(int dtype, const void *operands, size_t operand_bytes, void *out, int iters,
                   double *flops, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* DEEP8_HIP_H */
