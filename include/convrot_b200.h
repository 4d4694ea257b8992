/*
 * C ABI of the B200 (sm_100a) ConvRot W4A4 library, libconvrot_b200.so.
 *
 * Drop-in for the HIP library of 0xDELUXA/ComfyUI-INT4-ConvRot-RDNA4
 * (_int4/int4_gemm.hip). Paths below are relative to that project.
 *
 * Conventions (same as the reference exports, _int4/int4_gemm.hip:627-741):
 *   - all pointers are device pointers; the caller allocates every output;
 *   - `stream` is a cudaStream_t passed as void* (NULL = legacy default stream);
 *   - launches are asynchronous and nothing synchronises inside a call;
 *   - return 0 on success, -1 when a shape/pointer precondition fails (nothing
 *     is launched; ck_convrot_last_error() explains), otherwise a cudaError_t.
 *
 * Layouts (the reference codec, _int4/_codec.py:19-36):
 *   packed int4 matrix [rows, K/2] int8, row-major; byte j of a row holds
 *   column 2j in its low nibble and column 2j+1 in its high nibble, both two's
 *   complement. Scales are float32, one per row (tokens) / output channel.
 */
#ifndef CONVROT_B200_H
#define CONVROT_B200_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Fused ConvRot rotation + row-wise int4 quantization + packing.
 * Replaces ck_convrot_quant_int4 (_int4/int4_gemm.hip:650-660), bound by
 * convrot_quant_int4 (_int4/hip_loader.py:74-92).
 *   x        [M, K] activations, in_dtype 0 = f32, 1 = bf16, 2 = f16
 *   qout     [M, K/2] int8 packed codes
 *   scaleout [M] f32 row scales
 * G in {16, 64, 256}, K % G == 0, K % 16 == 0. Quantizer arithmetic follows
 * the eager path (_int4/eager.py:112-120) in the activation dtype. */
int ck_convrot_quant_int4(const void* x, int in_dtype, void* qout, void* scaleout,
                          int M, int K, int G, void* stream);

/* Row-wise int4 quantization + packing of an already rotated activation
 * (rotation skipped). Replaces quantize_signed_int4_rowwise
 * (_int4/eager.py:112-120) for device tensors; same arguments as above minus G. */
int ck_int4_quant_rowwise(const void* x, int in_dtype, void* qout, void* scaleout,
                          int M, int K, void* stream);

/* out[m, n] = ((float(D[m, n]) * xscale[m]) * wscale[n]) + bias[n],
 * D = exact int32 sum_k X[m, k] * W[n, k] over packed codes.
 * Replaces ck_int4_convrot_gemm (_int4/int4_gemm.hip:711-741), bound by
 * int4_convrot_gemm (_int4/hip_loader.py:158-207).
 *   Xp [M, K/2], Wp [N, K/2] packed int8 (16-byte aligned)
 *   xscale [M], wscale [N], bias [N] or NULL: f32
 *   out [M, N], out_dtype 0 = f32, 1 = bf16
 * K % 32 == 0 and K <= 65536. */
int ck_int4_convrot_gemm(const void* Xp, const void* Wp, const void* xscale, const void* wscale,
                         const void* bias, void* out, int M, int N, int K, int out_dtype,
                         void* stream);

/* Workspace bytes that ck_convrot_w4a4_linear needs for M rows of K: the
 * activation codes and the row scales [M] f32, each from a 256-byte boundary.
 * The codes take [M, K/2] bytes (packed) below 129 rows and [M, K] bytes (one
 * per code, for the A8 form below) from 129 rows on. No reference counterpart. */
size_t ck_convrot_w4a4_linear_workspace_size(int M, int K);

/* The whole W4A4 linear in one call: rotate + quantize x (as
 * ck_convrot_quant_int4) into `workspace`, then
 * out = ((float(D) * xs[m]) * wscale[n]) + bias[n] (as ck_int4_convrot_gemm).
 * Replaces the two-call sequence of the reference's Python convrot_w4a4_linear
 * (_int4/__init__.py:94-135: convrot_quant_int4 then int4_convrot_gemm); no
 * single HIP export does both. Differences from calling the two exports:
 *   - bias is read in its own dtype, bias_dtype 0 = f32, 1 = bf16, 2 = f16
 *     (widening is exact, so results equal an fp32-converted bias);
 *   - the GEMM launch is a programmatic dependent of the quantizer launch;
 *   - bf16 x with 129+ rows, K % 256 == 0 and G in {64, 256} takes the A8
 *     form: codes written one per byte, then ck_int4_convrot_gemm_a8 (same
 *     accumulators, same output bits).
 *   x [M, K] in_dtype (0 f32, 1 bf16, 2 f16); Wp [N, K/2]; wscale [N] f32;
 *   out [M, N] out_dtype (0 f32, 1 bf16); G in {16, 64, 256}, K % G == 0,
 *   K % 32 == 0; workspace 256-byte aligned, at least
 *   ck_convrot_w4a4_linear_workspace_size(M, K) bytes, no initial contents
 *   needed; two calls in flight at once need two workspaces. */
int ck_convrot_w4a4_linear(const void* x, int in_dtype, const void* Wp, const void* wscale,
                           const void* bias, int bias_dtype, void* out, int out_dtype,
                           int M, int N, int K, int G, void* workspace, size_t workspace_bytes,
                           void* stream);

/* ck_convrot_w4a4_linear for callers that cannot allocate device memory (a
 * host framework that owns every device buffer through its own arena and only
 * hands this library inputs and outputs, a plugin ABI with plain pointers and
 * no allocator): the same arguments minus the workspace, which is replaced by
 * a static 128 MiB device array per device, placed when the library's no-alloc
 * module loads on that device. The entry itself allocates nothing. No
 * reference counterpart: the reference always allocates its intermediates
 * with torch.
 *   - limit: ck_convrot_w4a4_linear_workspace_size(M, K) <= 134217728 bytes
 *     (e.g. M = 18432 rows at K = 12288); larger sizes return -1 before any
 *     CUDA call, with the reason in ck_convrot_last_error();
 *   - nothing in the scratch has to start at zero (it is fully rewritten by
 *     each call before it is read);
 *   - one scratch per device: calls that may overlap in time (other streams,
 *     other host threads) race on it; calls on one stream are ordered and safe;
 *   - the first call on each device does the setup (a cudaGetSymbolAddress
 *     with that device current), and so does the first call after that
 *     device's primary context was reset: make it before any stream capture;
 *   - with lazy module loading (the default) only processes that call this
 *     entry hold the 128 MiB; with CUDA_MODULE_LOADING=EAGER every process
 *     that loads the library holds it on each device it uses. */
int ck_convrot_w4a4_linear_noalloc(const void* x, int in_dtype, const void* Wp, const void* wscale,
                                   const void* bias, int bias_dtype, void* out, int out_dtype,
                                   int M, int N, int K, int G, void* stream);

/* ck_int4_convrot_gemm plus a fused Dynamic-LoRA side path:
 *   out[m, n] = (((float(D) * xscale[m]) * wscale[n]) + bias[n]) + lora_scale * L[m, n],
 *   L = lora_t[m, :] . lora_b[n, :]  (fp16 operands, fp32 tensor-core accumulation).
 * lora_t = x A^T [M, rank] and lora_b = B [N, rank] are fp16 row-major (the
 * reference's adapter dtype, int4_ops.py:165-167); rank a
 * multiple of 8 in [8, 64]; bias in bias_dtype as for ck_convrot_w4a4_linear.
 * Replaces the unfused per-adapter `out + v.h(x, out)`
 * of the node's forward (int4_ops.py:181-192, :383); no HIP export counterpart. */
int ck_int4_convrot_gemm_lora(const void* Xp, const void* Wp, const void* xscale, const void* wscale,
                              const void* bias, int bias_dtype, void* out, int M, int N, int K,
                              int out_dtype, const void* lora_t, const void* lora_b, int rank,
                              float lora_scale, void* stream);

/* ck_int4_convrot_gemm_lora on int8 operands X [M, K], W [N, K] (the W8A8 tier,
 * or int4 codes sign-extended by ck_int4_unpack / ck_convrot_quant_int4_unpacked,
 * which give the same D and so the same output bits); same epilogue, arguments
 * and return codes. No reference counterpart (the reference's int8 layers add
 * the LoRA side path after the GEMM, int4_ops.py:371-383). */
int ck_int8_convrot_gemm_lora(const void* X, const void* W, const void* xscale, const void* wscale,
                              const void* bias, int bias_dtype, void* out, int M, int N, int K,
                              int out_dtype, const void* lora_t, const void* lora_b, int rank,
                              float lora_scale, void* stream);

/* accum[m, n] += (float(D[m, n]) * xscale[m]) * wscale[n] into a caller-zeroed
 * f32 [M, N] buffer. Replaces ck_int4_convrot_gemm_splitk
 * (_int4/int4_gemm.hip:634-645). The reference splits K and adds float
 * partials with atomics; here D is reduced in int32 first, so the result is
 * deterministic. `nsplit` (>= 1) is accepted for ABI compatibility. */
int ck_int4_convrot_gemm_splitk(const void* Xp, const void* Wp, const void* xscale,
                                const void* wscale, void* accum, int M, int N, int K,
                                int nsplit, void* stream);

/* Raw exact int32 accumulators acc[M, N] = sum_k X[m, k] * W[n, k].
 * No reference counterpart as an export: the reference computes these inside
 * its GEMM (_int4/int4_gemm.hip:204-232); exposed for bit-exact parity checks. */
int ck_int4_gemm_s32(const void* Xp, const void* Wp, void* acc, int M, int N, int K, void* stream);

/* W8A8 tier (the int8 middle tier of mixed precision).
 *
 * Fused ConvRot rotation + row-wise int8 quantization, codes not packed.
 * Replaces ck_convrot_quant_int8 (_int4/int4_gemm.hip:664-672), bound by
 * convrot_quant_int8 (_int4/hip_loader.py:95-113); the quantizer arithmetic is
 * the eager one in the activation dtype (_int4/int8_eager.py:22-27: scale =
 * dtype(absmax / 127), q = rint(dtype(x / scale)) clamped to +-127).
 *   x [M, K] (in_dtype must be 1 = bf16), qout [M, K] int8 (16-byte aligned),
 *   scaleout [M] f32; G in {64, 256} and K % 256 == 0 (other dtypes, G = 16 or
 *   ragged K return -1: the caller keeps its torch path, as the reference's
 *   Python layer does for shapes its kernel does not take). */
int ck_convrot_quant_int8(const void* x, int in_dtype, void* qout, void* scaleout,
                          int M, int K, int G, void* stream);

/* out[m, n] = ((float(D[m, n]) * xscale[m]) * wscale[n]) + bias[n],
 * D = exact int32 sum_k X[m, k] * W[n, k] of int8 values.
 * Replaces ck_int8_convrot_gemm (_int4/int4_gemm.hip:676-705), bound by
 * int8_convrot_gemm (_int4/hip_loader.py:116-150).
 *   X [M, K], W [N, K] int8 (16-byte aligned), xscale [M], wscale [N], bias [N]
 *   or NULL: f32; out [M, N], out_dtype 0 = f32, 1 = bf16; K % 16 == 0. */
int ck_int8_convrot_gemm(const void* X, const void* W, const void* xscale, const void* wscale,
                         const void* bias, void* out, int M, int N, int K, int out_dtype,
                         void* stream);

/* Raw exact int32 accumulators of the int8 product (no reference export; for
 * parity checks, like ck_int4_gemm_s32). */
int ck_int8_gemm_s32(const void* X, const void* W, void* acc, int M, int N, int K, void* stream);

/* The rotation fused into the producer of x (no reference counterpart; the
 * reference quantizes what the model's LayerNorm/modulation kernels wrote):
 * each bf16 row is normalised and modulated as a Flux block does before its
 * QKV or MLP-up projection,
 *   y = bf16(bf16(bf16(1 + mod_scale[k]) * xn) + mod_shift[k]),
 *   xn = bf16((x - mean) * rstd), rstd = 1 / sqrt(var + eps)
 * (LayerNorm without affine, biased variance; fp32 statistics in a fixed order:
 * lane l of a warp sums elements l, l + 32, ... then an xor butterfly of the 32
 * lane sums), then rotated and quantized exactly as ck_convrot_quant_int4 would
 * quantize y. y never goes to memory. mod_scale / mod_shift: bf16 [K], one
 * vector for all M rows (call once per batch item), NULL = zeros (plain
 * LayerNorm). bf16 x only; G in {64, 256}; K % 256 == 0, K <= 6144.
 * unpacked = 1 writes one sign-extended int8 per code ([M, K], the A8 form's
 * operand), 0 packed codes ([M, K/2]). */
int ck_convrot_quant_int4_lnmod(const void* x, const void* mod_scale, const void* mod_shift, float eps,
                                void* qout, void* scaleout, int M, int K, int G, int unpacked, void* stream);

/* ck_convrot_w4a4_linear of the modulated LayerNorm of x (as above), one pass
 * over x: out = y @ W^T + bias with the int4 path's arithmetic; same workspace
 * size rule (ck_convrot_w4a4_linear_workspace_size). */
int ck_convrot_w4a4_linear_lnmod(const void* x, const void* mod_scale, const void* mod_shift, float eps,
                                 const void* Wp, const void* wscale, const void* bias, int bias_dtype,
                                 void* out, int out_dtype, int M, int N, int K, int G, void* workspace,
                                 size_t workspace_bytes, void* stream);

/* Column-split linear over peer memory (no reference counterpart: the
 * reference runs on one device). P ranks (one process per GPU) each own N/P
 * weight rows; every rank's GEMM stores its column block straight into every
 * rank's [M, ldo] output through peer mappings over NVLink, then
 * ck_peer_barrier tells each rank that all blocks have landed in its output.
 *
 * ck_peer_buffer_alloc: cudaMalloc of `bytes` (zeroed) and its 64-byte CUDA IPC
 * handle; ck_peer_buffer_open maps another process's buffer from its handle
 * (ck_peer_buffer_close unmaps it); ck_peer_buffer_free frees an own buffer. */
int ck_peer_buffer_alloc(size_t bytes, void** ptr, void* ipc_handle);
int ck_peer_buffer_open(const void* ipc_handle, void** ptr);
int ck_peer_buffer_close(void* ptr);
int ck_peer_buffer_free(void* ptr);

/* ck_int4_convrot_gemm_a8 (packed weights, int8 activation codes, optional
 * LoRA side path; same D, epilogue and output bits) storing its [M, N] result
 * as columns col0 .. col0 + N of the [M, ldo] row-major matrices outs[0 ..
 * nouts) (1 to 8 pointers, any of them peer mappings; ldo and col0 multiples
 * of 8). Plain stores, no multicast. */
int ck_int4_convrot_gemm_a8_peers(const void* X8, const void* Wp, const void* xscale, const void* wscale,
                                  const void* bias, int bias_dtype, void* const* outs, int nouts,
                                  int ldo, int col0, int M, int N, int K, int out_dtype,
                                  const void* lora_t, const void* lora_b, int rank,
                                  float lora_scale, void* stream);

/* Barrier of nranks (<= 8) ranks after their peer stores: flags[p] is rank p's
 * flag array (int32 [nranks], this process's mapping of it; zero when
 * allocated), counter a 4-byte device word of this rank (zero at the start,
 * advanced by every call, so the call can sit in a CUDA graph). Rank `rank`
 * writes this call's epoch into slot `rank` of every rank's flags (release,
 * system scope, after a system fence) and waits until every slot of its own
 * flags has reached it. A wait longer than timeout_ns records status 6
 * (ck_convrot_device_status) and returns instead of hanging. Every rank must
 * make the same sequence of calls. */
int ck_peer_barrier(void* const* flags, int nranks, int rank, void* counter, long long timeout_ns, void* stream);

/* Copy columns [offset, offset + width) (bytes) of `rows` rows of pitch
 * pitch_bytes from src to the same place in each of dsts[0 .. ndst) (peer
 * mappings allowed): one 2D copy per destination on `stream`, carried by the
 * copy engines over NVLink, so no SM time is taken from kernels running beside
 * it. The column-split linear sends each rank's block to its peers this way. */
int ck_peer_copy_columns(void* const* dsts, int ndst, const void* src, long long pitch_bytes,
                         long long offset_bytes, long long width_bytes, long long rows, void* stream);

/* Dynamic-LoRA down projection T = fp16(x) . down^T (no HIP export counterpart;
 * replaces the fp16 matmul the node's adapter runs on x, int4_ops.py:181-192,
 * with the adapters in fp16 as int4_ops.py:165-167 prepares them):
 *   x [M, K] in in_dtype (1 = bf16, converted to fp16 element by element with
 *   round to nearest even, as a cast does; 2 = f16), down [R, K] f16,
 *   t [M, R] f16 out; K % 8 == 0, R a multiple of 8 in [8, 64], all 16-byte
 *   aligned. fp32 accumulation on the tensor cores, one rounding to fp16; the
 *   summation order is fixed, so results repeat bit for bit. t is the lora_t
 *   operand of the fused LoRA GEMMs. */
int ck_lora_down(const void* x, int in_dtype, const void* down, void* t, int M, int K, int R, void* stream);

/* The int4 GEMM on int8 activation codes (A8 form; no reference counterpart):
 *   X8 [M, K] int8, one sign-extended code per byte (ck_convrot_quant_int4_unpacked),
 *   Wp [N, K/2] packed int4 weights (the reference codec), both 16-byte aligned;
 *   xscale [M], wscale [N] f32; bias [N] or NULL in bias_dtype (0 f32, 1 bf16, 2 f16);
 *   out [M, N], out_dtype 0 = f32, 1 = bf16, 3 = int32 exact accumulators D
 *   (scales and bias ignored); K % 128 == 0, K <= 65536.
 * Optional Dynamic-LoRA side path as ck_int4_convrot_gemm_lora (lora_t, lora_b
 * fp16 [M, rank] / [N, rank], rank a multiple of 8 in [8, 64]; both NULL: none).
 * The weights stay packed in HBM and are expanded on chip (into tensor memory
 * for grids of 74+ output tiles without LoRA, else in shared memory); the
 * activations go to the tensor cores as loaded. Same D, epilogue and output
 * bits as the packed-code GEMM. */
int ck_int4_convrot_gemm_a8(const void* X8, const void* Wp, const void* xscale, const void* wscale,
                            const void* bias, int bias_dtype, void* out, int M, int N, int K,
                            int out_dtype, const void* lora_t, const void* lora_b, int rank,
                            float lora_scale, void* stream);

/* Unpacked-code path (no reference counterpart). With both operands as one
 * sign-extended int8 per int4 code, sum_k x_k w_k is the int8 tensor-core product
 * over the same K: bit-identical results to the packed path on the faster int8
 * pipeline, at twice the bytes for the operands. */

/* packed [rows, K/2] -> codes [rows, K] int8 (column order kept, nibbles
 * sign-extended); both 16-byte aligned, K % 32 == 0. Run once per weight. */
int ck_int4_unpack(const void* packed, void* codes, long long rows, int K, void* stream);

/* ck_convrot_quant_int4 with unpacked output: codes [M, K] int8, scale [M] f32.
 * bf16 rows of whole 256-column tiles, G in {64, 256}; -1 otherwise. */
int ck_convrot_quant_int4_unpacked(const void* x, int in_dtype, void* qout, void* scaleout,
                                   int M, int K, int G, void* stream);

/* Workspace of ck_convrot_w4a4_linear_unpacked: align256(M * K) + align256(4 * M). */
size_t ck_convrot_w4a4_linear_unpacked_workspace_size(int M, int K);

/* ck_convrot_w4a4_linear with the weight given as unpacked codes Wcodes [N, K]
 * int8 (from ck_int4_unpack): the quantizer writes unpacked activation codes to
 * the workspace and the int8 pair GEMM (double-buffered accumulators) forms the
 * exact products; same epilogue, same results. Same argument rules as
 * ck_convrot_w4a4_linear plus those of ck_convrot_quant_int4_unpacked. */
int ck_convrot_w4a4_linear_unpacked(const void* x, int in_dtype, const void* Wcodes, const void* wscale,
                                    const void* bias, int bias_dtype, void* out, int out_dtype,
                                    int M, int N, int K, int G, void* workspace, size_t workspace_bytes,
                                    void* stream);

/* ---------------------------------------------------------------------------
 * MX4: microscaled 4-bit floats (OCP MXFP4) with the ConvRot rotation. No
 * reference counterpart (the reference's 4-bit format is int4).
 *
 * Values e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6; sign in bit 3) in blocks of 32 along
 * a row, one scale byte E8M0 a block (E stands for 2^(E - 127), 255 for NaN): a
 * block of amplitude a gets E = max(floor(log2 a) - 2 + 127, 0), codes are
 * rounded to nearest even and saturate at 6; a block holding an infinity or a
 * NaN gets 255. Two codes a byte, the even column in the low nibble. Scales of a
 * matrix [R, K] lie in tiles [ceil(R/128), ceil(K/128), 512]: row r and block b
 * at byte (r % 32) * 16 + (r / 32 % 4) * 4 + b % 4 of tile (r / 128, b / 4).
 *
 * dtype codes 0 = f32, 1 = bf16, 2 = f16. G in {0 (not rotated), 16, 64, 256},
 * K a multiple of 32 and of G. The rotation runs in fp32 in the radix-4 steps of
 * the int4 quantizers, without an intermediate rounding; it is its own inverse.
 * -------------------------------------------------------------------------- */

/* Bytes of the scale tiles of a [rows, K] matrix. */
size_t ck_mx4_scales_size(int rows, int K);

/* x [M, K], row stride ldx elements (>= K) -> codes [M, K/2] and scale tiles
 * (both 16-byte aligned; every byte of the tiles is written). */
int ck_mx4_quant(const void* x, int in_dtype, long long ldx, void* codes, void* scales, int M, int K, int G,
                 void* stream);

/* The values codes and scales stand for -> out [M, K] (16-byte aligned), rotated
 * back with G != 0; one rounding. */
int ck_mx4_dequant(const void* codes, const void* scales, void* out, int out_dtype, int M, int K, int G, void* stream);

/* Workspace of ck_mx4_linear: the row codes and their scale tiles (0, none needed,
 * up to 8 rows: one kernel quantizes and multiplies). */
size_t ck_mx4_linear_workspace_size(int M, int K);

/* out[m, n] = sum_k x[m, k] W[n, k] + bias[n]: x [M, K] (row stride ldx) is
 * rotated and quantized into the workspace (256-byte aligned), the weight is
 * given as codes [N, K/2] and scale tiles from ck_mx4_quant with the same G.
 * fp32 accumulation, one rounding. bias [N] or NULL in bias_dtype; out [M, N] in
 * x's dtype, 16-byte aligned. Two calls in flight at once need two workspaces. */
int ck_mx4_linear(const void* x, int dtype, long long ldx, const void* Wcodes, const void* Wscales,
                  const void* bias, int bias_dtype, void* out, int M, int N, int K, int G, void* workspace,
                  size_t workspace_bytes, void* stream);

/* Paged key/value cache: codes [pages, 2, heads, page, d/2], scales [pages, 2,
 * heads, page, d/32] (16-byte aligned), keys at index 0, values at 1, both rotated
 * along d. d in {64, 128, 256}; page a power of two; slot s (int64) is token
 * s % page of page s / page.
 *
 * append: k, v [T, heads, d] with strides in elements (token, head; d
 * contiguous) are rotated, quantized and written to their slots; a slot outside
 * the cache is skipped. Slots of one call must differ. */
int ck_mx4_cache_append(void* codes, void* scales, long long pages, int heads, int d, int page, int G,
                        const void* k, const void* v, int in_dtype, long long k_token, long long k_head,
                        long long v_token, long long v_head, const void* slots, int T, void* stream);

/* read: the slots' keys and values, rotated back, -> k, v [T, heads, d] (16-byte
 * aligned); a slot outside the cache reads as zeros. */
int ck_mx4_cache_read(const void* codes, const void* scales, long long pages, int heads, int d, int page, int G,
                      const void* slots, int T, void* k, void* v, int out_dtype, void* stream);

/* Workspace of ck_mx4_attention for `longest` = table_pages * page (0: none needed). */
size_t ck_mx4_attention_workspace_size(int B, int tq, int hq, int hkv, int d, long long longest);

/* Causal attention of the newest tq tokens of B sequences over the cache.
 *   q [B, tq, hq, d] (dtype 1 or 2; strides in elements, d contiguous), hq a
 *   multiple of hkv (query head h reads cache head h / (hq / hkv));
 *   table int32 [B, table_pages] (row stride table_ld): token j of sequence b is
 *   token j % page of page table[b][j / page]; a page outside [0, pages) hides
 *   its tokens; lens int32 [B] tokens in the cache (cut at table_pages * page,
 *   which may be 2^31 - 1024 at most);
 *   query t sees tokens up to position lens[b] - tq + t; one that sees none
 *   gives zeros; out [B, tq, hq, d] (16-byte aligned) in dtype. */
int ck_mx4_attention(const void* q, int dtype, long long q_seq, long long q_token, long long q_head,
                     const void* codes, const void* scales, long long pages, int page, const void* table,
                     long long table_ld, int table_pages, const void* lens, void* out, int B, int tq, int hq,
                     int hkv, int d, int G, float softmax_scale, void* workspace, size_t workspace_bytes,
                     void* stream);

/* Rotary positions. x [B, T, H, D] (dtype, strides in elements, D contiguous and even) -> out [B, T,
 * H, D] without gaps: pair i of a head, channels (2i, 2i + 1) where `interleaved`, else (i, i + P), is
 * turned by the angle p freqs[i], p the token's position on the axis whose section holds i; the channels
 * behind the 2P first are copied. positions [B, T, axes] by strides (pos_type 0 int32, 1 int64, 2 f32),
 * freqs [P] f64 radians a position, both on the device; sections [axes] (host): pairs of each axis, P in
 * all, 1 to 8 axes. inverse != 0 turns back. Angles are taken in 64 bits, one rounding. */
int ck_rope(const void* x, int dtype, long long x_batch, long long x_token, long long x_head, void* out,
            int B, int T, int H, int D, const void* positions, int pos_type, long long p_batch,
            long long p_token, long long p_axis, const void* freqs, const int* sections, int axes,
            int interleaved, int inverse, void* stream);

/* ck_mx4_cache_append with positions (as ck_rope, [T, axes]): keys are turned before they are rotated
 * and quantized, without a rounding between; values as in ck_mx4_cache_append. q [T, q_heads, d] turned
 * -> q_out [T, q_heads, d] in the same dtype (q_heads 0: none, q and q_out may be NULL). Tokens whose slot
 * lies outside the cache write no key and no value; their queries are turned. Slots of one call must
 * differ. */
int ck_mx4_cache_append_rope(void* codes, void* scales, long long pages, int heads, int d, int page, int G,
                             const void* q, const void* k, const void* v, int dtype, int q_heads,
                             long long q_token, long long q_head, long long k_token, long long k_head,
                             long long v_token, long long v_head, void* q_out, const void* slots, int T,
                             const void* positions, int pos_type, long long p_token, long long p_axis,
                             const void* freqs, const int* sections, int axes, int interleaved, void* stream);

/* Workspace of ck_mx4_tree_attention for `longest` = table_pages * page (0: none needed). */
size_t ck_mx4_tree_attention_workspace_size(int B, int tq, int hq, int hkv, int d, long long longest);

/* ck_mx4_attention for drafted tokens that form a tree: sequence b's nodes are its nodes[b] newest tokens
 * (int32 [B], cut to 0 .. tq; NULL: tq each). Node t sees the tokens before the nodes and those nodes j
 * whose byte mask[b * mask_seq + t * mask_row + j] is not zero (itself only if named); one that sees none
 * gives zeros, and so do the rows behind a sequence's nodes. mask_seq 0: one mask for all sequences. */
int ck_mx4_tree_attention(const void* q, int dtype, long long q_seq, long long q_token, long long q_head,
                          const void* codes, const void* scales, long long pages, int page, const void* table,
                          long long table_ld, int table_pages, const void* lens, const void* nodes,
                          const void* mask, long long mask_seq, long long mask_row, void* out, int B, int tq,
                          int hq, int hkv, int d, int G, float softmax_scale, void* workspace,
                          size_t workspace_bytes, void* stream);

/* Workspace of ck_convrot_w8a8_linear_rmsnorm: the int8 codes and the row scales. */
size_t ck_convrot_w8a8_linear_rmsnorm_workspace_size(int M, int K);

/* The W8A8 linear behind a root-mean-square norm: hidden = x + residual (rounded to dtype; residual NULL:
 * hidden is not written), y = R(h / sqrt(mean h^2 + eps) * norm_weight), xs = max(max |y|, 1e-10) / 127,
 * codes = y / xs to nearest even, out = ((float(D) * xs[m]) * wscale[n]) + bias[n] with the exact product
 * D. fp32 throughout, h unrounded; a row with an infinity or a NaN gives NaN, finite rows of any
 * magnitude are normalised. hidden must not overlap x or residual.
 *   x, residual [M, K] (row strides ldx, ldr >= K), hidden [M, K] (16-byte aligned) in dtype;
 *   norm_weight [K] in norm_dtype or NULL (ones); W [N, K] int8 and out [M, N] 16-byte aligned, wscale [N]
 *   f32, bias [N] in bias_dtype or NULL; out_dtype 0 f32, 1 bf16; G in {16, 64, 256}, K a multiple of G and
 *   at most 16384; workspace 256-byte aligned. */
int ck_convrot_w8a8_linear_rmsnorm(const void* x, const void* residual, int dtype, long long ldx, long long ldr,
                                   const void* norm_weight, int norm_dtype, float eps, const void* W,
                                   const void* wscale, const void* bias, int bias_dtype, void* hidden, void* out,
                                   int out_dtype, int M, int N, int K, int G, void* workspace,
                                   size_t workspace_bytes, void* stream);

/* Reads and clears the device status word that kernels set when a bounded
 * wait gives up (0 = ok). Synchronises `stream`. No reference counterpart:
 * the reference has no device-side timeouts. */
int ck_convrot_device_status(void* stream, int* status);

/* Failure-path self test: launches one thread that waits on an mbarrier nothing
 * arrives on, with the bounded wait every pipeline wait uses, cut to limit_ns
 * (0 < limit_ns <= 1e8). It gives up, records status 5 (read and cleared by
 * ck_convrot_device_status) and returns, leaving the context usable. No
 * reference counterpart: it exercises the timeout path without faulting a GPU. */
int ck_convrot_selftest_wait_timeout(long long limit_ns, void* stream);

/* Human-readable reason for the last -1 returned on this host thread. */
const char* ck_convrot_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* CONVROT_B200_H */
