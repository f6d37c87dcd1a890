/*
 * muon_sr_amd.h -- C ABI of libmuon_sr_amd.so, the MI355X (gfx950) kernels of
 * the muon_sr optimizer-step hot path.
 *
 * Conventions (every entry point):
 *  - All pointers are device pointers unless documented as host arrays; the
 *    library never allocates or frees device memory (workspace comes from the
 *    caller, sized by the matching *_workspace_bytes query).
 *  - bf16 tensors are passed as uint16_t bit patterns, contiguous.
 *  - Work is enqueued asynchronously on `stream` (a hipStream_t; NULL = the
 *    default stream).  Nothing synchronises.
 *  - Return 0 on success, else a hipError_t or one of the MSR_ERR_* codes
 *    below; msr_last_error() returns a message for the calling thread.
 *  - fp32 scalars are the reference's Python floats rounded to fp32, as a
 *    compiled Triton launch passes them.  Seeds are the reference's 32-bit
 *    seeds; the library derives each stream's Philox key (SEED + k typing).
 *  - noise_mode selects the stochastic-rounding noise source:
 *      MSR_NOISE_TRITON  word 0 of Philox4x32-10 at counter (offset, 0, 0, 0):
 *                        the same bits the reference's tl.randint produces;
 *      MSR_NOISE_PHILOX8 one Philox4x32-10 call per 8 consecutive offsets
 *                        (16 bits each): this library's fast stream;
 *      MSR_NOISE_INJECT  noise read from `inject` (uint16 [streams][n]); tests.
 *  - Entry points keep no global mutable state and are safe to call from
 *    several host threads (autograd hooks run on the engine thread).
 */
#ifndef MUON_SR_AMD_H
#define MUON_SR_AMD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ihipStream_t *msr_stream_t; /* == hipStream_t */

#define MSR_NOISE_TRITON 0
#define MSR_NOISE_PHILOX8 1
#define MSR_NOISE_INJECT 2

#define MSR_ERR_ARG 1001
#define MSR_ERR_ALIGN 1002
#define MSR_ERR_LAUNCH 1003
#define MSR_ERR_WORKSPACE 1004
#define MSR_ERR_OVERLAP 1005   /* operands overlap without being the same buffer (a data race) */

/* Library version (major*10000 + minor*100 + patch) and error text. */
int msr_version(void);
const char *msr_last_error(void);

/* ---------------------------------------------------------------------------
 * (c) SR gradient accumulation.
 * Replaces the _grad_accum_kernel launches of TritonSRAccumulator._accum_hook
 * (muon_sr/triton_adamw.py:206-229, launched at :260 and :264).
 *   acc[i] <- SR_bf16(f32(acc[i]) + f32(grad[i])),  noise offset i.
 * grad_is_f32: 0 = bf16 grad, 1 = fp32 grad.
 * zero_init != 0 treats acc as zero on input (fuses the zeros_like at :263);
 * acc is then write-only.  inject: uint16 [n].
 * ------------------------------------------------------------------------- */
int msr_sr_accum(uint16_t *acc, const void *grad, int32_t grad_is_f32, int64_t n, uint32_t seed,
                 int32_t zero_init, int32_t noise_mode, const uint16_t *inject, msr_stream_t stream);

/* (c) SR accumulation fused with the weight-gradient GEMM of a linear layer
 * y = x W^T: the bf16 weight gradient dW = dy^T x that autograd hands the
 * accumulation hook (muon_sr/triton_adamw.py:252-265) is accumulated into acc
 * as the hook's _grad_accum_kernel (:206-229) does, without being written:
 *   acc[o][i] <- SR_bf16( f32(acc[o][i]) + f32(RNE_bf16( sum_t dy[t][o] x[t][i] )) )
 * (fp32 products accumulated in fp32; noise of element offset o * in + i, as
 * msr_sr_accum on the contiguous [out][in] buffer).  No counterpart in the
 * reference, which runs the GEMM and the accumulation separately.
 * x: bf16 [tokens][in] (row stride ldx), dy: bf16 [tokens][out] (ldy), acc:
 * bf16 [out][in] contiguous; in and out multiples of 256, tokens a multiple of
 * 128 (else MSR_ERR_ARG: use the GEMM and msr_sr_accum).  zero_init, seed,
 * noise_mode and inject as msr_sr_accum. */
int msr_linear_wgrad_sr_accum(uint16_t *acc, const uint16_t *x, int64_t ldx, const uint16_t *dy, int64_t ldy,
                              int64_t tokens, int64_t in_features, int64_t out_features, uint32_t seed,
                              int32_t zero_init, int32_t noise_mode, const uint16_t *inject, msr_stream_t stream);

/* (c) SR gradient accumulation of many tensors in one launch.
 * Same arithmetic and noise as one msr_sr_accum call per item (noise offsets
 * restart at 0 in every tensor), for the hooks of one backward pass collected
 * by TritonSRAccumulator (muon_sr/triton_adamw.py:252-265, one launch per
 * parameter in the reference).  items: HOST array; any count (split into
 * launches internally).  noise_mode: MSR_NOISE_TRITON or MSR_NOISE_PHILOX8. */
typedef struct msr_accum_item {
    uint16_t *acc;      /* bf16 accumulator [n] */
    const void *grad;   /* bf16, or fp32 with MSR_ACCUM_GRAD_F32, [n] */
    int64_t n;
    uint32_t seed;
    int32_t flags;      /* MSR_ACCUM_ZERO_INIT | MSR_ACCUM_GRAD_F32 */
} msr_accum_item;
#define MSR_ACCUM_ZERO_INIT 1
#define MSR_ACCUM_GRAD_F32 2
int msr_sr_accum_multi(const msr_accum_item *items, int32_t count, int32_t noise_mode, msr_stream_t stream);

/* ---------------------------------------------------------------------------
 * BF16-moment AdamW step (PyTorch order: decay before the update).
 * Replaces _adamw_kernel / _adamw_step (muon_sr/triton_adamw.py:9-114).
 * Streams: ema uses SEED, ema_sq SEED+1, p SEED+2 (inject: uint16 [3][n]).
 * ------------------------------------------------------------------------- */
int msr_adamw_bf16_step(uint16_t *p, const uint16_t *g, uint16_t *ema, uint16_t *ema_sq, int64_t n,
                        float lr, float beta1, float beta2, float eps, float weight_decay,
                        float bias_correction, float bias_correction_sqrt, uint32_t seed,
                        int32_t noise_mode, const uint16_t *inject, msr_stream_t stream);

/* The same for many tensors of one parameter group in one launch (up to 56 per launch, split
 * internally); equal, bit for bit, to one call per item in order.  form MSR_ADAMW: each item as
 * msr_adamw_bf16_step (m, v: ema, ema_sq; bc1, bc2: bias_correction, bias_correction_sqrt).
 * form MSR_ADAMW_8BIT16: each item as msr_adamw8bit_step with quantized = 0 (m, v: the bf16
 * states; bc1, bc2 as there).  form MSR_ADAMW_CENTRALIZED: as MSR_ADAMW on the gradient that
 * msr_centralize_bf16(rows of item.cols elements, strength) gives, without writing it; tensors
 * 16-byte aligned, cols a multiple of 8 and at most MSR_ADAMW_CENTRAL_MAX_COLS (else
 * MSR_ERR_ARG: centralize first).  strength is unused in the other forms.  items: HOST array.
 * A list with an item that is refused is refused whole, before anything is launched.
 * noise_mode: MSR_NOISE_TRITON or MSR_NOISE_PHILOX8. */
typedef struct msr_adamw_item {
    uint16_t *p;
    const uint16_t *g;
    uint16_t *m, *v;
    int64_t n;
    float bc1, bc2;
    uint32_t seed;
    int32_t cols;       /* MSR_ADAMW_CENTRALIZED: elements of a row; else unused */
} msr_adamw_item;
#define MSR_ADAMW 0
#define MSR_ADAMW_8BIT16 1
#define MSR_ADAMW_CENTRALIZED 2
#define MSR_ADAMW_CENTRAL_MAX_COLS 4096
int msr_adamw_multi(const msr_adamw_item *items, int32_t count, int32_t form, float strength, float lr,
                    float beta1, float beta2, float eps, float weight_decay, int32_t noise_mode,
                    msr_stream_t stream);

/* ---------------------------------------------------------------------------
 * Gradient centralization of TritonAdamW, on the device.
 * Replaces the host-issued torch ops of muon_sr/triton_adamw.py:179-187
 * (g.to(fp32); g -= g.mean(dims 1..) * c; g.to(bf16)).  g, out: bf16
 * [rows][cols] (rows = dim 0 of a tensor of 2+ dims, else 1); out[r][j] =
 * bf16_rne(g[r][j] - (sum_j g[r][j] / cols) * alpha) with fp32 sums in a fixed
 * order.  workspace: msr_centralize_workspace_bytes(rows, cols) bytes of
 * device memory (the library does not allocate).  out may equal g.
 * ------------------------------------------------------------------------- */
int msr_centralize_workspace_bytes(int64_t rows, int64_t cols, size_t *bytes);
int msr_centralize_bf16(const uint16_t *g, uint16_t *out, int64_t rows, int64_t cols, float alpha,
                        void *workspace, size_t workspace_bytes, msr_stream_t stream);

/* msr_centralize_bf16 without a workspace argument and without allocating.
 * No counterpart in the reference: for callers that cannot allocate device
 * memory (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc).  The workspace is a static device array of
 * MSR_CENTRALIZE_NOALLOC_SCRATCH_BYTES in the library, one per GPU, held until
 * the process ends; its address is looked up on the first call for a device
 * (the device of `stream`, or the current device for the null stream).  Sizes
 * whose msr_centralize_workspace_bytes exceed it return MSR_ERR_WORKSPACE
 * (4 MiB covers about 500,000 rows of up to 16384 columns, e.g. a 128256 x 4096
 * embedding).  Same results as msr_centralize_bf16, bit for bit.  Calls that
 * overlap in time on one GPU share the array and race: serialise them (one
 * stream, or events). */
#define MSR_CENTRALIZE_NOALLOC_SCRATCH_BYTES (4 << 20)
int msr_centralize_bf16_noalloc(const uint16_t *g, uint16_t *out, int64_t rows, int64_t cols, float alpha,
                                msr_stream_t stream);

/* ---------------------------------------------------------------------------
 * (a) 8-bit blockwise AdamW step (bitsandbytes order: decay after the update).
 * Replaces the _adamw_8bit_kernel launch of TritonAdamW8bit.step
 * (muon_sr/triton_adamw_8bit.py:56-99, launched at :198-204).
 * quantized != 0: state1/state2 are uint8 codes [n], absmax1/absmax2 fp32
 *   [ceil(n/block)], qmap1 (signed) / qmap2 (unsigned) fp32 [256].
 *   qtable: NULL, or a device copy of msr_quant_table_build(qmap1, qmap2)
 *   (16-byte aligned) -- the same codes from a bucketed threshold table.
 *   With block 256, a qtable and 16-byte aligned p/g (8-byte aligned codes),
 *   whole pairs of blocks run through a fast kernel (correctly rounded sqrt and
 *   quotients from fp32 sequences valid on checked ranges, exact fallback
 *   per wave outside them) and the rest through the general kernel; both give
 *   the reference's bits.
 * quantized == 0: state1/state2 are bf16 moments [n]; absmax/qmap unused.
 * block: power of two in [32, 4096].  bc1 = 1-b1^step, bc2 = 1-b2^step.
 * Streams: p uses SEED, bf16 m SEED+1, bf16 v SEED+2 (inject: uint16 [3][n]).
 * ------------------------------------------------------------------------- */
int msr_adamw8bit_step(uint16_t *p, const uint16_t *g, void *state1, void *state2,
                       float *absmax1, float *absmax2, const float *qmap1, const float *qmap2,
                       const void *qtable, int64_t n, int32_t block, int32_t quantized,
                       float lr, float beta1, float beta2, float eps, float weight_decay,
                       float bc1, float bc2, uint32_t seed,
                       int32_t noise_mode, const uint16_t *inject, msr_stream_t stream);

/* The quantized step for many tensors of one parameter group in one launch (up to 56 per
 * launch, split internally): equal, bit for bit, to one msr_adamw8bit_step(quantized = 1) per
 * item in order, with the same codebooks, block, hyperparameters and bias corrections.  Tensors
 * that the fast kernel does not take (other codebooks, blocks outside 64-512, unaligned
 * operands) run one launch each.  items: HOST array.  A list with an item that is refused is
 * refused whole, before anything is launched.  noise_mode: MSR_NOISE_TRITON or MSR_NOISE_PHILOX8. */
typedef struct msr_adam8_item {
    uint16_t *p;
    const uint16_t *g;
    uint8_t *state1, *state2;       /* codes [n] */
    float *absmax1, *absmax2;       /* block scales [ceil(n/block)] */
    int64_t n;
    uint32_t seed;
    int32_t reserved;               /* 0 */
} msr_adam8_item;
int msr_adamw8bit_multi(const msr_adam8_item *items, int32_t count, const float *qmap1, const float *qmap2,
                        const void *qtable, int32_t block, float lr, float beta1, float beta2, float eps,
                        float weight_decay, float bc1, float bc2, int32_t noise_mode, msr_stream_t stream);

/* Host only: *apart is 1 if every item of the two lists would be accepted and no memory that a step of
 * one list writes is touched by a step of the other, so that the lists may be launched one after the other
 * whatever the order of their steps in the group; else 0.  block: the quantized list's. */
int msr_adamw8bit_apart(const msr_adam8_item *quantized, int32_t n_quantized, int32_t block,
                        const msr_adamw_item *bf16, int32_t n_bf16, int32_t *apart);

/* ---------------------------------------------------------------------------
 * (b) Muon momentum prologue over one shape group.
 * Replaces the grad->stack copy and the _muon_prepare_kernel launch of
 * _triton_muon_batch_step (muon_sr/triton_muon_sr.py:150-159) and, with
 * count == 1, _run_prepare (:88-98).
 *   grads: HOST array of `count` device pointers, each to numel_each bf16
 *          (grad_is_f32 == 0) or fp32 (grad_is_f32 != 0: read as fp32, as the
 *          reference's kernel reads an fp32 gradient on the per-parameter path,
 *          :34; its batched path copies gradients into a bf16 stack first).
 *   buf:   bf16 momentum stack [count][numel_each], updated in place (SR).
 *   out:   bf16 pre-NS update [count][numel_each] (RNE).
 * Noise offset of element j of matrix i: i*numel_each + j (stack offset).
 * inject: uint16 [count*numel_each].
 * ------------------------------------------------------------------------- */
int msr_muon_prepare(const void *const *grads, int32_t grad_is_f32, uint16_t *buf, uint16_t *out,
                     int64_t numel_each, int32_t count, float beta, int32_t nesterov,
                     uint32_t seed, int32_t noise_mode, const uint16_t *inject, msr_stream_t stream);

/* ---------------------------------------------------------------------------
 * (b) Muon parameter update over several matrices of one shape.
 * Replaces the per-parameter _muon_apply_kernel launches of
 * _triton_muon_batch_step and _run_apply (muon_sr/triton_muon_sr.py:53-80,
 * 105-113, 167-169).
 *   params: HOST array of `count` device pointers, each to numel_each bf16.
 *   upd:    bf16 Newton-Schulz output [count][numel_each] (parameter layout).
 *   seeds:  HOST array of `count` seeds (salt-1 deterministic seeds).
 *   p <- SR(p*(1-lr*wd) - lr*(f32(upd)*scale)), noise offset j within p.
 * inject: uint16 [count][numel_each].
 * ------------------------------------------------------------------------- */
int msr_muon_apply(uint16_t *const *params, const uint16_t *upd, int64_t numel_each, int32_t count,
                   float lr, float weight_decay, float scale, const uint32_t *seeds,
                   int32_t noise_mode, const uint16_t *inject, msr_stream_t stream);

/* ---------------------------------------------------------------------------
 * (b) Batched Newton-Schulz orthogonalisation on bf16 MFMA.
 * Replaces _newton_schulz(G, steps, out_dtype=None) (muon_sr/muon_sr.py:82-98)
 * for a contiguous bf16 stack G [batch][rows][cols]; out has the same shape.
 * The iteration runs on the wide orientation (transposed when rows > cols):
 *   X = G/(||G||_F + 1e-7);  repeat: A = X X^T; B = b A + c A A; X = a X + B X,
 * evaluated as B' = c A A + b A + a I, X = B' X: products accumulate in fp32,
 * A, B' and X are stored in bf16 between GEMMs.  The normalised input is not
 * rounded (G itself, or G scaled by a power of two when ||G||_F is below 2^-17
 * or at least 2^16, is the first iterate, and 1/(||G||_F + 1e-7) goes into the
 * first products' scale factors), and the bf16 rounding residuals of the
 * diagonals of A and B' are carried in fp32 into the next product.  Within
 * 1e-2 relative Frobenius of the exact iteration on Gaussian inputs.
 * steps == 0 returns the reference's bf16 normalisation bf16(G / bf16(bf16(
 * ||G||_F) + 1e-7)).
 * Results do not depend on `batch` (each matrix is computed independently).
 * The workspace holds the iterates and the products' tile counters: calls that
 * may run at the same time (other streams) need workspaces of their own.
 * ------------------------------------------------------------------------- */
int msr_ns_workspace_bytes(int64_t batch, int64_t rows, int64_t cols, size_t *bytes);
int msr_newton_schulz(const uint16_t *in, uint16_t *out, int64_t batch, int64_t rows, int64_t cols,
                      int32_t steps, float a, float b, float c, void *workspace, size_t workspace_bytes,
                      msr_stream_t stream);

/* ---------------------------------------------------------------------------
 * (b) Newton-Schulz and the Muon parameter update in one pass.
 * Replaces the _newton_schulz call and the _run_apply launches of one chunk of
 * _triton_muon_batch_step (muon_sr/triton_muon_sr.py:160-169), and of
 * _triton_muon_step (:116-120) with batch == 1.  Equal, bit for bit, to
 * msr_newton_schulz(upd -> X) followed by msr_muon_apply(params, X, ...), but
 * the last product's store applies the update to the parameters directly: X is
 * never written and the apply pass does not run.
 *   upd:    bf16 pre-NS update stack [batch][rows][cols] (read only)
 *   params: HOST array of `batch` device pointers, each to rows*cols bf16
 *   seeds:  HOST array of `batch` seeds (salt-1 deterministic seeds)
 *   p <- SR(p*(1-lr*wd) - lr*(f32(bf16(X))*scale)), noise offset = element index in p.
 * steps >= 1; workspace as msr_ns_workspace_bytes(batch, rows, cols).
 * inject: uint16 [batch][rows*cols].
 * ------------------------------------------------------------------------- */
int msr_muon_ns_apply(const uint16_t *upd, uint16_t *const *params, const uint32_t *seeds, int64_t batch,
                      int64_t rows, int64_t cols, int32_t steps, float a, float b, float c, float lr,
                      float weight_decay, float scale, int32_t noise_mode, const uint16_t *inject,
                      void *workspace, size_t workspace_bytes, msr_stream_t stream);

/* ---------------------------------------------------------------------------
 * (b) The whole Muon step of one chunk: momentum prologue, Newton-Schulz and
 * the parameter update.  Replaces, for one NS chunk of a shape group, the
 * grad->stack copy and _muon_prepare_kernel (muon_sr/triton_muon_sr.py:18-50,
 * 150-159), _newton_schulz (muon_sr/muon_sr.py:82-98) and the _run_apply
 * launches (triton_muon_sr.py:53-80, 160-169); with batch == 1, first == 0,
 * _triton_muon_step (:88-120).  Equal, bit for bit, to msr_muon_prepare over the
 * chunk's rows of the stack, then msr_newton_schulz, then msr_muon_apply (or,
 * with out, without the apply), but the update is made inside the
 * Newton-Schulz prologue, which writes it straight into the first iterate
 * (with its sum of squares): the update stack is never written or read.
 *   grads:  HOST array of `batch` device pointers (bf16, or fp32 with grads_f32)
 *   buf:    bf16 momentum of the chunk's first matrix, [batch][rows][cols],
 *           updated in place (SR); `first` = that matrix's index in its stack:
 *           noise offset of element j of matrix i = (first + i)*rows*cols + j
 *   params/apply_seeds: HOST arrays of `batch` (as msr_muon_ns_apply), or
 *   params == NULL and out: bf16 [batch][rows][cols] receives the NS output.
 * steps >= 1; workspace as msr_ns_workspace_bytes(batch, rows, cols).
 * inject_prepare: uint16 indexed by the stack offset above; inject_apply as
 * msr_muon_ns_apply's.
 * ------------------------------------------------------------------------- */
int msr_muon_fused_step(const void *const *grads, int32_t grads_f32, uint16_t *buf, int64_t first, int64_t batch,
                        int64_t rows, int64_t cols, float beta, int32_t nesterov, uint32_t prepare_seed,
                        int32_t steps, float a, float b, float c, uint16_t *out, uint16_t *const *params,
                        const uint32_t *apply_seeds, float lr, float weight_decay, float scale,
                        int32_t noise_mode, const uint16_t *inject_prepare, const uint16_t *inject_apply,
                        void *workspace, size_t workspace_bytes, msr_stream_t stream);

/* ---------------------------------------------------------------------------
 * (b) The whole Muon step of several shape groups in one call: one
 * msr_muon_fused_step per group, with the groups' matrices sharing each
 * Newton-Schulz product launch.  Replaces, for shape groups whose shapes are
 * transposes of each other (a model's tall and wide projections), the
 * per-group loop of muon_sr/triton_muon_sr.py:128-177 (group order does not
 * matter: groups touch disjoint memory).  Equal, bit for bit, to
 * msr_muon_fused_step called once per group with the same arguments (params,
 * apply_seeds and a group's prepare_seed as there); a shared launch only fills
 * the GPU's last round of tiles better than separate ones.
 *   groups: HOST array of n_groups; every group's shape is rows x cols or
 *           cols x rows of group 0's; pointers as in msr_muon_fused_step
 *           (grads, params, apply_seeds: HOST arrays of `batch` entries).
 * noise_mode: MSR_NOISE_TRITON or MSR_NOISE_PHILOX8.  steps >= 1; workspace as
 * msr_ns_workspace_bytes(sum of the groups' batch, rows, cols) of group 0.
 * ------------------------------------------------------------------------- */
typedef struct msr_muon_group {
    const void *const *grads;      /* bf16, or fp32 with grads_f32 */
    uint16_t *buf;                 /* momentum of the group's first matrix, [batch][rows][cols] */
    uint16_t *const *params;
    const uint32_t *apply_seeds;
    int64_t first;                 /* index of buf's first matrix in its stack (noise offsets) */
    int64_t batch, rows, cols;
    uint32_t prepare_seed;
    int32_t grads_f32;
    float scale;                   /* the group's sqrt(max(1, rows/cols)) */
} msr_muon_group;
int msr_muon_fused_steps(const msr_muon_group *groups, int32_t n_groups, float beta, int32_t nesterov,
                         int32_t steps, float a, float b, float c, float lr, float weight_decay,
                         int32_t noise_mode, void *workspace, size_t workspace_bytes, msr_stream_t stream);

/* ---------------------------------------------------------------------------
 * (b) The whole Muon step of matrices that are parameters of their own (momenta not stacked, a
 * prepare seed each): one msr_muon_fused_step with batch 1, first 0 per matrix, as
 * TritonMuonSR's per-parameter steps make it (_triton_muon_step, muon_sr/triton_muon_sr.py:88-120),
 * with matrices of one Newton-Schulz shape sharing product launches.  Equal, bit for bit, to
 * those calls in order; matrices that share memory which one of them writes run one by one.
 * A list with a matrix that is refused, or too large for the workspace, is refused whole, before
 * anything is launched.
 * matrices: HOST array, any shapes.  The workspace is what msr_muon_each_workspace_bytes gives
 * for the same list: the largest of the shared launches', bounded by them at 2^27 elements, each
 * matrix padded to multiples of 256 (or by one larger matrix): about 1 GiB.
 * ------------------------------------------------------------------------- */
typedef struct msr_muon_matrix {
    const void *grad;              /* bf16, or fp32 with grad_f32 */
    uint16_t *buf, *param;         /* momentum and parameter, [rows][cols] */
    int64_t rows, cols;
    uint32_t prepare_seed, apply_seed;
    int32_t grad_f32;
    float scale;                   /* sqrt(max(1, rows/cols)) */
} msr_muon_matrix;
int msr_muon_each_workspace_bytes(const msr_muon_matrix *matrices, int32_t count, size_t *bytes);
int msr_muon_each(const msr_muon_matrix *matrices, int32_t count, float beta, int32_t nesterov, int32_t steps,
                  float a, float b, float c, float lr, float weight_decay, int32_t noise_mode, void *workspace,
                  size_t workspace_bytes, msr_stream_t stream);

/* ---------------------------------------------------------------------------
 * The global norm of many gradients, and clipping by it.  No counterpart in the
 * reference (a training loop calls torch.nn.utils.clip_grad_norm_ between
 * backward and step).
 *   N = (sum over every element of every item of |g|^p)^(1/p), p = 1, 2, or inf
 *   c = min(1, max_norm / (N + 1e-6))       (fp32; NaN where N is NaN)
 *   out[i] = round(f32(g[i]) * c)           (nearest even for a bf16 out)
 * Sums are held in 64 bits, in a fixed order: squares of bf16 and fp32 values
 * neither overflow nor vanish, and a list gives the same bits every time.
 * items: HOST array, any count (empty tensors allowed).  out may be the item's
 * own grad (same type; not written where c is 1); any other sharing of memory
 * that is written is refused (MSR_ERR_OVERLAP).  norm_out: device fp32, the
 * unclipped N.  workspace: msr_grad_norm_workspace_bytes of the same list,
 * 8-byte aligned.  msr_grad_norm ignores out.
 * ------------------------------------------------------------------------- */
typedef struct msr_clip_item {
    const void *grad;   /* bf16, or fp32 with MSR_CLIP_GRAD_F32, [n] */
    void *out;          /* bf16, or fp32 with MSR_CLIP_OUT_F32 (fp32 grads only), [n] */
    int64_t n;
    int32_t flags;
    int32_t reserved;   /* 0 */
} msr_clip_item;
#define MSR_CLIP_GRAD_F32 1
#define MSR_CLIP_OUT_F32 2
#define MSR_NORM_1 1
#define MSR_NORM_2 2
#define MSR_NORM_INF 3
int msr_grad_norm_workspace_bytes(const msr_clip_item *items, int32_t count, size_t *bytes);
int msr_grad_norm(const msr_clip_item *items, int32_t count, int32_t norm, float *norm_out, void *workspace,
                  size_t workspace_bytes, msr_stream_t stream);
int msr_clip_grads(const msr_clip_item *items, int32_t count, int32_t norm, float max_norm, float *norm_out,
                   void *workspace, size_t workspace_bytes, msr_stream_t stream);

/* ---------------------------------------------------------------------------
 * Tokens sorted by expert and back, for mixture-of-experts layers.  No
 * counterpart in the reference.
 *
 * msr_order_tokens: a stable counting sort of the tokens * k slots (t, j) by
 * their expert ids[t][j] (int32, or int64 with ids_i64).  An id outside
 * [0, experts) has no expert: the slot is dropped.
 *   offsets  int32 [experts + 1]: expert e has the rows [offsets[e], offsets[e + 1])
 *   position int32 [tokens][k]: the row of a slot, -1 for a dropped one
 *   source   int32 [tokens * k]: the slot t * k + j of a row, -1 from row offsets[experts] on
 * tokens * k < 2^30, experts <= MSR_EXPERTS_MAX.  workspace:
 * msr_order_workspace_bytes, 4-byte aligned (may be NULL where that is 0).
 *
 * The four passes between tokens and rows, for elem = MSR_BF16 or MSR_F32
 * activations of width d and n = tokens * k rows (a position outside [0, n) is
 * taken as dropped; sums in fp32, one rounding to the stored type):
 *   msr_dispatch        rows[position[t][j]] = x[t]; rows without a slot are 0
 *   msr_dispatch_grad   dx[t] = sum_j drows[position[t][j]]
 *   msr_combine         y[t] = sum_j w[t][j] rows[position[t][j]]
 *   msr_combine_grad    drows[position[t][j]] = w[t][j] dy[t], 0 for rows without a slot;
 *                       dw[t][j] = <dy[t], rows[position[t][j]]>, 0 for dropped slots
 * offsets: as msr_order_tokens wrote it; `experts` is its index of the first row
 * without a slot.  x, dy: rows of ldx / lddy elements; every other tensor is
 * contiguous.  w and dw: welem.  drows or dw may be NULL (not wanted).
 * Outputs must not overlap inputs.
 * ------------------------------------------------------------------------- */
#define MSR_BF16 0
#define MSR_F32 1
#define MSR_EXPERTS_MAX 1024
int msr_order_workspace_bytes(int64_t tokens, int32_t k, int32_t experts, size_t *bytes);
int msr_order_tokens(const void *ids, int32_t ids_i64, int64_t tokens, int32_t k, int32_t experts, int32_t *offsets,
                     int32_t *position, int32_t *source, void *workspace, size_t workspace_bytes, msr_stream_t stream);
int msr_dispatch(const void *x, int64_t ldx, void *rows, const int32_t *position, const int32_t *offsets,
                 int32_t experts, int64_t tokens, int32_t k, int64_t d, int32_t elem, msr_stream_t stream);
int msr_dispatch_grad(const void *drows, void *dx, const int32_t *position, int64_t tokens, int32_t k, int64_t d,
                      int32_t elem, msr_stream_t stream);
int msr_combine(const void *rows, const void *w, void *y, const int32_t *position, int64_t tokens, int32_t k, int64_t d,
                int32_t elem, int32_t welem, msr_stream_t stream);
int msr_combine_grad(const void *dy, int64_t lddy, const void *rows, const void *w, void *drows, void *dw,
                     const int32_t *position, const int32_t *offsets, int32_t experts, int64_t tokens, int32_t k,
                     int64_t d, int32_t elem, int32_t welem, msr_stream_t stream);

/* ---------------------------------------------------------------------------
 * The experts' products over rows sorted by expert (offsets: device int32
 * [experts + 1], offsets[0] = 0, non-decreasing, as msr_order_tokens writes it;
 * read on the GPU only, and clamped to [0, rows]).  No counterpart in the
 * reference.  bf16 operands, fp32 accumulation, one rounding (the order of the sums, and so their last bits, may
 * depend on the sizes of the call; the same call gives the same bits):
 *   msr_experts_forward          y[r] = W[e] x[r]            for the rows r of expert e
 *   msr_experts_dgrad            dx[r] = W[e]^T dy[r]
 *   msr_experts_wgrad            dw[e] = sum_r dy[r] x[r]^T  (0 for an expert without rows)
 *   msr_experts_wgrad_sr_accum   acc[e] <- SR(acc[e] + f32(bf16(dw[e]))): the arithmetic and noise
 *                                of msr_sr_accum on the contiguous [experts][out][in] buffer, as
 *                                msr_linear_wgrad_sr_accum does for one weight
 * Rows from offsets[experts] on have no expert: their y and dx are 0, and dw does
 * not see them.  x, dx: [rows][in] (x with row stride ldx), dy, y: [rows][out] (dy: lddy),
 * W, dw, acc: [experts][out][in]; 16-byte aligned, in, out, ldx and lddy multiples
 * of 8; rows < 2^30, in and out at most 2^20, ldx and lddy at most 2^21, experts <=
 * MSR_EXPERTS_MAX; one expert's weights below 2 GiB.  An accumulator of an expert without rows is not touched.
 * ------------------------------------------------------------------------- */
int msr_experts_forward(const uint16_t *x, int64_t ldx, const uint16_t *w, uint16_t *y, const int32_t *offsets,
                        int64_t rows, int32_t experts, int64_t in_features, int64_t out_features, msr_stream_t stream);
int msr_experts_dgrad(const uint16_t *dy, int64_t lddy, const uint16_t *w, uint16_t *dx, const int32_t *offsets,
                      int64_t rows, int32_t experts, int64_t in_features, int64_t out_features, msr_stream_t stream);
int msr_experts_wgrad(uint16_t *dw, const uint16_t *x, int64_t ldx, const uint16_t *dy, int64_t lddy,
                      const int32_t *offsets, int64_t rows, int32_t experts, int64_t in_features, int64_t out_features,
                      msr_stream_t stream);
int msr_experts_wgrad_sr_accum(uint16_t *acc, const uint16_t *x, int64_t ldx, const uint16_t *dy, int64_t lddy,
                               const int32_t *offsets, int64_t rows, int32_t experts, int64_t in_features,
                               int64_t out_features, uint32_t seed, int32_t zero_init, int32_t noise_mode,
                               const uint16_t *inject, msr_stream_t stream);

/* ---------------------------------------------------------------------------
 * A language model's head with its softmax cross entropy, in pieces of the
 * vocabulary: the logits are never in memory.  No counterpart in the reference.
 *   S[n][v] = <x[n], W[v]>,  l[n] = log sum_v exp S[n][v],  loss[n] = l[n] - S[n][t[n]]
 *   G[n][v] = g[n] (exp(S[n][v] - l[n]) - [v = t[n]]),  dx = G W,  dW = G^T x
 * x: bf16, rows of ldx elements, any 2-byte alignment; W: bf16 [vocab][d],
 * 16-byte aligned; target: int32, or int64 with target_i64.  Rows whose target is
 * ignore_index have loss 0 and gradient 0, and what they hold reaches nothing; any
 * other target outside [0, vocab) makes its loss NaN, and with it the gradients.
 * reduction: MSR_LOSS_NONE (loss [rows]), _SUM or _MEAN over the rows that are not
 * ignored (loss [1]; 0 where there are none).  Products are of bf16 operands with
 * fp32 accumulation, dx and dW rounded once.  G is rounded to bf16, without the significand of
 * the first row's dloss, and but for the targets' elements in dx; of up to 32 rows that are not ignored (128 with MSR_LOSS_NONE) it is kept as two
 * bf16 numbers.
 * Logits of a magnitude below 2^127.
 *
 * msr_head_forward also writes what the backward pass reads: packed (bf16
 * [rows][d], 16-byte aligned: the rows that are not ignored, one after the other), kept
 * (int32 [3 * rows + 1]: their number, their places in x, their targets, and every
 * row's place in packed, or -1) and sums (fp32 [rows][2], packed order, 8-byte aligned:
 * M and s with l = M ln 2 + log s).
 * msr_head_backward: dloss fp32 [rows] with MSR_LOSS_NONE, else [1].  dx [rows][d]
 * or dw [vocab][d] may be NULL (not wanted).  noise_mode -1 stores dw; a noise mode
 * accumulates dw <- SR(dw + f32(bf16(dW))) with the arithmetic and noise of
 * msr_sr_accum on [vocab][d] (seed, zero_init and inject as there).
 * rows and vocab below 2^24, rows * vocab below 2^40, d a multiple of 8 up to 2^16.
 * workspaces: msr_head_workspace_bytes, 16-byte aligned.  The order of the sums, and so
 * their last bits, may depend on the sizes of the call; the same call gives the same bits.
 * ------------------------------------------------------------------------- */
#define MSR_LOSS_NONE 0
#define MSR_LOSS_SUM 1
#define MSR_LOSS_MEAN 2
int msr_head_workspace_bytes(int64_t rows, int64_t vocab, int64_t d, size_t *forward, size_t *backward);
int msr_head_forward(const uint16_t *x, int64_t ldx, const uint16_t *w, const void *target, int32_t target_i64,
                     int64_t ignore_index, int64_t rows, int64_t vocab, int64_t d, int32_t reduction, uint16_t *packed,
                     int32_t *kept, float *sums, float *loss, void *workspace, size_t workspace_bytes, msr_stream_t stream);
int msr_head_backward(const uint16_t *packed, const uint16_t *w, const int32_t *kept, const float *sums, const float *dloss,
                      int64_t rows, int64_t vocab, int64_t d, int32_t reduction, uint16_t *dx, uint16_t *dw,
                      int32_t noise_mode, uint32_t seed, int32_t zero_init, const uint16_t *inject, void *workspace,
                      size_t workspace_bytes, msr_stream_t stream);

/* ---------------------------------------------------------------------------
 * Embedding, and its gradient by sorted tokens.  No counterpart in the reference.
 *   msr_embedding                 y[i] = round(scale * W[ids[i]]), 0 for an id outside [0, vocab)
 *   msr_embedding_grad            dw[v] = round(scale * sum_{i: ids[i] = v} dy[i]), 0 without a token
 *   msr_embedding_grad_sr_accum   acc[v] <- SR(acc[v] + f32(bf16(dw[v]))) with the arithmetic and noise of
 *                                 msr_sr_accum on [vocab][d]; words without a token are not touched (with
 *                                 zero_init they are set to 0)
 * Sums in fp32, in an order that depends on the ids and sizes alone, the same for both.  Ids outside [0, vocab) and the id
 * `padding` (negative: none) give no gradient.  ids: int32, or int64 with ids_i64; W, y, dy, dw: elem
 * (MSR_BF16 or MSR_F32), contiguous but for dy's row stride lddy; aligned to their
 * types.  Fewer than 2^28 tokens and 2^27 words.  workspace:
 * msr_embedding_workspace_bytes, 8-byte aligned.
 * ------------------------------------------------------------------------- */
int msr_embedding(const void *ids, int32_t ids_i64, int64_t n, const void *w, int64_t vocab, int64_t d, float scale, void *y,
                  int32_t elem, msr_stream_t stream);
int msr_embedding_workspace_bytes(int64_t n, int64_t vocab, int64_t d, size_t *bytes);
int msr_embedding_grad(const void *ids, int32_t ids_i64, int64_t n, const void *dy, int64_t lddy, int64_t vocab, int64_t d,
                       float scale, int64_t padding, void *dw, int32_t elem, void *workspace, size_t workspace_bytes,
                       msr_stream_t stream);
int msr_embedding_grad_sr_accum(const void *ids, int32_t ids_i64, int64_t n, const uint16_t *dy, int64_t lddy, int64_t vocab,
                                int64_t d, float scale, int64_t padding, uint16_t *acc, uint32_t seed, int32_t zero_init,
                                int32_t noise_mode, const uint16_t *inject, void *workspace, size_t workspace_bytes,
                                msr_stream_t stream);

/* ---------------------------------------------------------------------------
 * Layer norm over rows of d elements, and its gradient.  No counterpart in the
 * reference.
 *   mean = mean(x), rstd = 1 / sqrt(mean((x - mean)^2) + eps), h = (x - mean) rstd, y = h w + b
 *   q = dy w, dx = rstd (q - mean(q) - h mean(q h)), dw = sum_n dy h, db = sum_n dy
 * x, y, dy, dx: elem, x and dy with row strides ldx and lddy; w (NULL: 1), b (NULL: 0), dw, db:
 * welem.  Statistics and sums in fp32, one rounding.  mean (fp32 [2][rows]: two numbers whose sum is
 * a row's mean, so that rows far from zero keep their digits) and rstd (fp32 [rows]) are written by the
 * forward pass and read by the other.  dx, dw, db may be NULL (not
 * wanted).  Aligned to their types.  workspace: msr_layer_norm_workspace_bytes (dw or
 * db wanted).  dw and db are sums in an order that depends on the sizes alone.
 * ------------------------------------------------------------------------- */
int msr_layer_norm(const void *x, int64_t ldx, const void *w, const void *b, float eps, int64_t rows, int64_t d, void *y,
                   float *mean, float *rstd, int32_t elem, int32_t welem, msr_stream_t stream);
int msr_layer_norm_workspace_bytes(int64_t rows, int64_t d, int32_t elem, size_t *bytes);
int msr_layer_norm_grad(const void *dy, int64_t lddy, const void *x, int64_t ldx, const void *w, const float *mean,
                        const float *rstd, int64_t rows, int64_t d, void *dx, void *dw, void *db, int32_t elem,
                        int32_t welem, void *workspace, size_t workspace_bytes, msr_stream_t stream);

/* ---------------------------------------------------------------------------
 * A router's balance loss.  No counterpart in the reference.  For the n tokens whose
 * mask (one byte each; NULL: all) is not 0,
 *   p[t] = softmax(logits[t]), counts[e] = their slots (t, j) with ids[t][j] = e, f[e] = counts[e] / (n k)
 *   loss = experts / n * sum_e f[e] sum_t p[t][e]      (0 where n is 0)
 *   dlogits[t][e] = dloss p[t][e] (u[e] - sum_j u[j] p[t][j]), u[e] = experts / n f[e]; 0 for the other tokens
 * ids outside [0, experts) are dropped slots.  Logits of -inf have probability 0 (a token without any
 * other: 0 everywhere).  logits: elem, row stride ld; ids: int32, or int64 with ids_i64,
 * contiguous [tokens][k]; counts int32 [experts]; stats (fp32 [2][tokens]: a token's largest logit m and
 * 1 / sum exp(logit - m)) and slope (u, fp32 [experts]) are written for the gradient.  tokens * k < 2^30, experts <= MSR_EXPERTS_MAX.
 * workspace: msr_balance_workspace_bytes.
 * ------------------------------------------------------------------------- */
int msr_balance_workspace_bytes(int64_t tokens, int32_t experts, size_t *bytes);
int msr_balance_loss(const void *logits, int64_t ld, const void *ids, int32_t ids_i64, const uint8_t *mask, int64_t tokens,
                     int32_t experts, int32_t k, float *loss, int32_t *counts, float *stats, float *slope, int32_t elem,
                     void *workspace, size_t workspace_bytes, msr_stream_t stream);
int msr_balance_grad(const void *logits, int64_t ld, const uint8_t *mask, const float *stats, const float *slope,
                     const float *dloss, int64_t tokens, int32_t experts, void *dlogits, int32_t elem, msr_stream_t stream);

/* ---------------------------------------------------------------------------
 * Diagnostics (no counterpart in the reference; used by the parity tests).
 * ------------------------------------------------------------------------- */

/* out[i] = 16-bit noise of stream (seed, k) at offset offset0 + i. */
int msr_noise_fill(uint16_t *out, int64_t n, int64_t offset0, uint32_t seed, uint32_t k,
                   int32_t noise_mode, msr_stream_t stream);

/* Streaming probe of the fused 8-bit step's memory accesses: the pair walk, loads and
 * stores of the fast kernel over n elements (n a multiple of 512; p, g 16-byte and the
 * codes 8-byte aligned; absmax1/2 hold n/256 floats), with the arithmetic replaced by one
 * integer operation per word (every buffer is overwritten).  `grid` work-groups of 256
 * threads, each holding `lds_bytes` (<= 64 KiB) of LDS that sets the work-groups per CU.
 * Measurement aid: no counterpart in the reference. */
int msr_stream_probe8(uint16_t *p, const uint16_t *g, uint8_t *state1, uint8_t *state2, float *absmax1,
                      float *absmax2, int64_t n, int32_t grid, int32_t lds_bytes, msr_stream_t stream);

/* out[i] = quantizer code of x[i] against qmap (reference search rule), or
 * through qtable when it is not NULL. */
int msr_quantize(const float *x, uint8_t *out, int64_t n, const float *qmap, int32_t is_signed,
                 const void *qtable, msr_stream_t stream);

/* Host-side construction of the quantizer table for a (signed, unsigned)
 * codebook pair (HOST pointers, 256 floats each) into a HOST buffer of
 * msr_quant_table_bytes() bytes.  Valid for codebooks on which the reference
 * search is monotone (the bitsandbytes dynamic maps are; proven exhaustively
 * by msr_quant_table_check). */
size_t msr_quant_table_bytes(void);
int msr_quant_table_build(const float *qmap_signed, const float *qmap_unsigned, void *table, size_t table_bytes);

/* Device self-check of a table against the search for every float bit
 * pattern u in [bits_lo, bits_hi] (<= bits(1.0f)): signed map at +x and -x,
 * unsigned map at x, through both the two-level lookup of the general 8-bit
 * kernel and the flat table of the fast one.  counts[i] = mismatches found by
 * work-group i. */
int msr_quant_table_check(const void *qtable, const float *qmap_signed, const float *qmap_unsigned,
                          uint32_t bits_lo, uint32_t bits_hi, uint32_t *counts, int32_t n_counts,
                          msr_stream_t stream);

/* Device self-check of the fast kernel's correctly rounded building blocks
 * against the IEEE operations, over the float bit patterns u in
 * [bits_lo, bits_hi]: kind 0 sqrt, alone and fused into the update's
 * sqrt(v) + eps (u <= bits(2^62)); kind 1 reciprocal
 * (bits(2^-60) <= u < bits(2^32)); kind 2 quotient m/d of the requantization
 * for 16 hashed m per d (bits(2^-60) <= u < bits(2)); kind 3 the hardware
 * fp32->bf16 round-to-nearest-even of the GEMM epilogues against the
 * bit-level rounding (any u); kind 4 the update's quotient n/d for 16 n per d
 * (+-0 and |n| in [2^-90, 2^60]; bits(2^-60) <= u < bits(2^32)); kind 5 the quotient m/d of
 * the bf16-moment step's scaled denominators for 16 m per d (0 and [2^-43, 2^44];
 * bits(2^16) <= u <= bits(2^32)).
 * counts[i] = mismatches found by work-group i.  Test support: no
 * counterpart in the reference. */
int msr_fastmath_check(int32_t kind, uint32_t bits_lo, uint32_t bits_hi, uint32_t *counts, int32_t n_counts,
                       msr_stream_t stream);

/* One product of the small-tile kernels in a given tile (64 or 128 wide) and ring (2 or 4 LDS stages),
 * which the library otherwise picks by size; row-major contiguous operands, m and n multiples of the tile, k of
 * 64, every extent at most 16384.
 *   product 0  d = alpha p p^T                          p [batch][m][k]; resid out
 *   product 1  d = alpha p p + beta p + diag I, the diagonal corrected for rvec (p symmetric, m = n = k;
 *              d_ii += rvec_i (beta + 2 alpha p_ii)); resid out
 *   product 2  d = alpha (p q + bf16(rvec) q)           p [batch][m][m], q [batch][m][n], rvec [batch][m]
 *   product 3  d <- SR(d + bf16(p^T q)), noise of seed  p [k][m], q [k][n]; batch 1
 * resid [batch][m]: fp32 rounding residuals of d's diagonal.  Test support: no counterpart in
 * the reference. */
int msr_tile_gemm(int32_t product, int32_t tile, int32_t stages, const uint16_t *p, const uint16_t *q, uint16_t *d,
                  int64_t batch, int64_t m, int64_t n, int64_t k, float alpha, float beta, float diag,
                  const float *rvec, float *resid, uint32_t seed, int32_t noise_mode, msr_stream_t stream);

/* Host only: the tile (64, 128 or 256) that an experts' product of these sizes takes, and whether it splits K
 * between groups of waves; product 0 forward, 1 dgrad, 2 wgrad, 3 wgrad_sr_accum.  Test support. */
int msr_experts_tile(int32_t product, int64_t rows, int32_t experts, int64_t in_features, int64_t out_features, int32_t *tile,
                     int32_t *split);

/* Host only: how a head of these sizes is computed: plan[7] = the tiles of the loss's logits, of the gradient's, of dx
 * and its splits of the vocabulary, of dW and its splits of the rows, and the words of a piece.  Test support. */
int msr_head_plan(int64_t rows, int64_t vocab, int64_t d, int32_t *plan);

/* Batched bf16 GEMM  D[b] = alpha * P[b] Q[b]^T + beta * C[b] + diag * I  (fp32 accumulate, RNE
 * bf16 out; the diag term is added where m == n).
 * P: [M][K] (row stride ldp), Q: [N][K] (ldq), C/D: [M][N] (ldc/ldd); C may be NULL when beta == 0.
 * M, N multiples of 256 and K a multiple of 128 (the NS workspace is padded to these). */
int msr_gemm_nt(const uint16_t *P, int64_t ldp, int64_t strideP, const uint16_t *Q, int64_t ldq,
                int64_t strideQ, const uint16_t *C, int64_t ldc, int64_t strideC, uint16_t *D, int64_t ldd,
                int64_t strideD, int64_t M, int64_t N, int64_t K, int64_t batch, float alpha, float beta,
                float diag, msr_stream_t stream);

/* The same with a K-major Q:  D[b] = alpha * P[b] Q[b] + beta * C[b] + diag * I,  Q: [K][N] (row
 * stride ldq).  This is the kernel of Newton-Schulz's X' = B' X.  Test support: no counterpart in
 * the reference. */
int msr_gemm_nn(const uint16_t *P, int64_t ldp, int64_t strideP, const uint16_t *Q, int64_t ldq,
                int64_t strideQ, const uint16_t *C, int64_t ldc, int64_t strideC, uint16_t *D, int64_t ldd,
                int64_t strideD, int64_t M, int64_t N, int64_t K, int64_t batch, float alpha, float beta,
                float diag, msr_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* MUON_SR_AMD_H */
