/*
 * anneal_hip.h — C ABI of libanneal_hip.so, the MI355X (gfx950) backend for anneal's training hot path.
 *
 * Plain C types only (pointers, sizes, int codes). Every call returns AH_OK (0) or an AH_ERR_* code;
 * the message of the last failure on the calling thread is available from ah_last_error().
 * A device handle serializes all work onto one HIP stream; calls on one handle are not re-entrant
 * (the reference funnels every call onto a single owner thread: backend/webgpu/open.go:68-80).
 *
 * Each declaration names the reference interface it replaces (paths inside georgebuilds/anneal).
 */
#ifndef ANNEAL_HIP_H
#define ANNEAL_HIP_H
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define AH_OK 0
#define AH_ERR_INVALID 1     /* bad argument / shape / handle */
#define AH_ERR_HIP 2         /* HIP runtime error */
#define AH_ERR_UNSUPPORTED 3 /* dtype or feature the device lacks (fail closed, executor.go:42-50) */
#define AH_ERR_COMPILE 4     /* hiprtc compilation failed */
#define AH_ERR_NOMEM 5

/* Buffer element types; numbering follows the reference's dtype set used on the device boundary
 * (backend/webgpu/executor.go:470-528): f16 is 2 bytes, every other type travels in 4 bytes. */
enum { AH_F32 = 0, AH_F16 = 1, AH_BF16 = 2, AH_I32 = 3, AH_BOOL = 4, AH_U32 = 5 };

typedef struct ah_device ah_device;
typedef struct ah_kernel ah_kernel;
typedef struct ah_graph ah_graph;
typedef struct ah_trainer ah_trainer;
typedef struct ah_plan ah_plan;

typedef struct {
    int32_t has_f16;     /* shader-f16 equivalent (always 1 on gfx950) */
    int32_t has_bf16;
    int32_t cu_count;
    int32_t wavefront;   /* 64 */
    int64_t hbm_bytes;
    int64_t lds_bytes_per_block;
    char arch[64];       /* e.g. "gfx950:sramecc+:xnack-" */
} ah_caps;

/* ── 1. device ───────────────────────────────────────────────────────────────
 * Replaces webgpu.Open (backend/webgpu/open.go:89) and Executor.Close (backend/device.go:12). */
const char *ah_last_error(void);
int ah_open(int ordinal, ah_device **out);
void ah_close(ah_device *dev);
int ah_get_caps(ah_device *dev, ah_caps *out);
int ah_sync(ah_device *dev);

/* ── 2. buffers and the dtype codec ──────────────────────────────────────────
 * Replaces the per-Run CreateBuffer / WriteBuffer / readBuffer of backend/webgpu/executor.go:83-179,397-468
 * and the codec of executor.go:470-528 / uop/dtype.go:392-487 (f32->f16 round-to-nearest-even with the
 * reference's NaN and overflow rules; bf16 = top 16 bits carried in a 4-byte slot). */
int ah_buf_alloc(ah_device *dev, int64_t n_elems, int32_t dtype, void **dptr);
int ah_buf_free(ah_device *dev, void *dptr);
int ah_upload(ah_device *dev, void *dptr, const float *src, int64_t n, int32_t dtype);
int ah_download(ah_device *dev, float *dst, const void *dptr, int64_t n, int32_t dtype);
int ah_upload_bytes(ah_device *dev, void *dptr, const void *src, int64_t nbytes);
int ah_download_bytes(ah_device *dev, void *dst, const void *dptr, int64_t nbytes);
uint16_t ah_f32_to_f16(float f);   /* uop/dtype.go:392 Float32ToFloat16 */
float ah_f16_to_f32(uint16_t h);   /* uop/dtype.go:447 Float16ToFloat32 */

/* ── 3./4. modules and launches ──────────────────────────────────────────────
 * Replaces CreateShaderModule + pipeline creation + Dispatch (backend/webgpu/executor.go:254-395).
 * `source` is either HIP C++ source (compiled once by hiprtc for gfx950, cached by source hash) or a
 * template key "tmpl:<name>;k=v;..." selecting a hand-written kernel (the names and their keys are
 * listed in anneal_amd/csrc/templates.cpp).
 * Kernel arguments: n_ptrs device pointers (data0 = output, data1.. = inputs, PARAM order as in
 * codegen/wgsl.go:58-76), then n_scalars int32 values (the params_n uniform of symbolic kernels). */
int ah_module_get(ah_device *dev, const char *source, const char *entry, ah_kernel **out);

/* The WGSL anneal's codegen renders (codegen/wgsl.go:41-238 RenderWGSL, the string the schedule cache
 * keeps in ExecItem.WGSL, schedule/cache.go:69-100) is also accepted as `source` by ah_module_get / ah_run:
 * it is rendered as HIP C++ (entry point `kernel`, the storage bindings in binding order, then the four
 * int32 fields of params_n for symbolic kernels) and compiled by hiprtc. This call exposes that rendering
 * on its own (no device needed): writes at most cap bytes of NUL-terminated HIP source to out and the
 * full size to *needed; AH_ERR_COMPILE if the WGSL is outside the subset the reference emits. */
int ah_translate_wgsl(const char *wgsl, char *out, int64_t cap, int64_t *needed);
/* Template selection for a rendered WGSL kernel (host only, no device). The kernel's body, in the form
 * codegen/lower.go:98-719 lowers and codegen/wgsl.go:41-386 renders it (one let per ALU node and load,
 * GIDVar axes, one accumulator and loop per reduce, f16 reduces widened and narrowed with f16(acc),
 * params_n for a symbolic batch), is parsed with every let substituted, and two families select a
 * hand-written kernel: a contraction REDUCE(ADD, MUL(a, b)) whose operands are loads, ReLU prologues
 * max(x, 0.0) or ReLU-backward mask prologues select(0.0, adj, z == max(z, 0.0)), stored as acc,
 * f16(acc), c*acc, acc + bias[n] or max(acc + bias[n], 0.0) -> "tmpl:gemm;..." (dtype f32 or f16, M/N/K
 * "sym" where symbolic); and a reduction REDUCE(ADD|MAX, load) along a row or down a column (or over a
 * whole 1-D buffer) stored into f32 -> "tmpl:reduce;...". Index expressions must evaluate as affine with
 * zero offset over the axes. Writes the key ah_module_get runs in the kernel's place to buf, or "". No
 * counterpart in the reference, whose backend renders every kernel: it exposes the selection
 * ah_module_get and ah_run make (AH_WGSL_TEMPLATES=0 turns it off). */
int ah_wgsl_template_key(const char *wgsl, char *buf, int32_t cap);
/* How ah_module_get runs a rendered WGSL kernel (host only): writes the template key when one is selected
 * (as above), "wave" when the kernel is rendered in the wave-per-output form (a single-reduce kernel:
 * one 64-lane wave per output element, the lanes striding the outermost reduce loop and combining their
 * partials with a shuffle tree, AH_WGSL_WAVE=0 turns it off), or "thread" for the one-thread-per-output
 * rendering of ah_translate_wgsl. AH_ERR_COMPILE if the WGSL is outside the subset. */
int ah_wgsl_plan(const char *wgsl, char *buf, int32_t cap);
int ah_launch(ah_device *dev, ah_kernel *k, const uint32_t grid[3], const uint32_t block[3],
              void *const *ptrs, int32_t n_ptrs, const int32_t *scalars, int32_t n_scalars);

/* ── 5. timing ───────────────────────────────────────────────────────────────
 * Replaces Benchmarker.Benchmark's wall-clock loop (backend/webgpu/benchmark.go:18-208) with hipEvents. */
typedef struct {
    double min_us, median_us, max_us, mean_us, stddev_us, cv;   /* backend/device.go:16-24 */
} ah_bench_result;

/* Wall time of everything enqueued on the device stream between start and stop (hipEvents). */
int ah_timer_start(ah_device *dev);
int ah_timer_stop(ah_device *dev, double *ms);

/* ── 6. graphs (JIT replay) ──────────────────────────────────────────────────
 * Replaces tensor.JIT's replay of captured ExecItems (tensor/jit.go:178-215): everything enqueued on the
 * device stream between begin and end is captured and can be replayed without host scheduling. */
int ah_graph_begin(ah_device *dev);
int ah_graph_end(ah_device *dev, ah_graph **out);
int ah_graph_replay(ah_device *dev, ah_graph *g);
void ah_graph_destroy(ah_graph *g);

/* ── Executor mirror (backend.Executor / Benchmarker / SymbolicExecutor, backend/device.go:10-37) ──
 * Items follow schedule.ExecItem (schedule/exec.go:6-32): bufs[0] is the output, bufs[1..] inputs in
 * PARAM order; slot >= 0 marks a slot shared by non-overlapping lifetimes, -1 a leaf or final output.
 * Final outputs are the bufs[0] that no later item reads; they are returned widened to f32 (4-byte
 * integer types as raw bits), keyed by uop_idx, in ah_output arrays owned by the library. */
typedef struct {
    uint32_t uop_idx;
    int64_t size;        /* elements; 0 when the leading dim is symbolic */
    int32_t dtype;
    int32_t slot;
    int32_t rank;
    const int64_t *shape;
} ah_buffer_desc;

typedef struct {
    const char *source;           /* HIP source or "tmpl:" key (replaces the WGSL string field) */
    const ah_buffer_desc *bufs;
    int32_t n_bufs;
    const char *const *sym_vars;
    int32_t n_sym_vars;
    int32_t local_size[3];
    int32_t workgroup_count[3];
} ah_exec_item;

typedef struct {
    uint32_t uop_idx;
    const float *data;
    int64_t n;
} ah_input;

typedef struct {
    uint32_t uop_idx;
    float *data;
    int64_t n;
} ah_output;

int ah_run(ah_device *dev, const ah_exec_item *items, int32_t n_items, const ah_input *inputs, int32_t n_inputs,
           ah_output **outputs, int32_t *n_outputs);                       /* Executor.Run, device.go:11 */
int ah_run_symbolic(ah_device *dev, const ah_exec_item *items, int32_t n_items, const ah_input *inputs,
                    int32_t n_inputs, const char *const *bind_names, const int64_t *bind_values,
                    int32_t n_bind, ah_output **outputs, int32_t *n_outputs); /* RunSymbolic, device.go:35-37 */
int ah_benchmark(ah_device *dev, const ah_exec_item *item, int32_t warmup, int32_t iterations,
                 ah_bench_result *out);                                     /* Benchmark, device.go:27-29 */
void ah_outputs_free(ah_output *outputs, int32_t n);

/* Persistent plans: the device half of tensor.JIT (tensor/jit.go:47-359), which captures one item list and
 * replays it through Run / RunSymbolic with fresh leaf data every step (replayStatic / replaySym,
 * jit.go:178-215). ah_plan_create copies the items, resolves every kernel once (compile errors surface here)
 * and ah_plan_run runs them with Run's contract (zeroed buffers, leaves from `inputs`, final outputs
 * returned as by ah_run). Buffers stay allocated between runs and grow when a larger symbolic binding
 * arrives. With AH_PLAN_GRAPH the kernel sequence of each binding is captured once as a HIP graph and
 * replayed afterwards (uploads and downloads stay outside the graph). ah_plan_stats reports
 * (captures, replays) like JIT.JITStats (jit.go:71-74). A plan belongs to its device handle's stream. */
#define AH_PLAN_GRAPH 1
int ah_plan_create(ah_device *dev, const ah_exec_item *items, int32_t n_items, ah_plan **out);
int ah_plan_run(ah_plan *plan, const ah_input *inputs, int32_t n_inputs, const char *const *bind_names,
                const int64_t *bind_values, int32_t n_bind, int32_t flags, ah_output **outputs, int32_t *n_outputs);
int ah_plan_stats(const ah_plan *plan, int64_t *captures, int64_t *replays);
void ah_plan_destroy(ah_plan *plan);

/* ── Hot-path kernels, callable directly ────────────────────────────────────── */

/* GEMM-shaped REDUCE(ADD, MUL) with fused epilogue (tensor/reduce.go:105-166 as scheduled for
 * Linear.Forward nn.go:154-162 and the backward rules gradient_ruleset.go:137-140,207-233,285-306).
 * C[m,n] = epi(sum_k A(m,k) B(n,k)); A stored [M,K] (ta=0) or [K,M] (ta=1); B [N,K] (tb=0) or [K,N] (tb=1). */
enum { AH_EPI_STORE = 0, AH_EPI_BIAS = 1, AH_EPI_BIAS_RELU = 2, AH_EPI_MSE = 3, AH_EPI_MASK = 4, AH_EPI_SGD = 5 };
typedef struct {
    int32_t dtype;          /* AH_F32 or AH_F16 (operands); accumulation is always f32 */
    int32_t epi;
    int32_t ta, tb;
    int32_t M, N, K;
    const void *A;
    const void *B;
    int64_t lda, ldb;
    void *C;
    int64_t ldc;
    const void *bias;
    const void *aux;
    int64_t ldaux;
    float scale;
    float *colsum;
    float *W32;
    void *W16;
    float lr;
    float *gout;
    float *lossacc;
    int32_t tile;           /* 0 = auto, 64, 128, 256 (register-staged f32 kernel), 1000 + i (f32 direct-to-LDS
                               configuration i, 0..4; see ah_gemm_tune) */
    int32_t variant;        /* f16 kernel variant: 0 = auto (the tuned choice if any), 1..39 = fixed tile /
                               wave / fetch / k-group / MFMA-shape choices (table Var<V>, gemm16_kernel.h);
                               the knob a BEAM-style search times (codegen/beam.go:41-541) */
} ah_gemm_desc;
int ah_gemm(ah_device *dev, const ah_gemm_desc *d);

/* BEAM over the f16 kernel variants (replaces BeamSearch timing candidate Opt sequences per kernel and
 * caching the winner, codegen/beam.go:41-541, :118-169). Times every variant of the contraction d
 * describes (iterations launches each, after one warm-up, on the device stream with hipEvents; two passes,
 * each variant timed by the lower of its two means), returns
 * the fastest and its mean time, and caches the choice on the device: later launches of the same
 * (ta, tb, M, N, K) with variant 0 use it. Where variant 0 by itself runs a kernel that is no variant (few
 * tiles, sizes that no tile divides, few outputs) and that kernel is the fastest, *best_variant is 0 and
 * nothing is cached (for few tiles: past K = 256). d is launched as given, so its outputs must be scratch
 * (the epilogue runs 2 * (iterations + 1) times per variant). Variants without k-groups differ only in
 * tiling and scheduling and accumulate each output over k in the same order (bit-identical results);
 * the k-group variants 10, 11, 15, 25, 28, 31 and 35-38 add two k-halves, which rounds differently in f32 (relative
 * 1e-6 level). For an f32 contraction (dtype AH_F32) the candidates are the f32 kernel's (tile, k-groups,
 * splits of K across workgroups) configurations and the direct-to-LDS kernel's, 58 in all, and
 * *best_variant is the winner's index: 0 is the shape's automatic choice, then the register-staged
 * kernel's tile 64 and 128 each with k-groups auto / 1 / 2 / 4 (as the tile admits) and splits auto / 1 /
 * 2 / 4 / 8 / 16 in that nesting order (a fixed k-group count takes no automatic split, so splits auto is
 * listed only with k-groups auto), indices 1-37; then the direct-to-LDS configurations 0-4 (tile 64 with
 * k 64 x 3 stages, 64 x 4, 32 x 4; tile 128 with k 32 x 4, 64 x 2), indices 38-42, then each of those
 * with K split across 2 / 4 / 8 workgroups (43-57; the partials folded in split order as the
 * register-staged kernel folds them). The automatic choice is
 * the direct-to-LDS kernel on 64-wide tiles when they number at least 256 (at least 128 for K <= 1024),
 * the register-staged kernel otherwise. Later f32 launches of the shape with tile, k-groups and splits all automatic use the
 * winner. Configurations add K in different orders, so their results differ at the rounding level;
 * those of one tile width without k-groups or splits give the same bits in either kernel. */
int ah_gemm_tune(ah_device *dev, const ah_gemm_desc *d, int32_t iterations, int32_t *best_variant, double *best_us);
/* BEAM's disk cache (codegen/beam.go:118-169): save (save != 0) the device's tuned choices to path, one
 * "dtype/ta/tb/M/N/K variant" line each under a header naming the gfx arch, or merge a saved file into
 * the device's cache (a file timed on another arch is ignored). The config-3 trainer loads and rewrites
 * the file named by the environment variable AH_GEMM_TUNE_CACHE around its tuning. */
int ah_gemm_tune_cache(ah_device *dev, const char *path, int32_t save);

/* ── The Opt seam and BEAM over the HIP templates ─────────────────────────────
 * Replaces codegen/opt.go's ApplyOpt/ApplyOpts (:29-72, :559-567) and codegen/beam.go's ActionSpace,
 * BeamSearch, BeamApplyToItems and disk cache (:41-541). An Opt {kind, axis, arg} (opt.go:41-46) edits a
 * template key's tuning parameters instead of an AST: LOCAL(axis 0|1, 8|16|32) the waves along M or N
 * (arg/8), UPCAST(axis 0|1, 2|4) the MFMA register tile per wave (f32 kernel: tile 64*arg), TILE(axis 2,
 * 8|16|32) the LDS stage (k 32 x 4 stages, 64 x 2, 64 x 3), VECTORIZE(axis 2, 4) 16-byte asm LDS-DMA
 * staging (f32: the direct-to-LDS kernel, whose stage TILE then sets; the key gets dma=i);
 * GROUP(axis 2, 2|4) k-groups, SCHEDULE(axis 0, 5..7) the DMA/fragment-read interleave and MFMA(axis 2,
 * 16|32) the f16 kernel's MFMA shape (16x16x32 or 32x32x16; bit-identical results) are MI355X additions.
 * Only "tmpl:gemm" keys have tunable parameters. */
enum { AH_OPT_IDENTITY = 0, AH_OPT_LOCAL = 1, AH_OPT_TILE = 2, AH_OPT_UPCAST = 3, AH_OPT_VECTORIZE = 4,
       AH_OPT_GROUP = 5, AH_OPT_SCHEDULE = 6, AH_OPT_MFMA = 7 };
typedef struct {
    int32_t kind, axis, arg;
} ah_opt;
/* ApplyOpts: the key with the sequence applied (NUL-terminated, at most cap bytes; *needed = full size);
 * AH_ERR_UNSUPPORTED if an Opt does not apply or the result is not an instantiated kernel. */
int ah_apply_opts(const char *key, const ah_opt *opts, int32_t n, char *out, int64_t cap, int64_t *needed);
/* ActionSpace (beam.go:53-72): every single Opt that changes the key's kernel; *n = count, at most cap
 * written to out. */
int ah_action_space(const char *key, ah_opt *out, int32_t cap, int32_t *n);
typedef struct {
    double min_us, base_us;   /* winner's and the unmodified kernel's min-of-N times */
    int32_t searched;         /* candidates benchmarked */
    int32_t from_cache;
    int32_t n_opts;
    ah_opt opts[8];           /* the winning sequence (empty: identity) */
} ah_beam_result;
/* BeamSearch (beam.go:271-408) over item (a "tmpl:" item, buffers as for ah_benchmark): beam width and
 * depth, each candidate timed by ah_benchmark (warmup, iters; min), kept only if its output is
 * bit-identical to the unmodified kernel's on fixed inputs (beam.go:410-451). The winner is cached per
 * process keyed by the FNV-64a hash of the item's key; a cached kernel is re-timed, not searched. A key
 * that runs the f16 split or dot kernel (see ah_gemm_tune) has no candidate with its bits: the winner is
 * the key itself. */
int ah_beam_search(ah_device *dev, const ah_exec_item *item, int32_t width, int32_t depth, int32_t warmup,
                   int32_t iters, ah_beam_result *out);
/* BeamApplyToItems' cache hit (beam.go:470-541): the cached specialised key for key, or key itself; the
 * stored hash of the specialised key guards against key-hash collisions. */
int ah_beam_apply(const char *key, char *out, int64_t cap, int64_t *needed);
/* The persistent cache (beam.go:100-150): save (save != 0) every cached winner to path, or merge path
 * into the process cache. */
int ah_beam_cache(const char *path, int32_t save);
void ah_beam_reset(void);   /* BeamCacheReset (beam.go:213) */

/* Softmax cross-entropy forward+backward composed from reference ops, one kernel:
 * m=Max, zs=z-m, e=Exp(zs), s=Sum e, logp=zs-Log(s), loss=Sum(onehot*logp)*(-1/B); dz includes the
 * row-max path with its tie split (tensor/gradient_ruleset.go:307-320). */
int ah_softmax_ce(ah_device *dev, const float *z, const int32_t *labels, int32_t B, int32_t C, float *dz,
                  float *loss);

/* Config-5 chain: Y = Shrink(Pad(Permute(X,(1,0)))), S = softmax(Y, 1),
 * out = S * recip(sqrt(mean(S*S,1) + 1e-6)) * g; loss = Sum(out); returns dX [R,Cc], dg [Cc]. dX may be X and
 * dg may be g. */
int ah_chain_step(ah_device *dev, const float *X, const float *g, int32_t R, int32_t Cc, float *dX, float *dg,
                  float *loss);
/* ah_chain_step without allocation. No counterpart in the reference: it is for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops). The chain's workspace is a
 * file-scope device array of 2^22 floats (16 MiB per GPU, held until the process ends), so
 * 64 + ceil(R/64)*Cc*4 + Cc*8 + ceil(Cc/16) must not exceed 2^22 (config 5, 8192 x 4096, needs 2.13M);
 * larger shapes fail with AH_ERR_INVALID. Asynchronous: the chain's kernel (three for shapes that do not
 * fit on chip in one round of workgroups) is enqueued on the device stream and the call returns (ah_sync waits). Every call on one GPU
 * shares that GPU's workspace, so calls of several device handles that overlap on one GPU race: their
 * outputs are undefined (those of later calls are not, as the kernel's counters are each handle's). */
int ah_chain_step_noalloc(ah_device *dev, const float *X, const float *g, int32_t R, int32_t Cc, float *dX,
                          float *dg, float *loss);

/* ── The ends of a language model's training step ─────────────────────────────
 * No counterpart in the reference (no softmax, no cross-entropy and no update rule but SGD: tensor/nn/nn.go:69-106). All calls
 * are asynchronous on the device stream and allocate nothing, so they can be captured by ah_graph_begin; each takes a workspace
 * of the caller's, whose size the *_workspace call gives for the same descriptor (pointers set or not, and W at a multiple
 * of 16 bytes or not, as in the call). The workspace needs 16-byte
 * alignment and no particular contents; calls of one device handle may share one. Graphs hold its address.
 *
 * Softmax cross-entropy of a linear head, whose logits are worked on in pieces of rows. X [N,D], W [V,D], bias [V] (may be null),
 * labels [N]:
 *   z = X W^T + bias, lse_n = log sum_v exp z_nv, rowloss_n = lse_n - z_n,label(n)
 *   P = exp(z - lse) - onehot(label), s = grad_scale (over the number of counted rows, if mean)
 *   dX = s P W, dW = s P^T X, dbias = s sum_n P
 * A row whose label is outside [0, V) does not count: its rowloss, lse and dX are 0, and what X holds there is not used (it
 * may be NaN). loss is the counted rows' sum, divided by their number if mean (0 when there are none; all gradients are 0 then).
 * Null dX, dW or dbias are not computed; with all three null the call does the loss alone. A bias of -inf rules a class out (as a
 * label it gives an infinite loss and the gradient above). A logit of +inf or NaN makes its row's loss, lse and dX NaN, and dW and
 * dbias, which sum over rows; the other rows are as without it.
 * dtype (X, W, bias) AH_F32 or AH_F16; grad_dtype (dX, dW) AH_F32, or AH_F16 where dtype is AH_F16. loss, rowloss, lse and dbias are
 * f32; losses and statistics are computed in f32 or wider. f32 operands take part in the products with 22 bits of each value (less
 * below 2^-14 of the operand's largest magnitude). P takes part with 22 bits for f32 gradients, for f16 ones with 11, and 22 at the
 * label; all down to an absolute 2^-40. Gradients of f16 that would underflow take a loss scale as grad_scale. Results repeat bit for
 * bit (for one piece_mb: more pieces round dW more often). Row strides ldx, ldw, lddx, lddw are in elements (an array's rows may
 * span 2^48 of them). Outputs may not overlap inputs or one another, from their first element to their last.
 * With gradients, up to piece_mb MiB of f32 logits are in the workspace at a time (whole, if they take no more). Beside them there are
 * X's counted rows and, if W is f32 or its rows are not 16-byte aligned (and there are more than 128 rows of X), W, each once more;
 * at most an eighth of a piece for statistics and db; V D floats for dW in f16 over several pieces; and partial sums of products, some
 * hundred MiB at most. */
typedef struct {
    int32_t dtype, grad_dtype;
    int32_t N, D, V;
    int32_t mean;
    const void *X;
    int64_t ldx;
    const void *W;
    int64_t ldw;
    const void *bias;
    const int32_t *labels;
    float *loss;           /* [1] */
    float *rowloss;        /* [N] or null */
    float *lse;            /* [N] or null */
    void *dX;
    int64_t lddx;
    void *dW;
    int64_t lddw;
    float *dbias;
    float grad_scale;
    int32_t piece_mb;      /* MiB of logits that are kept at a time with gradients, or of statistics without; 0: 2048. At least 256 rows are */
    void *ws;
    int64_t ws_bytes;
} ah_linear_ce_desc;
int ah_linear_ce_workspace(ah_device *dev, const ah_linear_ce_desc *d, int64_t *bytes);
int ah_linear_ce(ah_device *dev, const ah_linear_ce_desc *d);

/* Newton-Schulz orthogonalisation of a matrix G [rows, cols], or of `batch` of them:
 *   X = G / (|G|_F + eps); steps times: A = X X^T (X^T X if rows > cols), X <- (a I + b A + c A A) X (X (..)); O = X
 * dtype (of G) and out_dtype AH_F32 or AH_F16. The norm is summed in f64; products keep 22 bits of their operands (X down to
 * 2^-37) and sum in f32. The iterates before the last have to keep their singular values at 4 or less (a = 3.4445, b = -4.7750,
 * c = 2.0315 keeps them below 1.3; larger ones may end as infinities or NaN); |a| + |b| + |c| may be at most 15 and steps 1 to 64.
 * A zero matrix gives zeros, whatever eps, a non-finite one NaN. O may be G. ldg, ldo: row strides; stride_g, stride_o: from matrix
 * to matrix, in elements (read only for batch > 1). */
typedef struct {
    int32_t dtype, out_dtype;
    int32_t rows, cols, batch;
    int32_t steps;
    float a, b, c, eps;
    const void *G;
    int64_t ldg, stride_g;
    void *O;
    int64_t ldo, stride_o;
    void *ws;
    int64_t ws_bytes;
} ah_orthogonalize_desc;
int ah_orthogonalize_workspace(ah_device *dev, const ah_orthogonalize_desc *d, int64_t *bytes);
int ah_orthogonalize(ah_device *dev, const ah_orthogonalize_desc *d);

/* One weight update by an orthogonalised momentum (the place of AH_EPI_SGD in a training step):
 *   M_out = momentum M + G;  U = nesterov ? G + momentum M_out : M_out;  O = U orthogonalised as above
 *   W_out = (1 - lr decay) W - lr scale O;  W16_out = f16(W_out) (may be null)
 * G is of dtype AH_F32 or AH_F16; M, W and their outputs are f32. M_out may be M and W_out may be W; outputs may not overlap
 * anything else. M, W and the outputs share the row stride ldw and the matrix stride stride_w. */
typedef struct {
    int32_t dtype;
    int32_t rows, cols, batch;
    int32_t steps, nesterov;
    float a, b, c, eps;
    const void *G;
    int64_t ldg, stride_g;
    const float *M;
    float *M_out;
    const float *W;
    float *W_out;
    void *W16_out;
    int64_t ldw, stride_w;
    float lr, momentum, decay, scale;
    void *ws;
    int64_t ws_bytes;
} ah_muon_desc;
int ah_muon_workspace(ah_device *dev, const ah_muon_desc *d, int64_t *bytes);
int ah_muon_step(ah_device *dev, const ah_muon_desc *d);

/* ── A residual block of a training step, and clipping before its update ──────
 * No counterpart in the reference (no activation but ReLU, no norm layer, no clipping). As above: asynchronous on the device stream,
 * nothing allocated, a workspace of the caller's (where there is one) that calls of one handle may share and graphs hold.
 * An output shares no byte with another array of its call but where it says so; arrays of one row stride may lie side by side, as Z and U in
 * the halves of one [N, 2 F] array.
 *
 * Linear layer with its epilogue. X [N,D], W [F,D], bias [F]; U, R, Y, Z [N,F]:
 *   Z = X W^T + bias,  Y = R + scale act(Z) U        (elementwise; bias, U, R may be null: 0, 1, 0)
 * act: ReLU, GELU by erf or by tanh(sqrt(2/pi) (z + 0.044715 z^3)), SiLU z / (1 + exp(-z)). Z may be null; a backward pass needs it.
 * dtype (all arrays) AH_F32 or AH_F16; everything is computed in f32 from an f32 Z and each output rounded once. f32 operands take part in
 * the product with 22 bits of each value (less below 2^-14 of its row's largest magnitude), or with all 24 where there are at most 128
 * rows of 8 features or more. Y may be R. What is not finite in a row of X or W makes that row or column of the outputs infinite or NaN, and no
 * other.
 * N to 2^21, D and F to 2^20. Row strides ld* are in elements. */
enum { AH_ACT_NONE = 0, AH_ACT_RELU = 1, AH_ACT_GELU = 2, AH_ACT_GELU_TANH = 3, AH_ACT_SILU = 4 };
typedef struct {
    int32_t dtype, act;
    int32_t N, D, F;
    float scale;
    const void *X;
    int64_t ldx;
    const void *W;
    int64_t ldw;
    const void *bias;
    const void *U;
    int64_t ldu;
    const void *R;
    int64_t ldr;
    void *Y;
    int64_t ldy;
    void *Z;
    int64_t ldz;
    void *ws;
    int64_t ws_bytes;
} ah_linear_desc;
int ah_linear_workspace(ah_device *dev, const ah_linear_desc *d, int64_t *bytes);
int ah_linear(ah_device *dev, const ah_linear_desc *d);

/* Its gradients, given dY:
 *   dZ = scale dY U act'(Z),  dX = dZ W,  dW = dZ^T X,  dbias = sum_n dZ,  dU = scale dY act(Z);  dR is dY itself
 * act'(0) of ReLU is 0. Null dX, dW, dbias, dU are not computed; X is read for dW alone, W for dX alone (null otherwise), Z for an
 * act other than none and for dU. dtype (X, W, Z, U, dY, dU) AH_F32 or AH_F16, grad_dtype (dX, dW) AH_F32, or AH_F16 where dtype is; dbias
 * is f32. dZ takes part in the products with 22 bits for f32 gradients, 11 for f16 ones, f32 operands with 22 (all less below 2^-14 of
 * the array's largest magnitude). Results repeat bit for bit. */
typedef struct {
    int32_t dtype, grad_dtype, act;
    int32_t N, D, F;
    float scale;
    const void *X;
    int64_t ldx;
    const void *W;
    int64_t ldw;
    const void *Z;
    int64_t ldz;
    const void *U;
    int64_t ldu;
    const void *dY;
    int64_t lddy;
    void *dX;
    int64_t lddx;
    void *dW;
    int64_t lddw;
    float *dbias;
    void *dU;
    int64_t lddu;
    void *ws;
    int64_t ws_bytes;
} ah_linear_grad_desc;
int ah_linear_grad_workspace(ah_device *dev, const ah_linear_grad_desc *d, int64_t *bytes);
int ah_linear_grad(ah_device *dev, const ah_linear_grad_desc *d);

/* Norms after and before a block, fused with its gate and the residual sum. H, H_out (the residual stream), Y (the block's output), O (the
 * next block's input) [N,D]; row n of gate is row n / rows_per_gate (0: one row for all):
 *   H_out = skip H + scale gate post(Y),  O = pre(H_out)
 * post, pre: none, RMS x / sqrt(mean x^2 + eps) w, or layer (x - mean) / sqrt(var + eps) w + b; weights [D], may be null (1 and 0).
 * H null: no first term. Y null: no second one (gate and post then none). H_out or O may be null (O where pre is none); O is the norm of
 * H_out before its rounding. dtype (Y, O, gate, weights) AH_F32 or AH_F16; res_dtype (H, H_out) AH_F32, or AH_F16 where dtype is.
 * Computed in f32, rows of any finite size among them (a layer norm's as long as its sum is finite); H_out may be H. A row that is not finite
 * leaves the others alone. N to 2^27, D to 2^20. No workspace. */
enum { AH_NORM_NONE = 0, AH_NORM_RMS = 1, AH_NORM_LAYER = 2 };
typedef struct {
    int32_t dtype, res_dtype;
    int32_t N, D;
    int32_t post, pre;
    int32_t rows_per_gate;
    float eps, skip, scale;
    const void *H;
    int64_t ldh;
    const void *Y;
    int64_t ldy;
    const void *gate;
    int64_t ldgate;
    const void *post_w, *post_b, *pre_w, *pre_b;
    void *H_out;
    int64_t ldh_out;
    void *O;
    int64_t ldo;
} ah_residual_norm_desc;
int ah_residual_norm(ah_device *dev, const ah_residual_norm_desc *d);

/* Its gradients, given those of H_out and O (dH_out null: 0; dO is needed unless pre is none), from Y and the stored H_out:
 *   t = dH_out + pre'(dO),  dH = skip t,  dY = post'(scale gate t),  dgate = sum over its rows of scale t post(Y)
 * and the weights' gradients, sums over all rows. Null outputs are not computed. dgate is of dtype, the weights' gradients are
 * f32. Y is needed for dgate and where post is not none, H_out where pre is not none. Sums over rows run in a fixed order: results repeat
 * bit for bit. dH may be dH_out. A row's sums hold products of a gradient's entry with Y's and H_out's (less their means), gate and weights, in
 * f32: where those are past its range, so is the row, and where its mean square plus eps is (or is below 2^-126 and not eps itself) it
 * is NaN. */
typedef struct {
    int32_t dtype, res_dtype;
    int32_t N, D;
    int32_t post, pre;
    int32_t rows_per_gate;
    float eps, skip, scale;
    const void *Y;
    int64_t ldy;
    const void *gate;
    int64_t ldgate;
    const void *post_w, *post_b, *pre_w;
    const void *H_out;
    int64_t ldh_out;
    const void *dH_out;
    int64_t lddh_out;
    const void *dO;
    int64_t lddo;
    void *dH;
    int64_t lddh;
    void *dY;
    int64_t lddy;
    void *dgate;
    int64_t lddgate;
    float *dpost_w, *dpost_b, *dpre_w, *dpre_b;
    void *ws;
    int64_t ws_bytes;
} ah_residual_norm_grad_desc;
int ah_residual_norm_grad_workspace(ah_device *dev, const ah_residual_norm_grad_desc *d, int64_t *bytes);
int ah_residual_norm_grad(ah_device *dev, const ah_residual_norm_grad_desc *d);

/* The global norm of many tensors, and clipping by it:
 *   norm = unscale sqrt(sum over all entries of src^2),  coef = min(1, max_norm / (norm + eps)),  dst = unscale coef src
 * unscale: the inverse of a loss scale, or 1. A tensor is `count` consecutive elements (0 is allowed) of dtype AH_F32 or AH_F16, out_dtype
 * AH_F32, or AH_F16 where dtype is. dst null: the tensor is only counted; dst may be src where the types are the same, and is then
 * left alone where unscale coef is 1. norm and coef [1] are on the device and may be null. Squares are summed in f64 in a fixed order. If an entry
 * is infinite or NaN, so is norm; coef is then 0 and every dst is 0, so that the update that follows takes no step from them. max_norm may
 * be infinite. The array `tensors` is host memory and read during the call alone. 1 to 2^16 tensors of up to 2^40 elements in all. */
typedef struct {
    const void *src;
    void *dst;
    int64_t count;
    int32_t dtype, out_dtype;
} ah_tensor;
typedef struct {
    int32_t n;
    float max_norm, eps, unscale;
    const ah_tensor *tensors;
    float *norm;
    float *coef;
    void *ws;
    int64_t ws_bytes;
} ah_clip_desc;
int ah_clip_norm_workspace(ah_device *dev, const ah_clip_desc *d, int64_t *bytes);
int ah_clip_norm(ah_device *dev, const ah_clip_desc *d);

/* ── Device-resident training steps (one BASELINE config each) ───────────────
 * Replaces the reference step pattern: graph build -> tensor.Backward -> one tensor.Realize per gradient
 * -> host SGD (examples/mlp.go:112-142, tensor/nn/nn.go:69-106). Parameters stay resident as f32 masters
 * (plus f16 copies for f16 configs); SGD runs on the device inside the backward kernels. */
enum {
    AH_TRAIN_MLP_CE = 1,    /* dims {Bmax, D, H, C}: configs 1 and 4 */
    AH_TRAIN_CONVNET = 2,   /* dims {N, Hin, C1, C2, NC}: config 2 */
    AH_TRAIN_MLP3_F16 = 3,  /* dims {B, D0, D1, D2, D3[, adjoint]}: config 3; adjoint 1 keeps the masked
                               adjoints dZ2, dZ1 at f32 precision as two f16 planes (hi, lo) and contracts
                               both (dH1, dW2, dW1 then cost two passes over K); 0 (default) rounds them
                               to f16 */
    AH_TRAIN_CHAIN = 4,     /* dims {R, Cc}: config 5 */
};
/* Slot numbering per kind (host arrays are f32 unless noted; labels are int32):
 *  MLP_CE : 0 x, 1 labels, 2 W1, 3 b1, 4 W2, 5 b2, 6 loss, 7 dW1, 8 db1, 9 dW2, 10 db2,
 *           11 H1 (the last step's ReLU outputs, batch rows first; -0.0 marks a dead unit) — read only
 *  CONVNET: 0 x, 1 labels, 2 cw1, 3 cb1, 4 cw2, 5 cb2, 6 fw, 7 fb, 8 loss, 9 dcw1, 10 dcb1, 11 dcw2,
 *           12 dcb2, 13 dfw, 14 dfb
 *  MLP3   : 0 x, 1 t, 2 W1, 3 b1, 4 W2, 5 b2, 6 W3, 7 b3, 8 loss, 9 dW1, 10 db1, 11 dW2, 12 db2,
 *           13 dW3, 14 db3, 15 loss_sum (the f32 sum of squares before the f16 narrowing of the loss),
 *           16 H1, 17 H2 (the f16 ReLU outputs of the last step, widened; -0.0 marks a dead unit),
 *           18 d = f16(P - t) (the last step's loss adjoint before the factor 2/(B*D3)) — read only
 *  CHAIN  : 0 X, 1 g, 2 loss, 3 dX, 4 dg
 * Gradient slots are filled only by steps run with AH_STEP_STORE_GRADS.
 * Creating an MLP3 trainer tunes its f16 contractions for shapes the device has not tuned yet: each alone
 * (ah_gemm_tune), then each variant again inside running steps on hash-filled buffers (≈1.9 s in all at the
 * config-3 shape); every parameter, data and accumulator buffer is zero when create returns. */
#define AH_STEP_STORE_GRADS 1
#define AH_STEP_GRAPH 2      /* capture the step once per batch size as a hipGraph and replay it (tensor.JIT) */
int ah_trainer_create(ah_device *dev, int32_t kind, const int64_t *dims, int32_t n_dims, float lr,
                      ah_trainer **out);
void ah_trainer_destroy(ah_trainer *t);
int ah_trainer_set(ah_trainer *t, int32_t slot, const void *host, int64_t n);
int ah_trainer_get(ah_trainer *t, int32_t slot, void *host, int64_t n);
int ah_trainer_step(ah_trainer *t, int64_t batch, int32_t flags);
/* n consecutive steps (tensor.JIT's replay loop, tensor/jit.go:176-215, with the inputs left in place).
 * With AH_STEP_GRAPH the steps run as hipGraph launches of up to 16 steps each, each graph captured once
 * per (batch, flags, steps) and replayed: a graph launch has a fixed host and GPU cost, paid once per
 * graph rather than once per step. Without it, n eager steps. */
int ah_trainer_steps(ah_trainer *t, int64_t batch, int32_t flags, int32_t n);
/* Per-kernel probe: hipEvents around the index-th kernel launch of every following step. */
int ah_trainer_probe(ah_trainer *t, int32_t kernel_index);
/* Probe of launches first..last of every following step: one hipEvent before launch `first`, one after
 * launch `last`; last = first - 1 records the two events back to back (their own cost alone). Two spans
 * that differ by one launch give that launch's share of the step with the events' cost cancelled. */
int ah_trainer_probe_span(ah_trainer *t, int32_t first, int32_t last);
int ah_trainer_probe_read(ah_trainer *t, double *total_ms, int64_t *count);
int ah_trainer_kernel_count(ah_trainer *t, int64_t batch, int32_t *count);
/* Name of the index-th launch of a step, as counted by the last ah_trainer_kernel_count (NUL-terminated,
 * truncated to cap bytes). The reference's Benchmark reports per-kernel results by kernel
 * (backend/webgpu/benchmark.go); this names the trainer's launches for the same purpose. */
int ah_trainer_kernel_name(ah_trainer *t, int32_t index, char *buf, int32_t cap);

/* ── Checkpoint formats (host side; no device needed) ─────────────────────────
 * Readers for safetensors (tensor/safetensors/safetensors.go:150-434 Load / LoadTensors), NumPy .npy and
 * .npz with stored or deflated members (tensor/npy/npy.go:41-466 Load / LoadNPZ), decoding every tensor to f32 with the reference's
 * dtype policy (safetensors.go:21-35, npy.go:3-16): F32 exact, F64 -> f32, F16 / BF16 widened (safetensors),
 * integers by value with an error past 2^24, BOOL -> 0/1, any other dtype an error naming it; Fortran-order
 * arrays come back in C order. The decoded values are what a trainer uploads with ah_trainer_set. */
typedef struct ah_ckpt ah_ckpt;
int ah_ckpt_open(const char *path, ah_ckpt **out);   /* format from the file's magic bytes */
int32_t ah_ckpt_count(const ah_ckpt *c);
int ah_ckpt_entry(const ah_ckpt *c, int32_t i, const char **name, const char **dtype, int32_t *rank,
                  const int64_t **shape, int64_t *n_elems);
int ah_ckpt_read(const ah_ckpt *c, int32_t i, float *out, int64_t n);
void ah_ckpt_close(ah_ckpt *c);
/* Writer for F32 safetensors checkpoints as safetensors.Save writes them (safetensors.go:75-146): names
 * sorted, header JSON {"name":{"dtype":"F32","shape":[..],"data_offsets":[a,b]},..} padded with spaces to
 * a multiple of 8 bytes, data little-endian in name order. */
int ah_safetensors_save(const char *path, int32_t n, const char *const *names, const float *const *data,
                        const int64_t *const *shapes, const int32_t *ranks);

#ifdef __cplusplus
}
#endif
#endif
