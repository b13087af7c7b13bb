/* presk_hip.h -- the C ABI of the MI355X (gfx950) executor of Presk's realized
 * loop nests: a drop-in `KernelExec` for `--backend hip`.
 *
 * The reference's seam is `trait KernelExec` (crates/presk-kernel/src/host.rs:
 * 28-95), whose native implementations compile each `Kernel` once
 * (`trait KernelCompiler`, crates/presk-cranelift/src/lib.rs:48-53) into a
 * `KernelFn = unsafe extern "C" fn(bufs: *const *mut u8, lo: i64, hi: i64)`
 * (crates/presk-cranelift/src/lib.rs:38-42) and call it over a pointer table
 * [inputs..., output, overflow flag iff the kernel stores f16/e8m15]
 * (crates/presk-cranelift/src/lib.rs:1609-1629).  This ABI keeps that shape,
 * with device pointers and a HIP stream:
 *
 *   presk_hip_compile  <->  KernelCompiler::compile(&Kernel) -> KernelFn
 *   presk_hip_run      <->  the KernelFn call f(bufs, lo, hi)
 *   presk_hip_alloc/free/h2d/d2h/sync
 *                      <->  the host's `Buf`s made device-resident
 *                           (crates/presk-rt/src/lib.rs:760-915)
 *
 * A kernel arrives as its text (`impl Display for Kernel`,
 * crates/presk-kernel/src/ir.rs:495-595) plus the two facts the text does not
 * carry: its storage type (`Kernel::dtype`) and its lane width
 * (`Kernel::lanes`).
 *
 * Errors: every function returns 0 on success and a negative code otherwise;
 * presk_hip_last_error() then gives the message, which starts with the
 * reference's code: "E10001" for an executor error
 * (crates/presk-cranelift/src/lib.rs:34-36), "E7005" for a kernel whose
 * formats the executor does not compute (crates/presk-rt/src/lib.rs:567-591),
 * "E7007" for the overflow guard (crates/presk-kernel/src/host.rs:140-177).
 *
 * Threading: one host thread drives a device (as `KernelBackend` is
 * single-threaded, crates/presk-kernel/src/host.rs:256); launches are
 * asynchronous on the given stream, and a buffer is read on the host only
 * after presk_hip_sync on that stream.
 */
#ifndef PRESK_HIP_H
#define PRESK_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PRESK_HIP_OK 0
#define PRESK_HIP_ERR (-1)       /* E10001: executor or HIP error */
#define PRESK_HIP_REFUSED (-2)   /* E7005: formats not computed natively */
#define PRESK_HIP_OVERFLOW (-3)  /* E7007: a narrowing store overflowed */

/* How a kernel's reductions are ordered.
 * EXACT: every sum in index order, bit-identical to `--backend kernel`
 *        (ReductionOrder::Sequential, crates/presk-rt/src/lib.rs:251-285).
 * FAST:  contractions on MFMA tiles with f32 accumulation, a reassociating
 *        order the kernel's info names (the declared-order rule of
 *        crates/presk-rt/src/lib.rs:262-268); every other nest as in EXACT.  */
#define PRESK_HIP_EXACT 0
#define PRESK_HIP_FAST 1

typedef struct presk_hip_kernel presk_hip_kernel;

/* What a compiled kernel is: no counterpart in the reference beyond
 * `KernelExec::name` and the launch log (host.rs:317-321); used by the
 * harness to report the class chosen and the roofline of each launch. */
typedef struct {
    char kind[32];        /* "gemm", "rows", "generic", ... */
    char order[32];       /* "sequential", "mfma-k32", ... */
    int32_t guarded;      /* the pointer table ends with a u32 flag */
    int32_t n_inputs;
    int64_t split_bound;  /* the [lo,hi) range of presk_hip_run, or -1 */
    double flops;         /* algorithmic flops of one launch (2*I*J*K for a contraction) */
    double bytes;         /* algorithmic bytes: inputs once + output once, at storage width
                             (crates/presk-kernel/src/cost.rs:26-95) */
} presk_hip_info;

/* Selects the device and sets the executor up.  No counterpart in the
 * reference (its executors need none); must be called before any other
 * function that touches the device.  `device` -1 takes PRESK_HIP_DEVICE
 * (an ordinal; device 0 when unset).  The environment's other switches are
 * checked here, a malformed one failing the call (E10001):
 *   PRESK_HIP_MODE=exact|fast       every kernel compiled in that mode, whatever
 *                                   presk_hip_compile is asked (exact: the
 *                                   interpreter's order in every kernel);
 *   PRESK_HIP_GEMM_TILE=<bm>x<bn>[w8][/<splits>]
 *                                   contraction tiles (128 x 64/96/128, w8
 *                                   after 128x128 or 128x96 (f32) for eight
 *                                   waves; 256 x
 *                                   96/128 on f32 storage, 256 x 128/256 on
 *                                   16-bit) and k splits (1-64, single-entry
 *                                   contractions) in place of the planner's,
 *                                   where they apply; f32 operands and integer
 *                                   weights then multiply on the f32 MFMAs
 *                                   ("mfma-f32-k4"), whatever the planner's
 *                                   order was;
 *   PRESK_HIP_CACHE, PRESK_HIP_DUMP  the generated kernels' code-object cache
 *                                   and a directory to keep their sources in. */
int presk_hip_init(int device);

/* The message of the calling thread's last failed call ("" if none). */
const char *presk_hip_last_error(void);

/* KernelCompiler::compile (crates/presk-cranelift/src/lib.rs:48-53): reads the
 * kernel's text, chooses its HIP kernel, builds it.  `dtype` is "f64", "f32",
 * "bf16", "f16" or "e8m15"; `lanes` is Kernel::lanes; `mode` is
 * PRESK_HIP_EXACT or PRESK_HIP_FAST.  Refuses (PRESK_HIP_REFUSED) a kernel
 * whose formats are not its storage type's arithmetic (ir.rs:204-259), as
 * the native backend's `prepare` does (host.rs:416-434).  Integer weights
 * (`int8/<over>`, `int4/<over>..<end>`, BufKind::Quant, ir.rs:30) are
 * computed: each load is f32(q) * scale (crates/presk-rt/src/quant.rs:248-252).
 * After presk_hip_init, the kernel's code object is loaded here. */
int presk_hip_compile(const char *text, const char *dtype, int lanes, int mode, presk_hip_kernel **out);

/* The KernelFn call (crates/presk-cranelift/src/lib.rs:38-42): `bufs` holds
 * device pointers [inputs..., output, one f32 scales pointer per int8/int4
 * input in input order, overflow flag iff guarded] (lib.rs:1609-1629);
 * [lo, hi) is a range of the outermost loop's iterations when
 * presk_hip_kernel_info's split_bound is not -1 (Kernel::parallel_outer,
 * ir.rs:336-373): pieces that cover [0, split_bound) give the whole call's
 * bytes.  When split_bound is -1 the call is (0, 0).  `stream` is a hipStream_t (NULL: the
 * null stream).  Asynchronous: the overflow flag, a device u32 the caller
 * zeroes, is read after presk_hip_sync (E7007 if set). */
int presk_hip_run(const presk_hip_kernel *k, void *const *bufs, int64_t lo, int64_t hi, void *stream);

/* No counterpart in the reference: presk_hip_run for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc).  The same kernels and bits as
 * presk_hip_run; a class kernel's workspace (split-K partials, chunk sums,
 * mask bits) is the library's fixed scratch array of 64 MiB per device,
 * held from the library's load to the process's end, instead of memory
 * allocated on first use.  It calls no hipMalloc, hipFree or allocating
 * routine; a kernel compiled before presk_hip_init (no code object loaded
 * yet) or needing more scratch than 64 MiB is refused with an E10001 error.
 * Calls on one device share its scratch: calls that overlap on one device
 * (on several streams, or from several threads) race. */
int presk_hip_run_noalloc(const presk_hip_kernel *k, void *const *bufs, int64_t lo, int64_t hi, void *stream);

int presk_hip_kernel_info(const presk_hip_kernel *k, presk_hip_info *info);
void presk_hip_release(presk_hip_kernel *k);

/* The kernel's text as the executor read it, printed back as the reference
 * prints a kernel (ir.rs:495-595): the round trip that pins the reader.
 * Writes at most `cap` bytes including the terminator; returns the full
 * length, or a negative code. */
int64_t presk_hip_kernel_text(const presk_hip_kernel *k, char *buf, size_t cap);

/* Device memory and streams: the host's buffers made resident
 * (crates/presk-rt/src/lib.rs:760-915 holds them in host memory). */
int presk_hip_alloc(size_t bytes, void **dev);
int presk_hip_free(void *dev);
int presk_hip_h2d(void *dev, const void *host, size_t bytes, void *stream);
int presk_hip_d2h(void *host, const void *dev, size_t bytes, void *stream);
int presk_hip_memset(void *dev, int value, size_t bytes, void *stream);
int presk_hip_sync(void *stream);
int presk_hip_stream_create(void **stream);
int presk_hip_stream_destroy(void *stream);

/* Timing of launches with HIP events on the launch stream, in the shape of the
 * reference's per-launch `TimedExec` (crates/presk-kernel/src/cost.rs:719-780):
 * runs `k` `reps` times on `stream` after `warmup` untimed runs and stores the
 * mean milliseconds per launch. */
int presk_hip_time(const presk_hip_kernel *k, void *const *bufs, int64_t lo, int64_t hi, void *stream, int warmup,
                   int reps, double *ms_per_launch);

/* The host's conversion of a buffer at a kernel's edge, on the device: n
 * elements of type `from` at src stored as type `to` at dst, as
 * Buf::of(to, b.to_f64()) stores them (crates/presk-rt/src/lib.rs:868-876,
 * called at crates/presk-kernel/src/host.rs:793-829 when a mixed realization
 * hands a kernel a buffer of another type; the C export's presk_convert,
 * crates/presk-export-c/c/presk_rt.h:409-417).  Types "f64", "f32", "bf16",
 * "f16", "e8m15".  A buffer of the same type is copied as it is.  When `to` is
 * f16 or e8m15 and a finite value reaches its overflow threshold, *flag gets
 * bit 0 (if flag is not null): the host's E7007. */
int presk_hip_convert(const void *src, const char *from, void *dst, const char *to, int64_t n, uint32_t *flag,
                      void *stream);

/* One leaf of a `.psk.d` file decoded on the device, replacing the reader's
 * per-element Enc::decode (crates/presk-data/src/lib.rs:205-219, called from
 * `decode`, lib.rs:816-843) followed by Buf::of into the storage type.  `src`
 * holds the leaf's n elements as the file stores them (copied to device
 * memory); `enc` is the header's code: 0 f64, 1 f32, 2 bf16, 3 a format given
 * by its parameters, whose six header bytes `desc` points to (host memory;
 * Enc::of_description, lib.rs:143-166).  Each element is the exact f64 its
 * code denotes (Float::decode, crates/presk-format/src/lib.rs:460-476), stored
 * as type `to` stores an f64 (as presk_hip_convert does, overflow guard
 * included).  A description that is no format fails with E9002. */
int presk_hip_pskd_decode(const void *src, int enc, const uint8_t *desc, int64_t n, void *dst, const char *to,
                          uint32_t *flag, void *stream);
/* An `idx[bound]` leaf: n elements of the smallest unsigned integer holding
 * bound-1 (idx_width, crates/presk-data/src/lib.rs:289-296), little-endian,
 * widened to i64 at dst. */
int presk_hip_pskd_decode_idx(const void *src, uint64_t bound, int64_t n, int64_t *dst, void *stream);

/* A recorded launch sequence: a function body's kernels in the order the
 * host's call loop issues them (crates/presk-kernel/src/host.rs:887-1030 runs
 * each `let` of the body as one or more launches through `KernelExec::run`).
 * No counterpart in the reference's interface: a host that calls the same
 * body again and again (a training loop, a serving loop) records it once and
 * replays it.  `presk_hip_batch_add` copies the kernel's pointer table (its
 * inputs, output and, for a guarded kernel, the flag); the kernels and
 * buffers must outlive the batch.  `presk_hip_batch_graph` makes every later
 * `presk_hip_batch_run` one HIP graph launch of the whole sequence (lazy
 * module loads and workspaces are done first, outside the capture, and
 * nothing the sequence launches is a memset); without it each run issues the
 * launches one by one.  Adding a launch discards the graph. */
typedef struct presk_hip_batch presk_hip_batch;
int presk_hip_batch_create(presk_hip_batch **out);
int presk_hip_batch_add(presk_hip_batch *b, const presk_hip_kernel *k, void *const *bufs, int64_t lo, int64_t hi);
/* An edge conversion (presk_hip_convert) as a step of the sequence. */
int presk_hip_batch_add_convert(presk_hip_batch *b, const void *src, const char *from, void *dst, const char *to,
                                int64_t n, uint32_t *flag);
/* A training dropout mask (presk_hip_dropout_mask) as a step of the sequence:
 * the key is read from device memory at each run, so a replayed graph draws
 * the mask of whatever key the host last wrote there. */
int presk_hip_batch_add_dropout(presk_hip_batch *b, const void *key, double rate, const char *type, int64_t n,
                                void *dst);
int presk_hip_batch_graph(presk_hip_batch *b);
/* presk_hip_batch_graph with independent steps on up to `branches` (1-8)
 * parallel branches of the graph: a step follows every earlier step that
 * writes bytes it reads or writes, or reads bytes it writes (the overflow
 * flag aside: its stores commute), and every earlier launch of the same
 * compiled kernel (one workspace a kernel).  1 is presk_hip_batch_graph.
 * More than one branch is switched off in this build (E10001): a branched
 * capture ended in a host segmentation fault whose cause is not found. */
int presk_hip_batch_graph_branches(presk_hip_batch *b, int branches);
int presk_hip_batch_run(presk_hip_batch *b, void *stream);
void presk_hip_batch_release(presk_hip_batch *b);

/* A training dropout mask on the device: `DropoutMask` with training on
 * (crates/presk-kernel/src/host.rs:1610-1627 calling dropout_mask,
 * host.rs:1893-1926, which draws it on the host's workers).  n elements of
 * type "f64", "f32", "bf16", "f16" or "e8m15": element e is 1/(1-rate) where
 * the key's e-th uniform draw (uniform01 of its ChaCha20Rng stream read from
 * word 2e, crates/presk-interp/src/key.rs:43-55) is below 1-rate, else 0,
 * rounded as Buf::of rounds it -- the host's bits.  `key`: the 32-byte key in
 * device memory (4-byte aligned).  A rate outside [0, 1) is E7001, as the
 * host refuses it. */
int presk_hip_dropout_mask(const void *key, double rate, const char *type, int64_t n, void *dst, void *stream);

/* The losses of a large vocabulary and their gradients; no counterpart among
 * the reference's nests, where a loss is `cross_entropy` over logits in memory
 * (crates/presk-kernel/src/lower.rs:1459-1488).
 *
 * Of logits z [rows, vocab], with u = z / temperature:
 *   lse[r]  = log sum_v exp(u[r, v])
 *   loss[r] = T^2 * sum_v t[r, v] * (log t[r, v] - u[r, v] + lse[r])
 *   mean    = the counted rows' mean loss (0 when none counts), and their number
 *   dz[r]   = ct[r] * T * (exp(u[r] - lse[r]) - t[r])
 * The target t[r] of `top` 0 is one column, index[r] (temperature 1): the
 * softmax cross entropy.  With `top` k of 1 to 1024 it is the softmax of a
 * teacher's k logits at the same temperature, teacher[r, j] at column
 * index[r, j]; columns named twice have both weights.
 * A slot whose index is negative, or whose teacher logit is -inf, is unused; a
 * row with no used slot does not count: its loss and its row of dz are 0,
 * whatever its logits are.  A slot at or past `vocab` makes its row's loss and
 * cotangent NaN.  `ct` null: the mean's gradient, ct[r] = 1 / count.
 * Given and teachers' logits may be the type's lowest value (a mask): a row of
 * nothing else is uniform, in the value and in both together; the gradient
 * alone knows such a row by its f32 lse, in which its log sum is lost.
 *
 * presk_hip_head_loss: z = x . w with x [rows, model] and w [model, vocab], or
 * [vocab, model] when `tied`.  The logits are the workspace's: value and
 * gradient in one call keep up to 4 GiB of them in f32, past that, and for
 * either alone, they come in pieces of the vocabulary.  Gradients dx = dz . w^T and dw = x^T . dz, either
 * of which may be null.  The products accumulate in f32; in 16-bit storage the
 * factor ct[r] * (exp(u[r] - lse[r]) - t[r]) of dz is rounded to the storage type
 * before them (by a power of two in f16's range; of up to 64 rows what the
 * rounding left enters too, rounded itself), T and the mean's 1 / count come after.
 * A row of x that does not count still enters dw times zero, so it must be
 * finite.
 * presk_hip_distill: z = x, given (model 0, w null, top >= 1); dx is dz.
 *
 * `what`: PRESK_HIP_LOSS_VALUE writes loss, lse (f32 [rows]) and mean (f32 [2]),
 * those that are not null.  PRESK_HIP_LOSS_GRAD writes the gradients from the
 * forward's lse and, with ct null, its mean.  Both: value and gradients in one
 * call.  f16 outputs that overflow set bit 0 of *flag (if flag is not null), as
 * a guarded nest's stores do.
 * `work`: device memory of presk_hip_loss_workspace bytes (from the sizes and
 * the nullness of the pointers alone), 16-byte aligned, this call's until it
 * has run; nothing in it is kept between calls.  Every buffer is whole and
 * row-major; an output may not meet another buffer.  Nothing is allocated, and
 * only kernels are launched, so the calls may be captured.
 * Storage types f32, bf16 and f16 (others are E7005); rows from 0, model and
 * vocab below 2^22 (vocab of given logits below 2^30), and in f32 rows * model
 * and model * vocab below 2^31. */
typedef struct {
    const char* dtype;
    int64_t rows, model, vocab, top;
    int32_t tied;
    double temperature;
    const void* x;
    const void* w;
    const int64_t* index;
    const void* teacher;
    float* loss;
    float* lse;
    float* mean;
    const float* ct;
    void* dx;
    void* dw;
    uint32_t* flag;
    void* work;
    size_t work_bytes;
} presk_hip_loss;

#define PRESK_HIP_LOSS_VALUE 1
#define PRESK_HIP_LOSS_GRAD 2

/* The workspace of presk_hip_head_loss (model >= 1) or presk_hip_distill (model
 * 0) with these arguments; `work` and `work_bytes` are not read. */
int presk_hip_loss_workspace(const presk_hip_loss* a, int what, size_t* bytes);
int presk_hip_head_loss(const presk_hip_loss* a, int what, void* stream);
int presk_hip_distill(const presk_hip_loss* a, int what, void* stream);
/* Either as a step of a recorded sequence: the arguments are copied, the
 * buffers (the workspace among them) must outlive the batch. */
int presk_hip_batch_add_head_loss(presk_hip_batch* b, const presk_hip_loss* a, int what);
int presk_hip_batch_add_distill(presk_hip_batch* b, const presk_hip_loss* a, int what);

/* Attention of grouped heads without its weights in memory, and its gradients; no
 * counterpart among the reference's nests, where it is `ein`, `div`, `softmax` and
 * `ein` over weights in memory (crates/presk-kernel/src/lower.rs:250-303).
 *
 * Of queries q [batch, q_len, heads, head_dim] and keys and values k, v [batch,
 * k_len, kv_heads, head_dim], head h reading key head h / (heads / kv_heads):
 *   s[i, j] = scale * (q[i] . k[j]) over the keys that query i may read
 *   lse[i]  = log sum_j exp(s[i, j])              (-inf where it reads none)
 *   o[i]    = sum_j exp(s[i, j] - lse[i]) v[j]    (0 where it reads none)
 * and, of o's cotangent dout, with p = exp(s - lse):
 *   dv[j] = sum_i p[i, j] dout[i],  ds[i, j] = p[i, j] (dout[i] . v[j] - dout[i] . o[i])
 *   dq[i] = scale sum_j ds[i, j] k[j],  dk[j] = scale sum_i ds[i, j] q[i]
 * dk and dv summed over the heads of their group as well.
 * Query i of sequence b stands at position first[b] + i among the keys.  It may
 * read key j below lens[b] (null: k_len; taken into [0, k_len]) where
 *   causal:         j <= first[b] + i, and with a window also j > first[b] + i - window;
 *   mask_cols > 0:  j < first[b], or mask[b, i, j - first[b]] is not 0, whose
 *                   columns end at mask_cols (a tree of drafted tokens over a
 *                   cache; a mask of all keys has first 0 and k_len columns);
 *   neither:        always.
 * `first` null: k_len - q_len (the queries are the last keys), of a mask k_len -
 * mask_cols.  A key at or past lens[b] is not read, whatever it holds, and its
 * rows of dk and dv are 0; any other enters the sums of queries that may not read
 * it times 0, so it must be finite, also where no query reads it.
 * A tensor's element (b, i, h, d) is at p + b * batch + i * seq + h * head + d,
 * strides in elements and not negative, those of an input over batch or heads 0
 * where it is shared.  Rows of whole 16-byte vectors (address, strides and
 * head_dim) are loaded as such, others element by element.
 * Products accumulate in f32, and so do the sums of a softmax.  In 16-bit storage
 * the weights p and their cotangents ds are rounded to the storage type before
 * the products they enter, ds with what that rounding left as a second term where
 * queries read fewer than 64 keys or a mask says which; in f16 ds times a power of
 * two, 1 or more, that keeps small ones' bits and is taken out of the sums.  f32
 * elements enter as three bf16 parts, which are all of one of 2^-110 or more (a
 * smaller one may lose 2^-134), and six of their nine products (the rest is below
 * 2^-24); one that is infinite, or above 0x1.ffp127, gives NaN.
 *
 * `what`: PRESK_HIP_ATTN_VALUE writes o and, where it is not null, lse (f32 [batch,
 * heads, q_len]).  PRESK_HIP_ATTN_GRAD writes those of dq, dk and dv whose p is
 * not null from the forward's o and lse.  f16 outputs that overflow set bit 0 of
 * *flag (if flag is not null), of gradients any that is not finite: where ds
 * overflows they are not, whatever their sums would be.
 * `work`: device memory of presk_hip_attention_workspace bytes (from the sizes
 * alone), 16-byte aligned, this call's until it has run; nothing in it is kept
 * between calls.  An output may not meet another buffer (tensors whose rows lie
 * between each other's do not).  Nothing is allocated, and only kernels are
 * launched, so the calls may be captured; lens, first and mask are read then.
 * Storage types f32 (head_dim to 128), bf16 and f16 (to 256), others are E7005;
 * q_len, k_len, mask_cols and window below 2^28, a mask of batch * q_len * mask_cols
 * below 2^35 (of lengths in whole 32s); a row's stride (seq) at least head_dim
 * elements and below 2^24 bytes, of a single row anything from 0 to 2^40. */
typedef struct {
    void* p;
    int64_t batch, seq, head;
} presk_hip_heads;

typedef struct {
    const char* dtype;
    int64_t batch, heads, kv_heads, q_len, k_len, head_dim, window, mask_cols;
    int32_t causal;
    double scale;
    presk_hip_heads q, k, v, o, dout, dq, dk, dv;
    float* lse;
    const int64_t* lens;
    const int64_t* first;
    const uint8_t* mask;
    int64_t mask_batch, mask_row;
    uint32_t* flag;
    void* work;
    size_t work_bytes;
} presk_hip_attn;

#define PRESK_HIP_ATTN_VALUE 1
#define PRESK_HIP_ATTN_GRAD 2

int presk_hip_attention_workspace(const presk_hip_attn* a, int what, size_t* bytes);
int presk_hip_attention(const presk_hip_attn* a, int what, void* stream);
/* As a step of a recorded sequence: the arguments are copied, the buffers (the
 * workspace among them) must outlive the batch. */
int presk_hip_batch_add_attention(presk_hip_batch* b, const presk_hip_attn* a, int what);

/* The norm of each head of the queries and keys and their rotation by position in
 * one pass, and its gradients; among the reference's nests the rotation is `slice`,
 * `cos`, `sin`, products and `concat` (examples/coverage/llama.psk:36-48).
 *
 * Of a head's x (q [batch, seq, heads, head_dim] and k [.., kv_heads, ..]; kv_heads 0:
 * q alone), with `norm`:  u = g * x / sqrt(mean(x^2) + eps), gains gq for every head
 * of q and gk for those of k ([head_dim], null: ones); without it u = x.  Of the first
 * `rotary` elements of u, pair r turns by at[b, i] * freq[r] (f64 radians, freq
 * [rotary / 2], at i64 [batch, seq], null: i):
 *   y0 = u0 cos - u1 sin,  y1 = u1 cos + u0 sin
 * pair r being elements r and r + rotary / 2, or with `even` 2 r and 2 r + 1.  The
 * others of y are those of u.
 * PRESK_HIP_ROT_VALUE writes yq and yk (which may be q and k themselves);
 * PRESK_HIP_ROT_GRAD, from their cotangents dyq and dyk and, with `norm`, q and k,
 * writes dq and dk (which may be dyq and dyk) and those of dgq and dgk ([head_dim])
 * that are not null.  Sums in f32, angles in f64 (so that the cosine and sine of one
 * of 2^30 radians are within 2^-23 of those of its f64 product).  f16 outputs
 * that overflow set bit 0 of *flag (if flag is not null).  Tensors, `work` (null and 0
 * bytes do but for a gradient with `norm`), streams and graphs as
 * presk_hip_attention's. */
typedef struct {
    const char* dtype;
    int64_t batch, seq, heads, kv_heads, head_dim, rotary;
    int32_t norm, even;
    double eps;
    presk_hip_heads q, k, yq, yk, dyq, dyk, dq, dk;
    const double* freq;
    const int64_t* at;
    const void* gq;
    const void* gk;
    void* dgq;
    void* dgk;
    uint32_t* flag;
    void* work;
    size_t work_bytes;
} presk_hip_rot;

#define PRESK_HIP_ROT_VALUE 1
#define PRESK_HIP_ROT_GRAD 2

int presk_hip_head_rotary_workspace(const presk_hip_rot* a, int what, size_t* bytes);
int presk_hip_head_rotary(const presk_hip_rot* a, int what, void* stream);
int presk_hip_batch_add_head_rotary(presk_hip_batch* b, const presk_hip_rot* a, int what);

/* Seeded synthetic values written in place: n elements mean + std * z of
 * type "f32", "bf16" or "f16", z ~ N(0, 1) a function of (seed, element
 * index) alone (a splitmix64 hash and Box-Muller in f32).  Stands in for the
 * host's parameter initialization (`Normal` and `ones` are host primitives,
 * crates/presk-kernel/src/host.rs:1476; their draws come from ChaCha20 keys,
 * crates/presk-interp/src/run.rs:56-100) where a model's parameters are too
 * large to draw on the host and copy: the values are seeded N(0, std) but not
 * the reference's draws.  std = 0 fills the constant `mean`. */
int presk_hip_fill_normal(void *dst, const char *type, int64_t n, uint64_t seed, double mean, double std, void *stream);

/* A measurement aid with no counterpart in the reference: the matrix cores'
 * rate measured on this device, reported beside the vendor's nominal peak.
 * One timed launch (after an untimed one) of independent MFMA loops, eight
 * waves on every CU, each wave `iters` rounds of eight MFMAs: `type` "bf16"
 * (32x32x16) or "f32" (16x16x4).  *ms the launch's duration (HIP events on
 * `stream`), *flops the flops it performed. */
int presk_hip_mfma_probe(const char *type, int64_t iters, void *stream, double *ms, double *flops);

/* Self-test of the device's scalar functions over a domain block: the digest
 * (sum of splitmix64 finalizers of (i << 32 | out_i)) of function `fn` over
 * inputs [lo, hi), as tests/golden/digests.json holds the reference's.  For
 * fn 50 (expf) and 51 (erff) the result is instead the largest distance in
 * units in the last place between FAST mode's function and the
 * interpreter's over the inputs, and for fn 60 / 61 the count of inputs
 * where the two differ; fn 70-77 count the f32 dividends (the inputs' bit
 * patterns) whose quotient by one of eight fixed divisors through the
 * printed nests' division by a constant differs from the correctly rounded
 * division.  No counterpart in the reference; for the exhaustive device
 * checks. */
int presk_hip_scalar_digest(int fn, uint64_t lo, uint64_t hi, uint64_t *digest);

#ifdef __cplusplus
}
#endif
#endif
