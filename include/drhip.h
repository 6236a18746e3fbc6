/*
 * drhip.h -- C ABI of libdrhip.so, the device runtime under the DelayRepay
 * HIP fusion backend for AMD Instinct MI355X (gfx950).
 *
 * The reference's GPU backend (delayrepay/cuda.py) has no FFI of its own: it
 * reaches the device through CuPy (cupy.ElementwiseKernel -> NVRTC -> CUDA
 * driver launch, CuPy's memory pool, cupy.ndarray.get()).  This library is the
 * set of entry points a backend module needs in place of those CuPy services.
 * Each declaration names the reference call site whose CuPy service it
 * replaces.
 *
 * Conventions
 *   - plain C types only; device memory is passed as void* device addresses;
 *   - every function returning int returns 0 on success, otherwise a non-zero
 *     code (hipError_t, or 10000 + hiprtcResult for compiler errors, or a
 *     DRHIP_E* value below); drhip_last_error() then holds a message;
 *   - all work is issued on one library-owned stream, in order; a call
 *     returns once the work is queued unless stated otherwise;
 *   - not thread-safe: one host thread drives the library (the reference is
 *     single threaded as well: delayrepay/delayarray.py:27-32 keeps unguarded
 *     module globals).
 */
#ifndef DRHIP_H
#define DRHIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DRHIP_ENOTINIT 20001 /* drhip_init has not succeeded yet          */
#define DRHIP_EINVAL   20002 /* argument rejected before touching the GPU */
#define DRHIP_ERTC     10000 /* + hiprtcResult                            */

/* ---- life cycle --------------------------------------------------------- */

/* Select the device, create the stream, read device properties.  Idempotent.
 * Replaces the implicit CUDA context creation done by `import cupy`
 * (delayrepay/cuda.py:17). */
int drhip_init(int device);

/* Fixed facts about the device chosen by drhip_init. */
typedef struct drhip_device_info {
    char     name[128];
    char     arch[64];       /* gcnArchName, e.g. "gfx950:sramecc+:xnack-"  */
    int32_t  compute_units;
    int32_t  wavefront_size;
    int32_t  max_lds_bytes;  /* per workgroup                                */
    int32_t  l2_bytes;
    int64_t  total_mem;
    int32_t  clock_khz;
    int32_t  mem_clock_khz;
    int32_t  mem_bus_bits;
    int32_t  hiprtc_version; /* major * 1000 + minor of the run-time compiler   */
} drhip_device_info;
int drhip_device_info_get(drhip_device_info* out);

/* Thread-local message for the last non-zero return on this thread. */
const char* drhip_last_error(void);

/* ---- pooled device memory ----------------------------------------------
 * Replaces CuPy's default memory pool, from which cuda.py:96 `kern(*inputs)`
 * takes its output array and which frees on garbage collection.
 * Blocks are rounded up to a size class and recycled through per-class free
 * lists; nothing is returned to the driver until drhip_pool_trim().  Reuse is
 * safe without synchronisation because every kernel and copy runs on the one
 * library stream, in order. */
int drhip_malloc(void** dptr, size_t nbytes);
int drhip_free(void* dptr);

typedef struct drhip_pool_stats_t {
    uint64_t bytes_in_use;     /* handed out, class-rounded                 */
    uint64_t bytes_cached;     /* sitting in free lists                     */
    uint64_t bytes_peak;       /* high-water mark of in_use + cached        */
    uint64_t n_driver_allocs;  /* hipMalloc calls so far                    */
    uint64_t n_pool_hits;      /* drhip_malloc served from a free list      */
    uint64_t n_mallocs;        /* drhip_malloc calls so far                 */
} drhip_pool_stats_t;
int drhip_pool_stats(drhip_pool_stats_t* out);
/* Give every cached block back to the driver (synchronises first). */
int drhip_pool_trim(void);

/* ---- copies -------------------------------------------------------------
 * h2d replaces cupy.asarray / cupy.array on host data (delayarray.py:620-623
 * through cuda.fallback); d2h replaces cupy.ndarray.get() (delayarray.py:104)
 * and blocks until the bytes are in host memory; d2d is queued. */
int drhip_memcpy_h2d(void* dst_dev, const void* src_host, size_t nbytes);
int drhip_memcpy_d2h(void* dst_host, const void* src_dev, size_t nbytes);
int drhip_memcpy_d2d(void* dst_dev, const void* src_dev, size_t nbytes);
/* Fill nwords 32-bit (or 64-bit) words with a pattern, using a fill kernel
 * (no memset node, so the call is safe to record into a HIP graph). */
int drhip_fill32(void* dst_dev, uint32_t pattern, size_t nwords);
int drhip_fill64(void* dst_dev, uint64_t pattern, size_t nwords);
/* Plain streaming copy kernel (128-bit non-temporal loads and stores); used as
 * the measured ceiling of the memory system next to generated kernels and to
 * calibrate profiler byte counters.  nbytes must be a multiple of 16;
 * grid_blocks = 0 picks one run of 256 vectors per block. */
int drhip_copy_kernel(void* dst_dev, const void* src_dev, size_t nbytes,
                      unsigned grid_blocks);

/* Row-major C[m,n] = A[m,k] * B[k,n] in float (is_double = 0) or double, leading
 * dimensions in elements.  Replaces `_backend.fallback.dot` = cupy.dot -> cuBLAS
 * (delayarray.py:85) for matrix operands; eager, not part of the fused path.
 * Products with at least 64 rows and columns run on the matrix cores (128x128 tiles
 * of MFMA accumulators), smaller ones on a 64x64 vector-ALU tile. */
int drhip_matmul(int is_double, const void* a, const void* b, void* c, int64_t m, int64_t n,
                 int64_t k, int64_t lda, int64_t ldb, int64_t ldc);

/* Inclusive prefix sum of n contiguous elements; kind 0 float, 1 double, 2 int32,
 * 3 int64.  Replaces `_backend.fallback.cumsum` = cupy.cumsum (delayarray.py:558);
 * eager, not part of the fused path. */
int drhip_cumsum(int kind, const void* in_dev, void* out_dev, size_t n);

/* ---- operators of language models ----------------------------------------
 * No counterpart in the reference.  Device pointers and element strides of
 * (batch, head, row); the last dimension is dense.  Arguments that a GPU array
 * holds (lengths, positions ...) cannot be checked here: the kernels clamp
 * them to what the arrays hold.  Nothing is allocated: `work` is device memory
 * of at least the bytes that the *_work call of the same arguments gives (it is
 * only written before it is read within the call), so that the calls can be
 * captured. */

/* Attention of q[batch][hq][lq][d] to k, v[batch][hkv][lk][d] (hq a multiple of
 * hkv, d <= 128), float.  Row i stands at position start + i; key j counts for
 * it if j < lengths (lk without), with `causal` if also j <= position or
 * j < prefix, with `documents` if documents[j] = documents[position] (none at
 * positions outside the sequence).
 * Scores: scale q.k, with cap > 0 cap tanh(scale q.k / cap), with slopes less
 * slopes[head] |position - j|; |scale| and cap within 2^100, cap > 2^-100 if
 * positive.  o = softmax(scores) v, lse (may be NULL) the
 * logarithm of the sum of their exponentials; a row without keys gives zeros
 * and -inf.  drhip_attention_grad: dq, dk, dv from dout and the forward call's
 * o and lse. */
typedef struct drhip_attention_t {
    const float *q, *k, *v;
    float *o, *lse;               /* lse: dense [batch][hq][lq]                */
    const float* dout;            /* gradient only, with dq, dk, dv            */
    float *dq, *dk, *dv;
    const int32_t *lengths, *start, *prefix; /* [batch] or NULL                */
    const int32_t* documents;     /* [batch][lk] or NULL                       */
    const float* slopes;          /* [hq] or NULL                              */
    void* work;
    uint64_t work_bytes;
    int64_t q_stride[3], k_stride[3], v_stride[3], o_stride[3];
    int64_t dout_stride[3], dq_stride[3], dk_stride[3], dv_stride[3];
    int64_t documents_stride;
    int32_t batch, hq, hkv, lq, lk, d;
    int32_t causal;
    int32_t start_mode;           /* 0: start = length - lq, 1: start_value (or the array) */
    int32_t start_value, prefix_value;
    float scale, cap;
} drhip_attention_t;
int drhip_attention_work(const drhip_attention_t* a, int grad, uint64_t* bytes);
int drhip_attention(const drhip_attention_t* a);
int drhip_attention_grad(const drhip_attention_t* a);

/* Numbers of 64 bits as numbers of 32 that are equal where they are: y[batch][n] is
 * the place at which x[batch][n] first stands in its row (of documents for
 * attention).  `table`: device memory of batch rows of `slots` words, a power of
 * two of at least 2 n. */
typedef struct drhip_renumber_t {
    const int64_t* x;
    int32_t *y, *table;
    int64_t x_stride;             /* of rows                                   */
    int32_t batch, n, slots;
} drhip_renumber_t;
int drhip_renumber(const drhip_renumber_t* a);

/* y[n] = x[n] clamped to [low, high], numbers of 64 bits to 32 (of lengths and
 * their like). */
typedef struct drhip_clamp_t {
    const int64_t* x;
    int32_t* y;
    int64_t x_stride;
    int32_t n, low, high;
} drhip_clamp_t;
int drhip_clamp(const drhip_clamp_t* a);

/* Rotary positions of x[batch][heads][rows][d] (d <= 512), float or double: the
 * pair of elements number i < dims/2 turns by sign * position * frequency_i *
 * squeeze, frequency_i = 2^(i * step) or from the table, and is multiplied by
 * magnitude.  With a weight (weight_stride 0: [d], else [heads][d]) rows are first
 * divided by the root of their mean square + eps and multiplied by it.
 * With dweight the call is the gradient of the latter (sign -1): from x and dy, dx
 * goes to y and the weight's gradient, dense, to dweight. */
typedef struct drhip_rotary_t {
    const void* x;
    void* y;
    const void *weight, *dy;
    void* dweight;
    const void* positions;        /* int32 or int64 [batch or 1][rows]; NULL: first, first + 1 ... */
    const double* frequencies;
    void* work;
    uint64_t work_bytes;
    int64_t x_stride[3], y_stride[3], dy_stride[3];
    int64_t weight_stride, positions_stride, first;
    double step, squeeze, magnitude, sign, eps;
    int32_t batch, heads, rows, d, dims, d_pad; /* d_pad: d rounded up to 4    */
    int32_t interleaved, is_double, positions_wide;
} drhip_rotary_t;
int drhip_rotary_work(const drhip_rotary_t* p, uint64_t* bytes);
int drhip_rotary(const drhip_rotary_t* p);

/* One token for each row of logits[batch][vocabulary]: weights exp(logit /
 * temperature), the top_k largest of them (0: all), the first of those that
 * hold top_p of their weight, of these the ones of at least min_p of the
 * largest; the token is the first by number at which their sum exceeds
 * uniforms[row] of it.  temperature 0: the largest.  Equal logits: the lower
 * number is the larger.  A row without a logit above -inf gives -1.  Parameters:
 * an array of one for each row, or one for all.  `one` is the weight of the
 * largest as a whole number, at most 2^62 / vocabulary. */
typedef struct drhip_sample_t {
    const float* logits;
    const void* uniforms;         /* float or double [batch]                   */
    int64_t* tokens;
    const float *temperature, *top_p, *min_p;
    const int32_t* top_k;
    int64_t logits_stride;
    double temperature_all, top_p_all, min_p_all, one;
    int32_t top_k_all, batch, vocabulary, uniforms_wide;
} drhip_sample_t;
int drhip_sample(const drhip_sample_t* p);

/* The library's stream (a hipStream_t), for ordering work of other libraries
 * with it. */
int drhip_stream(void** stream);

/* ---- run-time compilation ----------------------------------------------
 * Replaces cupy.ElementwiseKernel(...) construction (cuda.py:35-43), i.e.
 * NVRTC + module load.  `src` is HIP C++ text holding one or more
 * `extern "C" __global__` functions.  The library always passes
 * --offload-arch=<device arch or DRHIP_ARCH>; `opts` are added after it.
 * On success *module is an opaque handle.  drhip_compile needs no GPU when
 * `module` is NULL: it then only compiles, which lets a build machine check
 * generated source; the code object can be fetched with drhip_code_get. */
int drhip_compile(const char* src, const char* name, const char* const* opts,
                  int nopts, void** module);
/* Code object of the most recent successful drhip_compile on this thread
 * (valid until the next compile).  For the on-disk kernel cache. */
int drhip_code_get(const void** code, size_t* nbytes);
/* Load a code object produced earlier by drhip_compile (disk-cache hit). */
int drhip_load_code(const void* code, size_t nbytes, void** module);
int drhip_module_unload(void* module);
int drhip_get_function(void* module, const char* kernel_name, void** func);
/* Compiler diagnostics of the most recent drhip_compile on this thread. */
const char* drhip_compile_log(void);

/* ---- launch -------------------------------------------------------------
 * Replaces `kern(*inputs)` (cuda.py:95-96).  `args` is the kernel's argument
 * block laid out exactly as the kernel's parameters (natural alignment, as a
 * C struct), `args_bytes` its size.  1-D grid of `grid_x` blocks of `block_x`
 * threads, `lds_bytes` of dynamic LDS. */
int drhip_launch(void* func, unsigned grid_x, unsigned block_x,
                 unsigned lds_bytes, const void* args, size_t args_bytes);

/* drhip_launch for a kernel that needs device scratch memory (the partial results a
 * reduction kernel hands to its finalising kernel), for callers that cannot allocate:
 * code under HIP graph capture, tight serving loops, harnesses that forbid hipMalloc.
 * It has no counterpart in the reference (whose reductions are CuPy library calls,
 * delayarray.py:516-518).  The call allocates nothing: the scratch memory is one static
 * device array of drhip_scratch_bytes() bytes (4 MiB) that every GPU the library runs on
 * holds until the process ends.  Its address on the current device is written into the
 * pointer slot at byte offset `scratch_arg_offset` of the argument block (a multiple of
 * 8; the slot's previous contents are ignored), then the kernel is launched exactly as
 * drhip_launch would.  The kernel may use the first `scratch_bytes` bytes; a request
 * above drhip_scratch_bytes(), or an argument block above DRHIP_MAX_ARGS_BYTES, is
 * refused with DRHIP_EINVAL.  All calls on a GPU share the array and it keeps the last
 * call's contents: a kernel must write what it later reads (nothing is cleared), work
 * queued through this library is ordered by its one stream, and users of the array that
 * overlap on one GPU by any other route race. */
#define DRHIP_MAX_ARGS_BYTES 4096
int drhip_launch_scratch(void* func, unsigned grid_x, unsigned block_x, unsigned lds_bytes,
                         const void* args, size_t args_bytes, size_t scratch_arg_offset,
                         size_t scratch_bytes);
size_t drhip_scratch_bytes(void);

/* ---- HIP graphs -----------------------------------------------------------
 * Capture the launches issued between begin and end into a graph and replay
 * them with one call: for launch-bound loops (small arrays, many sweeps).  The
 * reference has no counterpart (it launches kernel by kernel, cuda.py:96).
 * Between begin and end only drhip_launch, drhip_fill32/64 and
 * drhip_copy_kernel may be called (no allocation, copy or synchronisation);
 * captured kernels keep the device addresses they were recorded with. */
int drhip_graph_begin(void);
int drhip_graph_end(void** graph_exec);
int drhip_graph_launch(void* graph_exec);
int drhip_graph_destroy(void* graph_exec);

/* ---- synchronisation and timing ---------------------------------------- */
int drhip_sync(void);
int drhip_event_create(void** ev);
int drhip_event_destroy(void* ev);
int drhip_event_record(void* ev);            /* on the library stream      */
int drhip_event_sync(void* ev);
int drhip_event_done(void* ev, int* done);   /* 1 once the work before it is done */
int drhip_event_elapsed_ms(void* start, void* stop, float* ms);

/* Counters for the bench harness. */
typedef struct drhip_counters_t {
    uint64_t n_compiles;
    uint64_t n_code_loads;
    uint64_t n_launches;
    uint64_t compile_ns;     /* wall time spent inside hiprtc              */
} drhip_counters_t;
int drhip_counters(drhip_counters_t* out);

#ifdef __cplusplus
}
#endif
#endif /* DRHIP_H */
