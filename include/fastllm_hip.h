/*
 * fastllm_hip.h -- C-ABI of the MI355X (gfx950) quantized-matvec backend.
 *
 * Drop-in for the reference runtime's CUDA execution path of the quantized
 * decode hot path (qdox-labs/fast-llm): the ACT_Q8 / STREAM_DOT /
 * STREAM_DOT_IDX task kinds and the GGUF Q8_0 / Q4_K / Q6_K row-dots behind
 * them.  Plain C types only: device pointers are void* / float*, streams and
 * events are opaque void* (hipStream_t / hipEvent_t), sizes are integers.
 *
 * Every entry point returns FLH_OK (0) or a negative FLH_ERR_* code and
 * records a message readable with flh_last_error() (per calling thread).
 * The reference aborts on every error (src/runtime/gpu_exec.cu:15-17,
 * src/runtime/graph.cpp:100-103); a host wrapper that wants that behaviour
 * aborts on a non-zero return.
 *
 * Numerics contract: with fast=1 and the reference default masks, every
 * STREAM_DOT output is BITWISE equal to the reference CPU int8 path
 * (src/runtime/kernels.h:1002-1258 on x86: fl_dot_i8_q8_0, fl_dot_i8k_q4_K,
 * fl_dot_i8k_q6_K), ACT_Q8 bytes equal fl_exec_act_q8, and flh_dequant
 * equals dequant_chunk (src/runtime/kernels.h:162-242).
 */
#ifndef FASTLLM_HIP_H
#define FASTLLM_HIP_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------- codes -- */
enum {
    FLH_OK = 0,
    FLH_ERR_ARG = -1,          /* invalid argument (freeze()-style validation) */
    FLH_ERR_HIP = -2,          /* HIP runtime error */
    FLH_ERR_UNSUPPORTED = -3,  /* task kind / format / shape not implemented */
    FLH_ERR_NOMEM = -4,        /* arena exhausted or hipMalloc failed */
    FLH_ERR_STATE = -5,        /* flh_init not called / no device */
    FLH_ERR_IO = -6,           /* file missing or unreadable (GGUF) */
    FLH_ERR_FORMAT = -7        /* malformed GGUF file */
};

/* TaskKind values (include/fastllm/fastllm.h:19-45), stable. */
enum {
    FLH_TASK_STREAM_DOT = 0, FLH_TASK_MERGE = 1, FLH_TASK_SIGNAL = 2,
    FLH_TASK_ACT_Q8 = 3, FLH_TASK_STREAM_DOT_IDX = 4, FLH_TASK_RMSNORM = 5,
    FLH_TASK_ADD2 = 6, FLH_TASK_ROPE_DS2 = 7, FLH_TASK_KV_APPEND = 8,
    FLH_TASK_ATTN_HEAD = 9, FLH_TASK_ROUTER_SEL = 10, FLH_TASK_SILU_MUL = 11,
    FLH_TASK_WMERGE = 12
};

/* Fmt values (include/fastllm/fastllm.h:56-57), stable. */
enum {
    FLH_FMT_F32 = 0, FLH_FMT_Q8_0 = 1, FLH_FMT_Q5_0 = 2, FLH_FMT_Q4_K = 3,
    FLH_FMT_Q6_K = 4, FLH_FMT_IQ2_XXS = 5, FLH_FMT_IQ3_XXS = 6
};

/* Max activation columns per multi-column tile (fastllm.h:61 kMaxDotCols). */
#define FLH_MAX_DOT_COLS 16u

/*
 * Task record, byte-for-byte the layout of fastllm::Task
 * (include/fastllm/fastllm.h:65-97; enum class members are uint8_t), so a
 * frozen graph's task table can be passed as-is.  Pointers w / x / y / aux
 * are DEVICE pointers here (the reference uses unified memory), except that
 * for ROUTER_SEL / SILU_MUL / WMERGE aux points to a HOST-readable param
 * block (flh_router_p etc.) whose own pointers are device pointers.
 */
typedef struct __attribute__((aligned(128))) flh_task {
    uint32_t id;
    uint8_t kind;              /* FLH_TASK_* */
    uint8_t affinity;
    uint8_t fmt;               /* FLH_FMT_* */
    uint16_t n_consumers;
    uint32_t consumers[6];
    const void * w;
    uint64_t w_bytes;
    const void * x;
    void * y;
    uint32_t rows, cols;
    int32_t dep_init;
    int32_t dep_count;
    uint32_t epoch;
    uint64_t handoff_ts;
    const void * aux;          /* STREAM_DOT_IDX: device u32 expert-id slot */
    uint64_t aux2;             /* STREAM_DOT_IDX: expert stride in bytes */
    uint32_t nx, xstride, ystride;
} flh_task;

/* Decode-op param blocks, layouts of RmsNormP / RouterP / SiluMulP / WmergeP
 * (src/runtime/decode_params.h:23-29, 68-97). */
typedef struct flh_rmsnorm_p {
    const float * wnorm; const float * x; float * y; float eps; uint32_t n;
} flh_rmsnorm_p;
typedef struct flh_router_p {
    const float * logits; uint32_t * ids; float * gates;
    uint32_t n_expert, top_k, norm; float scale;
} flh_router_p;
typedef struct flh_silu_mul_p {
    const float * gate; const float * up; float * h; uint32_t n;
} flh_silu_mul_p;
typedef struct flh_wmerge_p {
    const float * parts; const float * gates; const float * add1;
    const float * add2; float * y; float scale; uint32_t n_parts, n, n_full;
} flh_wmerge_p;

/* ------------------------------------------------------------- runtime -- */
/* Last error message of the calling thread ("" if none). */
const char * flh_last_error(void);

/* Select and initialise a device; must precede every call below that touches
 * the GPU.  Replaces the device setup inside gpu_start()
 * (src/runtime/gpu_exec.cu:457-496; prototype runtime_internal.h:292).
 * Each call also (re-)reads the launch-tuning overrides FLH_* from the
 * environment (development sweeps; the defaults are the measured best); no
 * launch reads the environment itself. */
int flh_init(int device);

/* Device facts: compute units, HBM bytes, wave size, name. */
int flh_device_info(int * num_cus, size_t * hbm_bytes, int * wave_size,
                    char * name, size_t name_len);

/* Launch plan of the multi-column matrix-core dot for a Q4_K matrix of
 * rows x cols with nx activation columns on this device: out[0] = K halves,
 * out[1] = activations carried in the chunk DMA, out[2] = rows per batch,
 * out[3] = ring depth.  FLH_ERR_UNSUPPORTED if that kernel does not take the
 * shape.  No counterpart in the reference (whose multi-column kernel has one
 * plan): a query for tests and tuning, launches nothing. */
int flh_mfma_plan(uint32_t rows, uint32_t cols, uint32_t nx, uint32_t * out);

/* Reference default dispatch masks for the CPU int8 path this backend
 * matches (src/runtime/kernels.h:920,937). */
void flh_default_masks(uint32_t * i8_mask, uint32_t * i8k_mask);

/* Row bytes of a weight row and the activation buffer size with both q8
 * appendices (src/runtime/quants.h:97-99, 326-330). */
uint64_t flh_row_bytes(int fmt, uint32_t cols);
size_t flh_x_alloc_bytes(uint32_t cols);

/* ------------------------------------------------------------- memory -- */
/* Device bump arena over one hipMalloc: replaces Arena::create's
 * cudaMallocManaged arena (src/runtime/arena.cpp:54-74).  Allocations are
 * never freed individually; destroy releases everything. */
typedef struct flh_arena flh_arena;
int flh_arena_create(size_t bytes, flh_arena ** out);
int flh_arena_alloc(flh_arena * a, size_t bytes, size_t align, void ** out);
size_t flh_arena_used(const flh_arena * a);
int flh_arena_destroy(flh_arena * a);

/* Plain device buffers (outside any arena). */
int flh_malloc(size_t bytes, void ** out);
int flh_free(void * p);
/* Pinned host memory (hipHostMalloc): host-readable and device-visible; the
 * place for the decode-op param blocks a task table points to (see
 * flh_exec_tasks).  No counterpart in the reference, whose managed arena
 * is host-readable as it is (src/runtime/arena.cpp:54-63). */
int flh_host_alloc(size_t bytes, void ** out);
int flh_host_free(void * p);
int flh_upload(void * dst_dev, const void * src_host, size_t n, void * stream);
int flh_download(void * dst_host, const void * src_dev, size_t n, void * stream);
/* device-to-device copy of n bytes on a stream (asynchronous) */
int flh_copy(void * dst_dev, const void * src_dev, size_t n, void * stream);
/* zero n bytes with a fill kernel (safe inside HIP graph capture) */
int flh_zero(void * dst_dev, size_t n, void * stream);

/* ------------------------------------------------------------ streams -- */
/* Replaces gpu_make_stream / gpu_stop_sync (src/runtime/gpu_exec.cu:387,498).
 * Streams are created at default priority. */
int flh_stream_create(void ** out);
int flh_stream_sync(void * stream);
int flh_stream_destroy(void * stream);
int flh_event_create(void ** out);
int flh_event_record(void * event, void * stream);
int flh_event_elapsed_ms(void * start, void * stop, float * ms);
int flh_event_destroy(void * event);

/* HIP graph capture of work issued on one stream (replaces the reference's
 * persistent-kernel launch amortisation, src/runtime/gpu_exec.cu:156-344,
 * for a frozen graph: capture once, replay per token).  Every kernel of
 * this library is capture-safe (no hipMemsetAsync, no host syncs).  The
 * handle is this library's own: launch and destroy it here.
 *
 * A replay is one operation of its stream: work that other threads issue there
 * through this library comes before or after all of it.  On a stream of
 * flh_stream_create a short chain of kernels (at most 5, 7 with 0.5 MiB of
 * weights each on average, 16 with 12 MiB) is replayed kernel by kernel (less idle
 * time on the device; 2.6 to 4 us of the caller's time per kernel); a replay of it that
 * fails may have run in part.  On any other stream, and for any other graph, a replay is
 * the runtime's own graph launch.  What other code issues there directly (a HIP call on the
 * handle) from another thread at the same time may fall between the kernels of either. */
int flh_graph_capture_begin(void * stream);
int flh_graph_capture_end(void * stream, void ** graph_exec);
int flh_graph_launch(void * graph_exec, void * stream);
int flh_graph_destroy(void * graph_exec);

/* ---------------------------------------------------------------- ops -- */
/* ACT_Q8 (TaskKind 3; fl_exec_act_q8, src/runtime/quants.h:404-416; GPU
 * gact_q8, src/runtime/kernels_gpu.h:881-891): for each of nx columns
 * x_p = x + p*xstride (16-B aligned, fl_x_alloc_bytes(cols) bytes each),
 * write the q8_1 appendix at y_q81 + p*xstride floats (NULL = the canonical
 * fl_xq_of(x_p, cols)) and the q8_K appendix at fl_xqk_of(x_p, cols).
 * nx > 1: columns are quantised at once, so xstride * 4 >= fl_x_alloc_bytes
 * (cols) (FLH_ERR_ARG otherwise). */
int flh_act_q8(float * x, void * y_q81, uint32_t cols, uint32_t nx,
               uint32_t xstride, void * stream);

/* STREAM_DOT / STREAM_DOT_IDX tile (TaskKind 0/4; exec_task_block,
 * src/runtime/gpu_exec.cu:64-140, exec_task_cpu, src/runtime/kernels.h:
 * 1002-1258):  y[p*ystride + r] += dot(W[r], x + p*xstride), r < rows,
 * p < nx (0 means 1), W = w + (id_slot ? *id_slot * estride : 0) with the
 * id read ON THE DEVICE.  Validation as Graph::freeze
 * (src/runtime/graph.cpp:84-90): cols % block == 0, w_bytes == rows *
 * row_bytes, id_slot => estride != 0; and, since the columns run at
 * once, nx > 1 => ystride >= rows (overlapping outputs: FLH_ERR_ARG).
 * Alignment: x, y 4 bytes; w and estride 4 bytes for F32 / Q4_K, 2 bytes for
 * the 2-byte block formats (a row tile of rows 2 mod 4 bytes long).
 * fast = 0: canonical fp32 dequant-dot (fl_dot_row_any order, bitwise);
 * fast = 1: q8_K path for K formats whose bit is in i8k_mask, else q8_1
 * path for formats in i8_mask, else the "fast" fp32 dequant order
 * (dot_row_fast / dot_row_fast_q8_0 / dot_row_fast_dequant; F32 weights
 * always), exactly as exec_task_cpu.  cols = 0: every row's dot is 0.
 * int8 paths read the appendices written by flh_act_q8. */
int flh_stream_dot(int fmt, const void * w, uint64_t w_bytes, uint32_t rows,
                   uint32_t cols, const float * x, float * y, uint32_t nx,
                   uint32_t xstride, uint32_t ystride, const uint32_t * id_slot,
                   uint64_t estride, int fast, uint32_t i8_mask,
                   uint32_t i8k_mask, void * stream);

/* ACT_Q8 immediately followed by its STREAM_DOT consumer (the pair every
 * int8 tile of the reference graph builder emits, src/model/decoder.cpp:
 * 874-880,899-906), fused into one launch when the tile takes the q8_K path:
 * the kernel quantises x itself, workgroup 0 still writes both appendices,
 * and every output bit equals flh_act_q8 followed by flh_stream_dot (which is
 * what runs for any other format / mode).  No reference counterpart: the
 * reference always runs the two tasks separately. */
int flh_act_q8_stream_dot(int fmt, const void * w, uint64_t w_bytes, uint32_t rows,
                          uint32_t cols, float * x, float * y, uint32_t nx,
                          uint32_t xstride, uint32_t ystride,
                          const uint32_t * id_slot, uint64_t estride, int fast,
                          uint32_t i8_mask, uint32_t i8k_mask, void * stream);

/* RMSNORM of the column x (fl_op_rmsnorm, src/runtime/decode_params.h:101-106)
 * into xn -- fp32 y followed by its ACT_Q8 appendices, as flh_rmsnorm_act_q8
 * writes them with write_app = 1 -- then the single-column dot of it,
 * y[r] += dot(W[r], ACT_Q8(xn)) as flh_stream_dot: the decoder's
 * norm -> quant -> matvec chain (src/model/decoder.cpp:874-880; the tasks
 * RMSNORM, ACT_Q8, STREAM_DOT).  A Q4_K dot on the int8 path with at most
 * 8192 columns runs all three in one launch; anything else runs
 * flh_rmsnorm_act_q8 then flh_stream_dot.  The results are those of the two
 * calls, bit for bit.  x, wnorm and xn 16-byte aligned; xn must not overlap x. */
int flh_rmsnorm_stream_dot(int fmt, const void * w, uint64_t w_bytes, uint32_t rows,
                           uint32_t cols, const float * x, const float * wnorm, float eps,
                           float * xn, float * y, int fast, uint32_t i8_mask,
                           uint32_t i8k_mask, void * stream);

/* Execute a task table in array order on one stream (replaces the persistent
 * executor's per-task dispatch, exec_task_block, src/runtime/gpu_exec.cu:
 * 64-140, for a topologically ordered table such as run_serial walks,
 * src/runtime/graph.cpp:116-148).  Supported kinds: STREAM_DOT,
 * STREAM_DOT_IDX, ACT_Q8, MERGE, SIGNAL, RMSNORM, ROUTER_SEL, SILU_MUL,
 * WMERGE (an RMSNORM followed by the ACT_Q8 of its output is one
 * flh_rmsnorm_act_q8 launch, and with a single-column STREAM_DOT of that
 * activation after them, one flh_rmsnorm_stream_dot);
 * anything else -> FLH_ERR_UNSUPPORTED before any launch.  Consecutive
 * STREAM_DOT row tiles of one matrix (same fmt/cols/x/nx/strides, w and y
 * contiguous) are fused into one launch, and an ACT_Q8 followed by its
 * single-column q8_K consumer runs as flh_act_q8_stream_dot; results are
 * unchanged.  Masks are used as given, the same way as by every other entry
 * point (the same dot gives the same bits through any of them): pass the
 * reference's CPU masks (flh_default_masks) for the int8 parity path.  With
 * the reference's GPU defaults (kI8MaskGpuDefault / kI8KMaskGpuDefault,
 * src/runtime/kernels.h:927-940) Q6_K takes the fp32 dequant route (the
 * same order on one wave per row, about 2x the int8 route's time at the
 * vocab head); with the CPU masks IQ2_XXS / IQ3_XXS take it.
 * The param blocks that RMSNORM, ROUTER_SEL, SILU_MUL and WMERGE tasks point
 * to through aux are read by the host when the table is issued, so they must
 * be host-readable (host, pinned or managed memory; flh_host_alloc gives
 * pinned memory): a block in device memory is rejected with FLH_ERR_ARG
 * before anything is launched.  The buffers those blocks name, and every
 * other Task pointer, are device memory. */
int flh_exec_tasks(const flh_task * tasks, uint32_t n, int fast,
                   uint32_t i8_mask, uint32_t i8k_mask, void * stream);

/* Bit-exact dequantisation of whole rows to fp32, out[r*cols + c]
 * (dequant_chunk, src/runtime/kernels.h:162-242). */
int flh_dequant(int fmt, const void * w, uint32_t rows, uint32_t cols,
                float * out, void * stream);

/* ------------------------------------------------------------------ MoE -- */
/* Grouped expert matvec (the STREAM_DOT_IDX expert tiles of
 * src/model/decoder.cpp:941-996, grouped by expert): for every routed pair
 * i = tok*top_k + slot with e = ids[i],
 *   y[i*ystride + r] += dot(W_e[r], x + xi*xstride),  W_e = w + e*estride,
 * xi = tok (x_per_slot = 0) or i (x_per_slot = 1).  Each expert's weights
 * are streamed once for all of its pairs (Q4_K, Q6_K: the q8_K int8 path);
 * Q8_0, Q5_0, IQ2_XXS and IQ3_XXS run the q8_1 int8 path one pair at a time,
 * as the reference's per-pair tiles do: one routed launch where its plan
 * holds the shape (16-byte aligned w, x and estride, at most ~14.5K columns;
 * IQ: a multiple of 2048), else one STREAM_DOT_IDX tile per pair (up to 16384
 * columns; the ids must then be < n_expert, as ROUTER_SEL writes them).
 * cols a positive multiple of 256 (0 is FLH_ERR_ARG).  Every output is bitwise equal to the per-pair
 * STREAM_DOT_IDX tile. */
int flh_moe_dot(int fmt, const void * w, uint64_t estride, uint32_t rows,
                uint32_t cols, const uint32_t * ids, uint32_t ntok,
                uint32_t top_k, uint32_t n_expert, const float * x,
                uint32_t xstride, uint32_t x_per_slot, float * y,
                uint32_t ystride, void * stream);

/* ROUTER_SEL for ntok tokens (fl_op_router_sel, decode_params.h:234-265):
 * logits [ntok][n_expert], ids/gates [ntok][top_k]. */
int flh_router_sel(const float * logits, uint32_t ntok, uint32_t n_expert,
                   uint32_t top_k, uint32_t norm, float scale, uint32_t * ids,
                   float * gates, void * stream);
/* ROUTER_SEL followed by the grouped expert matvec of its routing, as one
 * launch where the grouped kernels take it (n_expert <= 64, top_k <= 8,
 * ntok*top_k <= 256; otherwise two): every workgroup routes the ntok tokens
 * itself with the same float operations as flh_router_sel, one of them
 * writes ids and gates.  Outputs (ids, gates, y) equal flh_router_sel then
 * flh_moe_dot bit for bit.  Replaces the ROUTER_SEL task
 * (src/runtime/decode_params.h:234-265) and the STREAM_DOT_IDX expert tiles
 * it feeds (src/model/decoder.cpp:941-996) for one MoE layer. */
int flh_router_moe_dot(int fmt, const void * w, uint64_t estride, uint32_t rows,
                       uint32_t cols, const float * logits, uint32_t ntok,
                       uint32_t n_expert, uint32_t top_k, uint32_t norm, float scale,
                       uint32_t * ids, float * gates, const float * x, uint32_t xstride,
                       uint32_t x_per_slot, float * y, uint32_t ystride, void * stream);
/* SILU_MUL over ncol columns (fl_op_silu_mul, decode_params.h:267-272):
 * h[c*hstride + i] = silu(g[c*gstride + i]) * u[c*gstride + i]. */
int flh_silu_mul(const float * gate, const float * up, float * h, uint32_t n,
                 uint32_t ncol, uint32_t gstride, uint32_t hstride, void * stream);
/* SILU_MUL over ncol columns followed by ACT_Q8 of each h column, in one
 * launch: h holds ACT_Q8 buffers (fp32 h, then its q8_1 and q8_K appendices,
 * columns hstride floats apart, 16-byte aligned); the bytes written equal
 * flh_silu_mul followed by flh_act_q8 (fl_op_silu_mul then fl_exec_act_q8,
 * decode_params.h:267-272, quants.h:404-416; the decoder's down-projection
 * input, decoder.cpp:874-880).  flh_exec_tasks fuses such a task pair itself. */
int flh_silu_mul_act_q8(const float * gate, const float * up, float * h, uint32_t n,
                        uint32_t ncol, uint32_t gstride, uint32_t hstride, void * stream);
/* RMSNORM of one column (fl_op_rmsnorm, decode_params.h:101-106:
 * y = (x * s) * wnorm, s = 1 / sqrtf(mean(x^2) + eps)) with, when write_app,
 * the ACT_Q8 of y in the same launch (y is then an ACT_Q8 buffer, 16-byte
 * aligned, and its appendices get the bytes flh_act_q8 would write from
 * these y values: the decoder's norm -> quant chain, decoder.cpp:874-880).
 * The reference (CPU-only op) sums the squares strictly in order; here the
 * 16 waves of one workgroup sum them as a tree (lane partials over its
 * elements in order, wave and workgroup trees in a fixed order), so s
 * and y agree with the reference to float rounding, not bit for bit (the
 * tests bound it); everything after s is the reference's arithmetic. */
int flh_rmsnorm_act_q8(const float * x, const float * wnorm, float * y, uint32_t n, float eps,
                       int write_app, void * stream);
/* WMERGE over ncol columns (fl_op_wmerge, decode_params.h:274-295): column c
 * reads parts + c*pstride ([n_parts][n]), gates + c*n_parts, add1/add2 +
 * c*ystride, writes y + c*ystride. */
int flh_wmerge(const float * parts, const float * gates, const float * add1,
               const float * add2, float * y, float scale, uint32_t n_parts,
               uint32_t n, uint32_t n_full, uint32_t ncol, uint32_t pstride,
               uint32_t ystride, void * stream);

/* ------------------------------------------- paged cache and attention -- */
/* What a decoder layer runs between its QKV dots and its O dot: pages for
 * the tokens that requests add, rotary positions, the key/value cache, and
 * attention over it.  The reference has a flat fp32 cache and per-head tasks
 * for this (ROPE_DS2, KV_APPEND, ATTN_HEAD, src/runtime/decode_params.h:48-55,
 * 118-160, 183-232; CPU only); these entry points are this backend's own form for many
 * requests at once, so flh_exec_tasks goes on refusing those task kinds.
 * Lengths, tables and slots are read on the device, so a captured step can be
 * replayed while requests grow. */

/* Element types of activations and of the cache. */
enum { FLH_DT_F32 = 0, FLH_DT_F16 = 1, FLH_DT_BF16 = 2 };

/* "no page" / "no slot" */
#define FLH_KV_NONE 0xFFFFFFFFu

/* A paged key/value cache of one layer: n_pages pages of page_size tokens (a
 * power of two up to 65536).  Token t of a page, kv head h: d_k keys at
 * k + page*k_page + t*k_tok + h*k_head and d_v values at v + ... (strides in
 * elements, so heads may lie inside tokens or tokens inside heads, and k and v
 * may share an allocation).  dtype is F16 or BF16; d_k and d_v are multiples of
 * 8 up to 256; k and v are 16-byte aligned, strides multiples of 8 (page and token
 * strides below 2^31, head strides below 2^40).  A token's
 * slot is page*page_size + t; n_pages*page_size < 2^32 - 1. */
typedef struct flh_kv_cache {
    void * k, * v;
    uint32_t dtype, n_pages, page_size, n_kv_head, d_k, d_v;
    uint64_t k_page, k_tok, k_head, v_page, v_tok, v_head;
} flh_kv_cache;

/* Block tables and slot maps from request lengths.  Request s holds held[s]
 * tokens and adds add[s]; its row of table (table_stride entries) holds the
 * pages of the held ones.  Rows (new tokens) are packed: request s has rows
 * q_start[s] .. q_start[s+1], cut off at max_tok, and kv_len[s] = held[s] +
 * its rows.  Pages that a request now reaches are taken off free_pages
 * (n_free entries, in order, requests in order), from entry *taken_in on (NULL:
 * 0), and written into the table; *taken = *taken_in + the pages needed; other
 * table entries stay as they are.  slot[r] and pos[r] of row r: its cache slot
 * and its position in its request; behind the last row, up to max_tok, they are
 * FLH_KV_NONE and 0 (a captured step of max_tok rows may have fewer).
 * A row has slot FLH_KV_NONE when free_pages ran out (its table
 * entry is FLH_KV_NONE, and *taken > n_free), when its page lies behind
 * the table's row, or when its table entry is no page.  info[0]: rows;
 * info[1]: new tokens without a slot (0: all is well; those cut off at max_tok
 * count).  page_size: a power of two up to 65536; max_tok and table_stride * page_size at
 * most 2^31.  pos and info may be NULL.
 * kv_len may be held and taken may be taken_in (a captured step then advances
 * its requests by itself); nothing else may overlap.  free_pages and table
 * hold the page numbers of a flh_kv_cache. */
typedef struct flh_kv_plan_p {
    const uint32_t * held, * add, * free_pages, * taken_in;
    uint32_t * taken, * table, * q_start, * kv_len, * slot;
    int32_t * pos;
    uint32_t * info;
    uint32_t n_seq, page_size, n_free, table_stride, max_tok;
} flh_kv_plan_p;
int flh_kv_plan(const flh_kv_plan_p * p, void * stream);

/* Rotary frequencies of the elements first .. first + n_rot - 1 of a head.
 * Pair i (of n_rot / 2) is elements (i, i + n_rot/2) of that range with
 * FLH_ROPE_HALVES, (2i, 2i + 1) with FLH_ROPE_PAIRS; its angle is the token's
 * position on axis axis[i] (NULL: 0; axis[i] < n_axis <= 8) times freq[i]
 * (host doubles, radians per position; NULL: base^(-2i/n_rot)).  Several axes are
 * the time, height and width of image and video tokens.  n_rot: even, 2..1024.
 * Angles are kept as 64-bit fractions of a turn, so positions up to
 * 2^31 - 1 (and negative ones) lose nothing.  The table lives on the device of
 * flh_init; create waits for its upload. */
enum { FLH_ROPE_HALVES = 0, FLH_ROPE_PAIRS = 1 };
typedef struct flh_rope_table flh_rope_table;
int flh_rope_table_create(uint32_t n_rot, uint32_t first, int layout, double base, const double * freq,
                          uint32_t n_axis, const uint8_t * axis, flh_rope_table ** out);
int flh_rope_table_destroy(flh_rope_table * r);

/* (a, b) -> (a cos - b sin, a sin + b cos) over the pairs of n_head heads of
 * n_tok tokens, x -> y, d elements a head (first + n_rot <= d; the others are
 * copied); strides in elements.  pos[axis*pos_stride + token].  y may be x with
 * the same strides, else the two must not overlap.  The arithmetic is fp32 in
 * every dtype. */
int flh_rope(const flh_rope_table * r, uint32_t dtype, const void * x, uint64_t x_tok, uint64_t x_head, void * y,
             uint64_t y_tok, uint64_t y_head, uint32_t n_tok, uint32_t n_head, uint32_t d, const int32_t * pos,
             uint32_t pos_stride, void * stream);

/* The same for the queries of n_tok tokens (q -> q_out; n_head = 0: none) and
 * their keys, and the keys and values into the cache at slot[token], rounded
 * to its dtype; one launch.  Tokens whose slot is not in the cache (FLH_KV_NONE)
 * write nothing there.  Slots of one call must differ.  r = NULL: nothing is
 * rotated (pos is not read).  q, k and v may be columns of one product's rows
 * (any element strides); q_out as y of flh_rope, and apart from k and v; the cache must not
 * overlap them. */
typedef struct flh_rope_kv_p {
    const void * q; void * q_out; const void * k; const void * v;
    const int32_t * pos; const uint32_t * slot;
    uint64_t q_tok, q_head, qo_tok, qo_head, k_tok, k_head, v_tok, v_head;
    uint32_t dtype, n_tok, n_head, pos_stride;
} flh_rope_kv_p;
int flh_rope_kv_append(const flh_rope_table * r, const flh_kv_cache * cache, const flh_rope_kv_p * p, void * stream);

/* Attention of new tokens over the paged cache.  Request s has query rows
 * q_start[s] .. q_start[s+1] (ascending; rows from n_tok on are not computed, rows of no
 * request are left as they are in out) and keys 0 .. kv_len[s] - 1, key j at token j % page_size of page
 * table[s*table_stride + j / page_size].  causal: the rows are the last
 * tokens, row i of n = q_start[s+1] - q_start[s] at position p = kv_len - n + i, and see the keys
 * j <= p, with window > 0 also j > p - window; else every row sees every
 * key (an encoder's states as the cache) and window must be 0.  Query head h
 * reads kv head h / (n_head / n_kv_head).
 *   out[row][head] = sum_j softmax_j(scale q.k_j) v_j   over the keys seen,
 * 0 for a row that sees none (not a number for one that sees keys, all with scores of
 * -infinity; a score past the range of fp32 is infinite, and a q.k below it, whatever the scale, may
 * count as -infinity); keys not seen have no part in it, whatever the cache
 * holds there.  Keys whose table entry is no page of the cache, or lies
 * behind the table's row, are not seen (kv_len and a table's row: at most 2^30
 * tokens).  dtype of q and out: F32 over either cache, or the cache's own.  Scores,
 * maxima, weights and sums are fp32.  Into the products go, with F32, queries and weights in two
 * f16 terms (right to 2^-22 of a value) or three bf16 terms (2^-24); else weights in two terms
 * (2^-22, bf16 2^-16) where max_q * n_head / n_kv_head <= 32, and rounded once to the cache's type
 * where it is more (the sum that they are divided by is of the unrounded ones).  Over an F16
 * cache a weight is besides right only to 2^-32 of its row's largest.  scale: finite, >= 0.  q and out: any element strides,
 * aligned to an element; out must not overlap q (other columns of the same rows, or
 * beside each head, do not).  max_q: the most rows of a
 * request that the caller expects (it chooses the kernel, the results hold for
 * any).  Rows that see an infinite or NaN key or value, and those that share a
 * workgroup with one, are done one by one, which takes the call 30 to 300 times as
 * long.  ws: flh_paged_attn_ws_bytes of the same arguments (pointers and lengths
 * are not looked at; by the chosen kernel and the widths, not by the rows: 4 to 70 MB on 256
 * CUs), 16-byte aligned; its contents need not be kept or
 * cleared.  Calls on one stream may share one, whichever threads make them; calls on
 * several streams, and graphs that may be replayed at the same time, need one each. */
typedef struct flh_attn_p {
    const void * q; void * out;
    const uint32_t * q_start, * kv_len, * table;
    void * ws; size_t ws_bytes;
    uint64_t q_tok, q_head, o_tok, o_head;
    uint32_t dtype, n_head, n_seq, n_tok, max_q, table_stride, causal, window;
    float scale;
} flh_attn_p;
size_t flh_paged_attn_ws_bytes(const flh_kv_cache * cache, const flh_attn_p * p);
int flh_paged_attn(const flh_kv_cache * cache, const flh_attn_p * p, void * stream);

/* ------------------------------------------- trees of drafted tokens -- */
/* A step that verifies drafts which branch: flh_kv_plan (slots by row), flh_tree_plan, then the layers
 * (flh_rope_kv_append with its pos, flh_tree_attn), the vocabulary's product, flh_spec_verify,
 * flh_kv_compact and flh_kv_trim; nothing comes back to the host in between.  The reference
 * verifies runs of drafted tokens one sequence at a time, greedily, on the host
 * (tools/decode_main.cpp:332-370); these are this backend's own form.
 *
 * A request's rows are a tree: row 0 is its last token (whose keys and values are new, too), the
 * others drafted ones behind it. */

/* parent[r]: the row that row r of a request hangs on, by its index in the request, below its own; anything
 * else: row r is a root.  depth[r]: rows above it; bit b of its mask_stride words of mask: row b of the
 * request is r itself or above it (rows b >= 32 * mask_stride have no bit), with window > 0 only those
 * less than window above it; pos[r] (may be NULL, then kv_len too): kv_len[s] - rows of the
 * request + depth[r].  Rows n_tok and behind, and rows of no request, are left as they are.
 * mask_stride: 1 .. 32768.  Each row's line is walked up, for each word, so the time grows with the trees' depth:
 * n_tok * n_tok * mask_stride is at most 2^44 (2^22 rows with a word each).  Outputs must not overlap anything. */
typedef struct flh_tree_plan_p {
    const uint32_t * q_start; const int32_t * parent; const uint32_t * kv_len;
    uint32_t * mask, * depth; int32_t * pos;
    uint32_t n_seq, n_tok, mask_stride, window;
} flh_tree_plan_p;
int flh_tree_plan(const flh_tree_plan_p * p, void * stream);

/* flh_paged_attn for a tree's rows (causal must be set): row i of a request's n sees the keys
 * j < kv_len - n (with window > 0 those with j > kv_len - n + depth[row] - window) and key kv_len - n + b for
 * each bit b of its words of mask (any bits, also of rows behind it; the window is not applied to them).
 * A row that sees no key gives 0.  depth (NULL without a window) counts as at most n - 1.
 * Everything else is as flh_paged_attn's. */
typedef struct flh_tree_p {
    const uint32_t * mask, * depth;
    uint32_t mask_stride;
} flh_tree_p;
size_t flh_tree_attn_ws_bytes(const flh_kv_cache * cache, const flh_attn_p * p);
int flh_tree_attn(const flh_kv_cache * cache, const flh_attn_p * p, const flh_tree_p * t, void * stream);

/* Which rows of each request's tree stand, and the token behind them.  target: logits of row r at
 * target + r * t_row (vocab of them, any stride, aligned to an element).  draft (NULL: tokens drafted
 * without a distribution): logits, in the same way, that the children of row r were drawn from, each by itself; rows
 * without children are not read.  token[r]: the drafted token (a request's row 0 has none); one that is not below vocab does not
 * stand.  parent as in flh_tree_plan (NULL: each row hangs on the one before); of a row's children the first max_child (1 .. 64) are
 * looked at, of a request's rows the first 256.
 * p = softmax(inv_temp[s] * target) and q of the draft (inv_temp NULL: 1; infinity: greedy, p is 1 at
 * the first of the largest, whatever the draft; what is not >= 0 counts as 0).  A logit that is no number counts as -infinity, infinity as
 * the largest float.  From row 0 on, a row's children are tested in order: the first one stands if
 * u_accept * q(x) < p(x), and each that does not stand leaves max(p - q, 0), over its sum, as p for the next
 * (without a draft: p without its token; where that is nothing at all, none of the next stands).  The path goes on at
 * the first that stands; where none does, or there is none, next is the first token whose sum of what is left of p, up to and with it, passes u_next[s] times the
 * whole (nothing left: of p).  Then the tokens of the path and next together are distributed as p alone would
 * have them, u_accept and u_next being uniform in [0, 1).  Weights, sums and borders are in 64 bits: a weight is right to
 * 2^-45 of itself and 0 below 2^-1000 of its row's largest (one below 2^-600 counts as about that in the row's sum); without a draft
 * what fallen tokens leave is 1 less their p, right to 2^-52 of the whole.
 *   n_path[s]: rows of the path, row 0 with it (0 for a request without rows); path[s * path_stride + j]: its
 * rows, by their index in the request, ascending; FLH_KV_NONE behind them.  A path ends at path_stride rows, as if the last one
 * had no children (whether one would have stood or not).  next[s]: the token (FLH_KV_NONE where the target allows
 * none, or there is no row).
 * logp (or NULL): entry j of a request, the logarithm of p (of the row, as it was) at the token behind the path's row j: that of row
 * j + 1, at last next; 0 behind.  len (or NULL, then kv_len may be): kv_len[s] - rows + n_path[s], what the
 * request holds then (all of its rows, also those that n_tok cuts off).  ws: flh_spec_verify_ws_bytes of the same arguments, 16-byte aligned, as
 * flh_paged_attn's.  Outputs must not overlap anything, but len may be kv_len.  vocab: 1 .. 2^22; all n_tok rows of target, and
 * of draft, have to be there, also those of no request; n_tok and n_seq, times the
 * vocabulary's chunks of 4096, below 2^24. */
typedef struct flh_verify_p {
    const void * target, * draft;
    const uint32_t * q_start, * token; const int32_t * parent;
    const float * inv_temp, * u_accept, * u_next; const uint32_t * kv_len;
    uint32_t * n_path, * path, * next; float * logp; uint32_t * len;
    void * ws; size_t ws_bytes;
    uint64_t t_row, d_row;
    uint32_t dtype, n_seq, n_tok, vocab, path_stride, max_child;
} flh_verify_p;
size_t flh_spec_verify_ws_bytes(const flh_verify_p * p);
int flh_spec_verify(const flh_verify_p * p, void * stream);

/* ------------------------------------------------- pages between steps -- */
/* caches: a host array of n_cache layers' caches, alike but for k and v (one launch for up
 * to 64 of them). */

/* The rows of a path into place: in every layer, token path[s * path_stride + j] of request s (j < n_path[s]; by
 * row, slot as flh_kv_plan gave it) is moved to the slot of its row j, so that the path's tokens follow one another
 * behind the cached ones.  path ascends with path[j] >= j, as flh_spec_verify's does (an entry that is no row
 * of the request, or has no slot, is left out).  n_tok: entries of slot. */
typedef struct flh_kv_compact_p {
    const uint32_t * q_start, * slot, * n_path, * path;
    uint32_t n_seq, n_tok, path_stride;
} flh_kv_compact_p;
int flh_kv_compact(const flh_kv_cache * caches, uint32_t n_cache, const flh_kv_compact_p * p, void * stream);

/* n_copy copies in every layer: n_tok[i] tokens from slot src[i] on to slot dst[i] on, as far
 * as both pages reach; a slot that is not in the cache (FLH_KV_NONE): none.  No slot that is written may be
 * another copy's, or this one's, source or target. */
int flh_kv_copy(const flh_kv_cache * caches, uint32_t n_cache, const uint32_t * src, const uint32_t * dst, const uint32_t * n_tok,
                uint32_t n_copy, void * stream);

/* Requests that share pages.  shared[page]: how many hold it besides the first (0: it is one request's, or
 * free), n_pages entries.  The free list is flh_kv_plan's: free_pages[*taken ..] are free.
 *
 * flh_kv_fork: request dst[i] (a row of table that holds nothing) takes over the first len[i] (NULL: all) tokens of
 * request src[i], at most what it holds and its row of the table reaches.  Full pages are shared; for a partly
 * filled last one dst gets a page off the free list and copy i of the
 * lists (copy_src, copy_dst: slots, copy_n: tokens; FLH_KV_NONE, FLH_KV_NONE, 0 where there is none), which
 * flh_kv_copy has to run before dst is read or src's page written again.  kv_len[dst[i]] is set.  Where the list ran out
 * the entry is FLH_KV_NONE (those tokens are not seen), *taken > n_free, and info[1] (info may be NULL) counts it;
 * info[0]: copies.  An entry that is no page is FLH_KV_NONE in dst, too.  dst differ from each other and from every src; a
 * pair of which one is not below n_seq, or that is one and the same, is left out.  n_fork: at most 2^21.
 *
 * flh_kv_trim: request s holds min(kv_len[s], keep[s]) tokens afterwards (held[s]; may be kv_len).  Pages
 * behind them are left: their table entries are FLH_KV_NONE, and those that nobody holds any more go back to
 * the free list, in the order of the requests' and pages that left them last, the last one to be taken next (*taken
 * goes down; a list of n_free entries takes back what was taken off it).  A last page that is partly filled and shared is left to the others: the
 * request gets one off the list, and a copy in the lists (as above; run it before the next flh_kv_plan, n_seq entries), so that it may append.  shared NULL: nothing
 * is shared, and the lists are not written.  info[0]: pages put back; info[1]: pages that the list has no
 * room for, and copies that found no page (the entry is FLH_KV_NONE).  n_seq * table_stride below 2^31 - 1.
 * Entries of table that are no page are left out.  Nothing may overlap but held and kv_len. */
typedef struct flh_kv_fork_p {
    const uint32_t * src, * dst, * len;
    uint32_t * kv_len, * table; const uint32_t * free_pages; uint32_t * taken, * shared;
    uint32_t * copy_src, * copy_dst, * copy_n, * info;
    uint32_t n_fork, n_seq, n_pages, page_size, n_free, table_stride;
} flh_kv_fork_p;
int flh_kv_fork(const flh_kv_fork_p * p, void * stream);
typedef struct flh_kv_trim_p {
    const uint32_t * kv_len, * keep;
    uint32_t * held, * table, * free_pages, * taken, * shared;
    uint32_t * copy_src, * copy_dst, * copy_n, * info;
    uint32_t n_seq, n_pages, page_size, n_free, table_stride;
} flh_kv_trim_p;
int flh_kv_trim(const flh_kv_trim_p * p, void * stream);

/* ---------------------------------------------------------------- GGUF -- */
/* GGUF v2/v3 reader (replaces fastllm::Gguf, src/model/gguf.h:28-79,
 * src/model/gguf.cpp:133-303).  The file is mmapped read-only; metadata and
 * tensor infos are parsed at open.  Split models named
 * "<stem>-NNNNN-of-MMMMM.gguf" map every shard: metadata comes from the shard
 * named, tensors are merged in shard order, each with offsets relative to its
 * own shard's data section; split.tensors.count, when present, must equal the
 * tensors mapped.  Where Gguf::open aborts (bad magic / version / KV type /
 * n_dims, truncation) this returns FLH_ERR_FORMAT; a missing file or shard
 * gives FLH_ERR_IO (Gguf::open returns false).  Stricter than the reference:
 * a tensor payload past the end of its file, an array of an unsized element
 * type and a general.alignment that is not a power of two are FLH_ERR_FORMAT.
 * Host-only: nothing before flh_gguf_upload* touches the GPU. */
typedef struct flh_gguf flh_gguf;

/* One tensor info (GgufTensor, src/model/gguf.h:19-27).  Pointers stay valid
 * until flh_gguf_close. */
typedef struct flh_gguf_tensor {
    const char * name;
    size_t name_len;
    uint32_t type;             /* ggml_type id */
    int32_t fmt;               /* FLH_FMT_* (Gguf::fmt_of), -1 if none */
    int32_t n_dims;
    uint64_t ne[4];            /* unused dims are 1 */
    uint64_t offset;           /* relative to its shard's data section */
    uint64_t nbytes;           /* payload bytes; 0 for types with no size */
    int32_t shard;
    const void * data;         /* host pointer into the mapping (Gguf::data) */
} flh_gguf_tensor;

/* A STREAM_DOT weight bound from a tensor (DecoderImpl::load_tensor,
 * src/model/decoder.cpp:186-206): cols = ne[0], rows = ne[1], nexp = ne[2]
 * for 3-D expert stacks (else 1), estride = rows*row_bytes when nexp > 1. */
typedef struct flh_weight {
    int32_t fmt;
    uint32_t rows, cols, nexp;
    uint64_t row_bytes, w_bytes, estride;
    const void * host;         /* mapping pointer of expert 0 */
    uint64_t tensor;           /* tensor index */
} flh_weight;

int flh_gguf_open(const char * path, flh_gguf ** out);
int flh_gguf_close(flh_gguf * g);
uint32_t flh_gguf_alignment(const flh_gguf * g);   /* of the named shard */
int flh_gguf_n_shards(const flh_gguf * g);
uint64_t flh_gguf_n_tensors(const flh_gguf * g);
int flh_gguf_tensor_info(const flh_gguf * g, uint64_t i, flh_gguf_tensor * out);
/* index of the first tensor of that name (Gguf::find), -1 if none */
int64_t flh_gguf_find(const flh_gguf * g, const char * name);
/* Gguf::fmt_of / Gguf::type_name (src/model/gguf.cpp:82-109) */
int flh_gguf_fmt_of(uint32_t ggml_type);
const char * flh_gguf_type_name(uint32_t ggml_type);
/* Metadata (Gguf::has / kv_i / kv_f / kv_s / kv_sarr, gguf.cpp:267-293):
 * integer kinds and bool read as int64, f32/f64 as double, each readable
 * through the other getter; strings and string arrays verbatim (len
 * receives the byte length, strings may hold NUL bytes).  Arrays of other
 * element types are skipped.  kv_sarr_len is -1 for an absent key. */
int flh_gguf_has(const flh_gguf * g, const char * key);
int64_t flh_gguf_kv_i(const flh_gguf * g, const char * key, int64_t dflt);
double flh_gguf_kv_f(const flh_gguf * g, const char * key, double dflt);
const char * flh_gguf_kv_s(const flh_gguf * g, const char * key, const char * dflt,
                           size_t * len);
int64_t flh_gguf_kv_sarr_len(const flh_gguf * g, const char * key);
const char * flh_gguf_kv_sarr_at(const flh_gguf * g, const char * key, uint64_t i,
                                 size_t * len);
/* FLH_ERR_ARG for a missing tensor, FLH_ERR_UNSUPPORTED for a type with no
 * Fmt (the two failures of load_tensor). */
int flh_gguf_weight(const flh_gguf * g, const char * name, flh_weight * out);

/* Host -> device.  The reference reads the mapping in place through unified
 * memory (decoder.cpp:203); here weights are copied into HBM once.  Bytes go
 * through a ring of pinned staging buffers filled by host threads while the
 * DMA engine drains the previous one; both calls return when every byte is
 * on the device.  flh_gguf_upload copies tensor i to dst (dst_bytes >=
 * nbytes).  flh_gguf_upload_all allocates, per shard, one 256-B aligned arena
 * block for the span of its tensor payloads and copies that span as-is, so
 * dev_ptrs[i] (n_tensors entries) = block + offset keeps the file's alignment;
 * dev_ptrs[i] = NULL where nbytes = 0.  Uploads from several threads are
 * serialised. */
int flh_gguf_upload(const flh_gguf * g, uint64_t i, void * dst, uint64_t dst_bytes,
                    void * stream);
int flh_gguf_upload_all(const flh_gguf * g, flh_arena * arena, void ** dev_ptrs,
                        void * stream);

/* ----------------------------------------------------- synthetic inputs -- */
/* dst[i] = mean + stddev * N(0,1) from a counter-based generator keyed by
 * (seed, i); a fraction outlier_frac of entries is multiplied by
 * outlier_scale.  Deterministic for a given (seed, n). */
int flh_fill_normal(float * dst, size_t n, uint64_t seed, float mean,
                    float stddev, float outlier_frac, float outlier_scale,
                    void * stream);
/* fp32 rows -> Q8_0 / Q4_K / Q6_K blocks on the device; flh_quantize_host
 * produces the same bytes on the host.  (The reference ships no weight
 * quantizer; these are this backend's own, for synthetic weights.) */
int flh_quantize(int fmt, const float * src, uint32_t rows, uint32_t cols,
                 void * dst, void * stream);
int flh_quantize_host(int fmt, const float * src, uint32_t rows, uint32_t cols,
                      void * dst);

#ifdef __cplusplus
}
#endif
#endif /* FASTLLM_HIP_H */
