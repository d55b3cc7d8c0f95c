/*
 * myos_cuda.h — C ABI of the B200 (sm_100a) Qwen2.5 BF16 token loop.
 *
 * This is the drop-in boundary for the MyOS reference's decode path. Each
 * entry point names the reference interface it stands in for (paths are
 * relative to the reference project). Plain pointers and sizes only; no
 * PyTorch or C++ types cross it. All numeric work runs on the GPU: there is
 * no CPU fallback, and every call fails with MYOS_ERR_CUDA when no usable
 * sm_100 device is present.
 *
 * Numerics contract (same as the reference): weights are little-endian BF16,
 * promoted to f32 inside the kernels; every activation, accumulator and the
 * logits are f32. Reductions run in a fixed parallel order (deterministic
 * run to run) instead of the reference's serial left-to-right chain, so
 * results agree to within float reassociation, not bit for bit. Elementwise
 * steps (RMSNorm scaling, bias, RoPE with a host-built libm cos/sin table,
 * residual adds, SiLU's division form, softmax's e/sum) use the reference's
 * operation order without contraction.
 *
 * Error contract: every int-returning call returns MYOS_OK (0) or a status
 * below; on error the KV cursor and the logits are unchanged
 * (crates/model_core/src/qwen25_block.rs:129-134) and myos_last_error()
 * holds a one-line message. One context drives one device stream and is not
 * thread-safe; separate contexts may be used from separate threads.
 */
#ifndef MYOS_CUDA_H
#define MYOS_CUDA_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif
#ifdef __cplusplus
extern "C" {
#endif

/* Status codes. Names follow the reference's error enums. */
enum myos_status {
  MYOS_OK = 0,
  MYOS_ERR_SHAPE = 1,          /* BlockError::Shape, Bf16OpError::Shape, GqaError::Shape */
  MYOS_ERR_TOKEN = 2,          /* BlockError::Token, Bf16OpError::TokenOutOfBounds */
  MYOS_ERR_ROW_OOB = 3,        /* Bf16OpError::RowOutOfBounds */
  MYOS_ERR_POSITION = 4,       /* BlockError::Position */
  MYOS_ERR_CACHE_FULL = 5,     /* KvError::Full */
  MYOS_ERR_CACHE_RANGE = 6,    /* KvError::Range */
  MYOS_ERR_WEIGHT_MISSING = 7, /* QwenBf16Error::Missing */
  MYOS_ERR_WEIGHT_DTYPE = 8,   /* QwenBf16Error::DType */
  MYOS_ERR_WEIGHT_SHAPE = 9,   /* QwenBf16Error::Shape */
  MYOS_ERR_WEIGHT_LENGTH = 10, /* QwenBf16Error::Length, WeightError::LengthMismatch */
  MYOS_ERR_DUPLICATE = 11,     /* WeightError::Duplicate */
  MYOS_ERR_EMPTY_NAME = 12,    /* WeightError::EmptyName */
  MYOS_ERR_PARSE = 13,         /* WeightError::Parse */
  MYOS_ERR_UNSUPPORTED = 14,   /* WeightError::UnsupportedDType */
  MYOS_ERR_IO = 15,            /* WeightFileError::Io */
  MYOS_ERR_CUDA = 16,          /* CUDA runtime failure or no sm_100 device */
  MYOS_ERR_NCCL = 17,          /* collective failure (tensor-parallel contexts) */
  MYOS_ERR_TIMEOUT = 18,       /* a bounded device-side wait gave up */
  MYOS_ERR_ARG = 19,           /* null pointer or invalid option */
  MYOS_ERR_SCRATCH_LIMIT = 20, /* request needs more than the fixed no-allocation scratch
                                  (MYOS_NOALLOC_SCRATCH_BYTES); no reference counterpart */
};

/* Tensor storage tags, weight_loader::DType (crates/weight_loader/src/lib.rs:36-49). */
enum myos_dtype { MYOS_F32 = 0, MYOS_F16 = 1, MYOS_BF16 = 2 };

/* KV-cache element type. The reference cache is f32
 * (crates/model_core/src/kv_cache.rs:89-125); bf16 halves its HBM traffic. */
enum myos_kv_dtype { MYOS_KV_F32 = 0, MYOS_KV_BF16 = 1 };

/* model_core::BlockShape + AttnShape (crates/model_core/src/qwen25_block.rs:53-75,
 * crates/model_core/src/attn_wire.rs:44-63). tied_head = 1 uses
 * model.embed_tokens.weight as the output projection (the reference's only
 * mode, qwen25_block.rs:290-301); 0 reads lm_head.weight (Qwen2.5-14B). */
typedef struct myos_shape {
  uint32_t hidden;
  uint32_t num_q_heads;
  uint32_t num_kv_heads;
  uint32_t head_dim;
  float rope_theta;
  uint32_t intermediate;
  uint32_t vocab;
  uint32_t num_layers;
  float rms_eps;
  uint32_t tied_head;
} myos_shape;

/* Context options. max_seq is KvShape::max_seq
 * (crates/model_core/src/kv_cache.rs:28-45); the reference CLI passes
 * n_prompt + steps (crates/runtime/src/main.rs:549-555). */
typedef struct myos_opts {
  int32_t device;      /* CUDA ordinal */
  uint32_t max_seq;    /* KV slots per layer */
  int32_t kv_dtype;    /* enum myos_kv_dtype */
  int32_t use_graphs;  /* 1: replay each token step as one CUDA graph */
} myos_opts;

typedef struct myos_ctx myos_ctx;

/* BlockShape::qwen25_1_5b() (qwen25_block.rs:63-74) and the 14B geometry. */
myos_shape myos_shape_qwen25_1_5b(void);
myos_shape myos_shape_qwen25_14b(void);

/* Allocates the weight arena, KV cache (KvCache::new, kv_cache.rs:99-125) and
 * the workspace (BlockWorkspace::new, qwen25_block.rs:96-114) in HBM. */
int myos_ctx_create(const myos_shape* shape, const myos_opts* opts, myos_ctx** out);
void myos_ctx_destroy(myos_ctx* ctx);

/* Tensor parallelism over `size` GPUs, one process (and one context) per
 * GPU. The reference runs one process on one device and has no sharded
 * mode; this splits the same token step: q/k/v rows and attention by head,
 * o_proj and down_proj by input column (each projection's epilogue stores
 * its rows into every rank's inbox over peer memory and a small kernel
 * sums the ranks' parts in rank order; MYOS_TP_COMM=nccl, or GPUs that
 * cannot map each other's memory, use NCCL allreduce instead), gate/up by
 * row, and the output head by vocabulary row with a global first-maximum
 * pick. A rank's device waits on the others are bounded in time (60 s) and
 * end the call with MYOS_ERR_TIMEOUT; the context is not usable after that.
 * Weights are passed
 * whole to myos_load_tensor / myos_load_safetensors on every rank; each
 * rank keeps its slice. Every rank makes the same calls with the same
 * arguments, in the same order (host output pointers may be null on ranks
 * that do not read them). Needs size | num_q_heads, num_kv_heads,
 * intermediate and vocab (MYOS_ERR_SHAPE otherwise); a rank's MLP rows and
 * o_proj input columns are zero-padded to multiples of 256. The tensor-core prefill sums each chunk's
 * residual parts with an NCCL allreduce. Batched decode, the persistent step
 * kernel and myos_profile_kernels are single-GPU paths (MYOS_ERR_UNSUPPORTED).
 * At most 8 ranks (MYOS_ERR_ARG otherwise). */
typedef struct myos_tp {
  int32_t size;
  int32_t rank;
  uint8_t unique_id[128]; /* from myos_tp_unique_id on one rank, sent to all */
} myos_tp;

/* A fresh NCCL unique id (the rendezvous token every rank passes in). */
int myos_tp_unique_id(uint8_t out[128]);

/* Diagnostics of the tensor-parallel exchange on ONE GPU (no peers, no
 * NCCL): runs the exchange's reduce kernel over an inbox of n ranks x H
 * words. fill = 1: the host first writes every word as the first exchange's
 * (value 0.25 * (p + 1) + i / 1024 for rank p, element i) and out receives
 * the sums over p in rank order (f32 adds). fill = 0: nothing writes the
 * inbox, so the kernel's bounded wait must give up after timeout_ms
 * (1..10000) and the call returns MYOS_ERR_TIMEOUT. No reference
 * counterpart. */
int myos_tp_reduce_selftest(int32_t device, uint32_t n, uint32_t H, int32_t fill,
                            uint32_t timeout_ms, float* out);

/* How a tensor-parallel rank holds one named tensor of the whole model:
 * of the [rows, cols] tensor (matrix = 0: a vector, cols = 1) it keeps rows
 * [row0, row0 + nrows) and columns [col0, col0 + ncols), stored in an
 * extent of store_rows x store_cols whose extra rows/columns are zero (the
 * o_proj input and MLP widths are padded to multiples of 256). Heads (q/k/v
 * rows, o_proj columns), MLP columns (gate/up rows, down_proj columns) and
 * the untied head's vocabulary rows are split in rank order; embedding and
 * norms are whole on every rank. kept = 0: the model never reads the
 * tensor. This is the slicing myos_load_tensor applies to the whole tensor
 * it is given, so a loader can produce just the kept part (the rest of the
 * buffer it passes is not read). No counterpart in the reference, which
 * runs the whole model in one process. */
typedef struct myos_tp_part {
  uint64_t rows;
  uint64_t cols;
  uint64_t row0;
  uint64_t nrows;
  uint64_t col0;
  uint64_t ncols;
  uint64_t store_rows;
  uint64_t store_cols;
  int32_t matrix;
  int32_t kept;
} myos_tp_part;
int myos_tp_slice(const myos_shape* shape, int32_t size, int32_t rank, const char* name,
                  myos_tp_part* out);
int myos_ctx_create_tp(const myos_shape* shape, const myos_opts* opts, const myos_tp* tp,
                       myos_ctx** out);
const char* myos_last_error(const myos_ctx* ctx);

/* One named tensor from any WeightMap-shaped source
 * (weight_loader::WeightMap::tensor_info/tensor_bytes, lib.rs:137-146, with
 * the per-name dtype/shape checks of model_core::qwen25_bf16::bf16_tensor,
 * qwen25_bf16.rs:72-82). Bytes are copied to HBM through pinned staging; the
 * caller may free them on return. Unknown names are ignored (the reference
 * never looks them up), and only BF16 is accepted for known names. */
int myos_load_tensor(myos_ctx* ctx, const char* name, int32_t dtype, const int64_t* shape,
                     int32_t rank, const void* bytes, size_t nbytes);

/* SafeTensorsMmap::open + parse (crates/weight_loader/src/mmap.rs:82-100,
 * safe_tensors.rs:30-43): maps the file read-only, validates the header the
 * way the safetensors crate does, and stages every known tensor into HBM. */
int myos_load_safetensors(myos_ctx* ctx, const char* path);

/* Host-only: SafeTensorsMmap::open + parse without a context or a GPU (the
 * reference CLI's check_safetensors, crates/runtime/src/main.rs:452-458).
 * n_tensors (nullable) receives the tensor count. err (nullable, err_len
 * bytes) receives the failure message. */
int myos_check_safetensors(const char* path, size_t* n_tensors, char* err, size_t err_len);

/* 1 when every tensor the shape needs has been loaded (preflight_weights,
 * qwen25_block.rs:599-643); otherwise 0 and myos_last_error names the first
 * missing key. */
int myos_weights_ready(myos_ctx* ctx);

/* model_core::prefill (qwen25_block.rs:323-543): the prompt at positions
 * kv_len.., KV written for every position, head on the last id only. logits
 * (nullable) receives vocab floats. Advances the cursor by n on success. */
int myos_prefill(myos_ctx* ctx, const uint32_t* ids, size_t n, float* logits);

/* model_core::forward_token (qwen25_block.rs:220-304): pos must equal
 * kv_len. logits (nullable) receives vocab floats. */
int myos_forward_token(myos_ctx* ctx, uint32_t token, size_t pos, float* logits);

/* model_core::greedy_decode (qwen25_block.rs:765-780): steps tokens, each
 * the first maximum of the current logits (greedy_token,
 * crates/model_core/src/lib.rs:157-167), fed back on the device. */
int myos_greedy_decode(myos_ctx* ctx, size_t steps, uint32_t* out_ids);

/* Teacher-forced decode: feeds ids[i] at step i (not the argmax) and writes
 * the argmax of the logits seen before each feed into argmax_out[i]. Used
 * by the parity protocol so every step stays comparable after a divergence. */
int myos_forced_decode(myos_ctx* ctx, const uint32_t* ids, size_t steps, uint32_t* argmax_out);

/* KvCache::len / clear (kv_cache.rs:140-142, 234-237). */
int myos_kv_len(const myos_ctx* ctx, size_t* len);
int myos_reset(myos_ctx* ctx);

/* KvCache::key_head / value_head (kv_cache.rs:239-252): head_dim f32 each.
 * In a tensor-parallel context `head` counts this rank's KV heads
 * (global head rank * num_kv_heads / size + head). */
int myos_kv_head(myos_ctx* ctx, uint32_t layer, uint32_t head, size_t pos, float* k, float* v);

/* BlockWorkspace::logits (qwen25_block.rs:118-125): vocab floats. */
int myos_logits(myos_ctx* ctx, float* out);

/* Times each decode-step kernel alone with CUDA events on the context's
 * stream. Kinds: 0 QKV (RMSNorm + q|k|v GEMV + bias), 1 attention, 2 o_proj
 * (+ residual), 3 gate/up (RMSNorm + GEMV + SiLU*up), 4 down (+ residual),
 * 5 head (final norm + GEMV + argmax). A pass launches each kind once per
 * layer, each launch on that layer's weights, so the weights a pass touches
 * exceed L2; launches follow each other with programmatic dependent launch
 * as inside a token step; ms_out[6] gets the mean device time of one launch
 * over iters passes, bytes_out[6] the algorithmic bytes one launch moves (weights +
 * activations + KV read at the current length). Needs kv_len < max_seq;
 * the KV cursor, logits and argmax are left as they were. */
int myos_profile_kernels(myos_ctx* ctx, int iters, float* ms_out, double* bytes_out);

/* Device time of the last prefill / decode call, from CUDA events (ms). */
int myos_last_timing(const myos_ctx* ctx, float* prefill_ms, float* decode_ms);

/* Kernel launches this library has enqueued in the calling process, all
 * contexts and devices together (a CUDA graph replay adds the kernels
 * captured in it). Diagnostics for benchmarks; no counterpart in the
 * reference, which runs on the CPU. */
int myos_launch_count(uint64_t* out);

/* ---------------------------------------------------------------------------
 * tensor_core operators on host slices (crates/tensor_core/src/lib.rs:54-74).
 * Same argument meaning and error behaviour as the Rust functions; the work
 * runs on the current CUDA device through the same kernels the engine uses.
 * ------------------------------------------------------------------------- */

/* tensor_core::gemv_bf16 (bf16.rs:80-122): y[i] = sum_j bf16(W[i,j]) * x[j]. */
int myos_gemv_bf16(float* y, size_t y_len, const uint8_t* w, size_t w_len, const float* x,
                   size_t x_len, size_t m, size_t k);
/* tensor_core::rmsnorm_bf16_weight (bf16.rs:231-249). */
int myos_rmsnorm_bf16_weight(float* y, size_t y_len, const uint8_t* w, size_t w_len,
                             const float* x, size_t x_len, float eps);
/* tensor_core::gqa_attn_f32 (gqa.rs:174-218). mask_kind 0 = Full, 1 = Causal (any
 * other value: MYOS_ERR_ARG). */
int myos_gqa_attn_f32(float* y, size_t y_len, const float* q, size_t q_len, const float* k,
                      size_t k_len, const float* v, size_t v_len, size_t num_q_heads,
                      size_t num_kv_heads, size_t head_dim, size_t seq_len, int32_t mask_kind,
                      size_t query_pos);
/* tensor_core::swiglu_mul_f32 (swiglu.rs:125-131). */
int myos_swiglu_mul_f32(float* h, size_t h_len, const float* gate, size_t gate_len,
                        const float* up, size_t up_len);
/* tensor_core::rope_f32 (rope.rs:107-115), one position for every head. */
int myos_rope_f32(float* y, size_t y_len, const float* x, size_t x_len, uint32_t position,
                  size_t head_dim, float theta);
/* model_core::greedy_token (lib.rs:157-167) as the two-stage device argmax. */
int myos_greedy_token(const float* logits, size_t n, uint32_t* out);

/* ---------------------------------------------------------------------------
 * Device-pointer kernels (for callers that already hold HBM buffers, and the
 * isolated GEMV microbench). stream may be 0. No allocation, no sync.
 * ------------------------------------------------------------------------- */

/* y[m] (f32) = W[m,k] (bf16, row-major, 16-byte aligned rows when k%8==0) x[k] (f32). */
int myos_dev_gemv_bf16(float* d_y, const void* d_w, const float* d_x, size_t m, size_t k,
                       void* stream);

/* Greedy generation for nseq independent sequences at once. No direct
 * counterpart in the reference, which decodes one sequence per process
 * (model_core greedy_decode, qwen25_block.rs:765-780): this stands in for
 * running greedy_decode on each prompt. Sequence b's prompt is
 * ids[off_b .. off_b + lens[b]) (prompts concatenated in order);
 * out_ids[b * steps + s] receives its s-th generated id. Every prompt runs
 * through the tensor-core prefill into its own KV slab; each decode step then
 * runs the projections and the head of all sequences as GEMMs (each f32
 * activation as three stacked bf16 terms that sum to it exactly,
 * M = 3 nseq). 1 <= nseq <= 128 and
 * lens[b] + steps <= max_seq; needs a shape the GEMM prefill supports
 * (MYOS_ERR_SHAPE otherwise). The context's own cache and cursor are not
 * touched. */
int myos_batch_generate(myos_ctx* ctx, size_t nseq, const uint32_t* ids, const uint32_t* lens,
                        size_t steps, uint32_t* out_ids);

/* The teacher-forced form of myos_batch_generate (the per-sequence
 * myos_forced_decode, model_core forward_token fed given ids, for a batch):
 * step s of sequence b embeds feed[b*steps + s] instead of the argmax, and
 * argmax_out[b*steps + s] receives the argmax of b's logits before step s
 * (the prediction the fed token is scored against). logits, when non-null,
 * receives every sequence's final logits [nseq][vocab]. Same rules and
 * errors as myos_batch_generate; feed ids must be < vocab. */
int myos_batch_forced_decode(myos_ctx* ctx, size_t nseq, const uint32_t* ids, const uint32_t* lens,
                             size_t steps, const uint32_t* feed, uint32_t* argmax_out,
                             float* logits);

/* Size of the fixed device array that myos_dev_gqa_attn_f32_noalloc takes its
 * scratch from (one per device). */
#define MYOS_NOALLOC_SCRATCH_BYTES (2u << 20)

/* No counterpart in the reference (its attention runs on the host). The same
 * split-KV attention as myos_gqa_attn_f32 (tensor_core::gqa_attn_f32,
 * crates/tensor_core/src/gqa.rs:174-218; same arguments and shape rules, same
 * split geometry and so the same results) on caller-held device buffers
 * y[hq*d], q[hq*d], k[hkv][seq][d], v[hkv][seq][d], for callers that must not
 * allocate: code running while a device-memory budget is fixed (an allocator
 * that owns all free HBM, a pool sized at start-up) or on a path that may not
 * call cudaMalloc/cudaFree, which synchronize the device. It allocates
 * nothing: the split partials and merge counters live in one static device
 * array of MYOS_NOALLOC_SCRATCH_BYTES (2 MiB); a request needing more
 * ((hkv*4 + hq*nsplit*(d+2)*4 bytes, each part rounded up to 256, with
 * nsplit = min(64, ceil(keys/32))) returns MYOS_ERR_SCRATCH_LIMIT before any
 * device work. The counters must be zero at kernel start; each call clears
 * them on its stream first. The first call on a device resolves the array's
 * address (cudaGetSymbolAddress); make that call before any stream capture.
 * Calls share the array: calls that run concurrently (different streams or
 * unordered threads) race and corrupt each other's results. Every pointer
 * must be 4-byte aligned, and with d % 4 == 0 d_k and d_v 16-byte aligned
 * (their rows are read as 16-byte vectors); mask_kind is 0 (Full) or 1
 * (Causal). Other values return MYOS_ERR_ARG before any device work.
 * stream may be 0; asynchronous (no sync). */
int myos_dev_gqa_attn_f32_noalloc(float* d_y, const float* d_q, const float* d_k,
                                  const float* d_v, size_t hq, size_t hkv, size_t d, size_t seq,
                                  int32_t mask_kind, size_t query_pos, void* stream);

/* ---------------------------------------------------------------------------
 * Serving over a paged KV cache (device pointers). No counterpart in the
 * reference, whose cache is one contiguous f32 slab for one sequence
 * (crates/model_core/src/kv_cache.rs:89-125). One serving step of a batch is:
 * tables and slot maps from the requests' lengths (myos_dev_paged_tables);
 * per layer the q/k/v rows normed, rotated and stored into the pages
 * (myos_dev_qk_norm_rope_store) and the attention of each sequence's newest
 * token over its pages (myos_dev_paged_attn); the head's logits put under the
 * requests' controls, with the greedy id (myos_dev_logit_controls).
 *
 * Common rules: the calls run on the current device, on `stream` (0: the
 * default stream) of that device, and every pointer is memory of that device.
 * They allocate nothing, do not synchronize, and can be captured into a graph.
 * A kernel's first call on a device loads it and raises its shared-memory limit,
 * which belongs outside a capture; there are several kernels to a call (by cache
 * type and head_dim, by rows and vocabulary), so make one call of each shape that
 * will be captured. Arguments that the host can see are checked before
 * any device work: MYOS_ERR_ARG for null pointers, invalid options and
 * misaligned addresses or strides, MYOS_ERR_SHAPE for sizes. What only the
 * device can see (lengths, page ids, slots, positions, token ids) is checked
 * there, and never read or written through when out of range; each call says
 * what happens then. Unless a call says otherwise its outputs overlap neither
 * each other nor its inputs. Strides count elements, not bytes. A call with no
 * rows returns MYOS_OK and does nothing.
 * ------------------------------------------------------------------------- */

/* One layer's paged K/V cache. Element (page, head, slot, i) of K is
 * k[page * page_stride + head * head_stride + slot * slot_stride + i] (V the
 * same, with the same strides), so [page][head][slot][dim] and
 * [page][slot][head][dim] are both possible. head_dim is a multiple of 8, at
 * most 256; page_size at most 65536, a power of two or not; k, v and the
 * strides are multiples of 16 bytes. The token at position p of a sequence
 * lies in page table[p / page_size], slot p % page_size. */
typedef struct myos_paged_kv {
  void* k;
  void* v;
  uint64_t page_stride;
  uint64_t head_stride;
  uint64_t slot_stride;
  uint32_t num_pages;
  uint32_t page_size;
  uint32_t num_kv_heads;
  uint32_t head_dim;
  int32_t kv_dtype; /* enum myos_kv_dtype */
  uint32_t reserved; /* 0 */
} myos_paged_kv;

/* Gives each of nseq requests (at most 16384) the pages that its new tokens
 * need, and maps the step's token rows to cache slots. Request b holds
 * d_ctx_lens[b] tokens in the pages of table row b (d_block_table +
 * b * table_stride, max_blocks entries) and adds d_new_lens[b]; negative
 * lengths count as 0. Rows of the step are packed: request b's are
 * d_seq_starts[b] .. d_seq_starts[b + 1] (written here, nseq + 1 values,
 * clipped to max_rows). New pages come from the END of d_free_pages
 * [0 .. *d_num_free) (free_cap entries; *d_num_free is clipped to it), in
 * request order, and are appended to the table row in place.
 * A request is admitted when its tokens fit the table row (max_blocks *
 * page_size, and at most 2^31 - 1) and the row buffer (max_rows), and the pages
 * needed by the requests up to and including it (those that fit) do not exceed
 * *d_num_free; a request that needs no page is not held up by the free list. A
 * refused request keeps its length, takes no page, and its rows get slot -1.
 * Outputs:
 * per row d_slots (page * page_size + slot in page; -1: none, also where the
 * page id is outside 0 .. num_pages), d_positions (0 without a slot's
 * request), d_row_seq (the request; -1 for rows behind the last one, whose
 * slot is -1 and position 0); per request d_kv_lens, its length after the
 * step; d_result[2]: the free pages left (the next call's *d_num_free, same
 * d_free_pages) and the number of refused requests. d_kv_lens must not be
 * d_ctx_lens and d_result must not hold d_num_free (MYOS_ERR_ARG): blocks of
 * one launch read the one while another block writes the other. */
int myos_dev_paged_tables(int32_t* d_block_table, size_t table_stride, size_t max_blocks,
                          const int32_t* d_ctx_lens, const int32_t* d_new_lens, size_t nseq,
                          const int32_t* d_free_pages, size_t free_cap,
                          const int32_t* d_num_free, uint32_t page_size, uint32_t num_pages,
                          int64_t* d_slots, int32_t* d_positions, int32_t* d_row_seq,
                          size_t max_rows, int32_t* d_kv_lens, int32_t* d_seq_starts,
                          int32_t* d_result, void* stream);

/* One pass over the q|k|v rows of a projection (f32; row r at d_qkv +
 * r * qkv_stride: num_q_heads, then kv->num_kv_heads key heads, then as many
 * value heads, head_dim each): per-head RMSNorm of q and k with a BF16 weight
 * of head_dim values (d_q_gamma, d_k_gamma; null: that one is not normed, the
 * Qwen2.5 form), NeoX rotation of each q and k head's first rot_dim values
 * (pairs i, i + rot_dim / 2; the rest passes through; 0: no rotation) by row
 * d_positions[r] of the tables d_cos, d_sin [num_pos][rot_dim / 2]
 * (myos_rope_table), then q to d_q (row r at r * q_stride, num_q_heads *
 * head_dim values) and K, V to slot d_slots[r] of the cache, in its type
 * (bf16: round to nearest even). A row whose slot is outside the cache
 * (negative: padding) is not stored, its q is computed. A row whose position
 * is outside the tables is not stored and its q is NaN. d_q may be d_qkv (same
 * stride, in place); two rows of one call must not name the same slot.
 * rot_dim is a multiple of 8 and at most head_dim; all f32 pointers and row
 * strides are multiples of 16 bytes, the weights 8-byte aligned. Order of the
 * steps as in myos_rmsnorm_bf16_weight and myos_rope_f32. */
int myos_dev_qk_norm_rope_store(float* d_q, size_t q_stride, const float* d_qkv,
                                size_t qkv_stride, size_t rows, size_t num_q_heads,
                                const myos_paged_kv* kv, const void* d_q_gamma,
                                const void* d_k_gamma, float eps, const float* d_cos,
                                const float* d_sin, size_t num_pos, size_t rot_dim,
                                const int32_t* d_positions, const int64_t* d_slots, void* stream);

/* Bytes of the work buffer of myos_dev_paged_attn. */
#define MYOS_PAGED_WORK_BYTES (16u << 20)

/* Attention of one new token per sequence over the cache: out[b] (num_q_heads
 * * head_dim f32 at b * out_stride) = softmax(scale * q[b] . K) V over the keys
 * at positions [max(0, len - window), len) of sequence b, len = d_kv_lens[b]
 * clipped to [0, max_blocks * page_size], window 0: all; query head h reads
 * KV head h / (num_q_heads / num_kv_heads), a group of at most 8 (as in
 * tensor_core::gqa_attn_f32); (max_blocks * page_size / 32 + 1) * nseq *
 * num_kv_heads is below 2^31. d_lse (nullable, [nseq][num_q_heads]) receives
 * the natural log of the sum of exp(scale * q . k). Keys of a page whose table
 * entry is outside the cache are left out. A sequence with no keys gives zeros
 * and lse -inf. Slots behind len are never read, whatever they hold; the keys
 * and values that are attended to, q and scale are finite (keys of an f32 cache
 * and q with it below 2^128 - 2^116), but for a query head of NaN (the store's
 * mark of a row without angles), whose out and lse are NaN.
 * d_work: MYOS_PAGED_WORK_BYTES of device memory, 16-byte aligned, zeroed once
 * before its first use; each call leaves it ready for the next. Calls that may
 * run at the same time (other streams, graphs) need buffers of their own.
 * Deterministic: the same inputs give the same bits. q and out pointers and row
 * strides are multiples of 16 bytes. */
int myos_dev_paged_attn(float* d_out, size_t out_stride, float* d_lse, const float* d_q,
                        size_t q_stride, size_t nseq, size_t num_q_heads,
                        const myos_paged_kv* kv, const int32_t* d_block_table,
                        size_t table_stride, size_t max_blocks, const int32_t* d_kv_lens,
                        float scale, uint32_t window, void* d_work, size_t work_bytes,
                        void* stream);

/* The controls of myos_dev_logit_controls; every pointer may be null. */
typedef struct myos_logit_controls_args {
  /* Tokens of each row so far, prompt first: row r at r * history_stride,
   * history_lens[r] of them (clipped to 0 .. history_width; null: all), the
   * first prompt_lens[r] the prompt (null: none). Ids outside the vocabulary
   * are passed over. */
  const int32_t* history;
  uint64_t history_stride;
  uint64_t history_width;
  const int32_t* prompt_lens;
  const int32_t* history_lens;
  /* Per row: a token seen in prompt or output has x / r where x > 0, else
   * x * r; then x - frequency * (times in the output); then x - presence if it
   * is in the output. Null: the step is left out. They need `history`. */
  const float* repetition;
  const float* frequency;
  const float* presence;
  /* Row r adds bias_vals[e] to token bias_ids[e] for e in bias_starts[r] ..
   * bias_starts[r + 1] (clipped to 0 .. num_bias); of several entries of one
   * token the last counts. */
  const int32_t* bias_starts;
  const int32_t* bias_ids;
  const float* bias_vals;
  uint64_t num_bias;
  /* Grammar masks: bit t % 32 of word t / 32 set: token t is allowed, else its
   * logit becomes -inf. Row r uses mask mask_rows[r] (outside 0 .. num_masks:
   * none; null: mask r, for num_masks >= rows). */
  const uint32_t* mask;
  uint64_t mask_stride;
  uint64_t num_masks;
  const int32_t* mask_rows;
} myos_logit_controls_args;

/* Puts the rows of logits [rows][vocab] under the requests' controls, in the
 * order penalties, bias, mask, each step rounded to f32, and picks the greedy
 * id of the result (myos_greedy_token's rule: the first maximum; NaN and -inf
 * never win, a row of nothing else gives 0). d_out receives the controlled
 * logits (may be d_logits with the same stride: in place; null: only the ids),
 * d_ids the ids (null: none); not both null. c null: no controls. vocab,
 * history_width and num_bias are at most 2^30, the last two together below 2^31. */
int myos_dev_logit_controls(float* d_out, size_t out_stride, const float* d_logits,
                            size_t logits_stride, size_t rows, size_t vocab,
                            const myos_logit_controls_args* c, uint32_t* d_ids, void* stream);

/* Host: cos and sin of the rotary angles, [num_pos][rot_dim / 2] f32 each,
 * built as tensor_core::rope_f32 builds its row (rope.rs:186-194). */
int myos_rope_table(float* cos_out, float* sin_out, size_t num_pos, size_t rot_dim, float theta);

/* Library version string and the build's target architecture. */
const char* myos_version(void);

#ifdef __cplusplus
}
#endif
#if defined(__GNUC__)
#pragma GCC visibility pop
#endif
#endif
