/*
 * hllm_rocm: MI355X (gfx950) decoder stage worker, C ABI.
 *
 * One `hllm_rocm_stage` is one loaded stage (a contiguous layer range, plus the token
 * embedding on the first stage and final norm + LM head + sampling on the last) on one
 * GPU. It is the device side of an hLLM `runtime::StageBackend`
 * (cpp/include/hllm/runtime/stage_backend.hpp:69-107) created by a `BackendFactory`
 * (cpp/include/hllm/runtime/backend_factory.hpp:28-47). Plain pointers and sizes only;
 * no exceptions cross this boundary. Every call returns an `hllm_status`; on failure,
 * `hllm_rocm_last_error()` holds a message for the calling thread.
 *
 * Threading mirrors the reference contract: passes on one stage are serialized by the
 * caller's scheduler (cpp/src/worker/scheduler.cpp:60-112); sequence allocation and
 * release may run concurrently with a pass and take the stage's own lock
 * (cpp/src/cuda/stage.cpp:185-202,345).
 */
#ifndef HLLM_ROCM_H
#define HLLM_ROCM_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HLLM_ROCM_ABI_VERSION 2u

/* runtime::ErrorCode (cpp/include/hllm/runtime/error.hpp:10-17), numbered from 1. */
typedef enum {
  HLLM_OK = 0,
  HLLM_INVALID_REQUEST = 1,
  HLLM_INCOMPATIBLE_WORKER = 2,
  HLLM_RESOURCE_EXHAUSTED = 3,
  HLLM_DEADLINE_EXCEEDED = 4,
  HLLM_CANCELLED = 5,
  HLLM_INTERNAL = 6,
} hllm_status;

/* runtime::DataType subset used by dense checkpoints (cpp/include/hllm/runtime/safetensors.hpp:15-29). */
typedef enum { HLLM_DTYPE_F32 = 0, HLLM_DTYPE_F16 = 1, HLLM_DTYPE_BF16 = 2 } hllm_dtype;

typedef struct hllm_rocm_stage hllm_rocm_stage;

/* model::DenseConfig + model::DenseSource ownership (cpp/include/hllm/model/dense_source.hpp:15-44)
 * + the device resources of this worker. */
typedef struct {
  uint32_t abi_version;             /* HLLM_ROCM_ABI_VERSION */
  uint64_t hidden_size;
  uint64_t intermediate_size;
  uint64_t attention_heads;
  uint64_t key_value_heads;
  uint64_t head_dimension;
  uint64_t maximum_sequence_length;
  uint64_t vocabulary_size;
  float rms_norm_epsilon;
  float rope_theta;
  uint32_t query_key_norm;          /* Qwen3 per-head q/k RMSNorm */
  uint32_t layer_start, layer_end;  /* owned layers [start, end) */
  uint32_t first_stage;             /* owns the token embedding */
  uint32_t final_stage;             /* owns final norm, LM head, sampling */
  uint32_t tied_head;               /* LM head is the token embedding */
  uint32_t execution_dtype;         /* HLLM_DTYPE_F16 or HLLM_DTYPE_F32 (plan execution dtype) */
  uint32_t weight_dtype;            /* resident weights: F16, or F32 with F32 execution */
  int32_t device;                   /* HIP device ordinal */
  uint64_t kv_cache_bytes;          /* paged KV pool size; 0 = 90% of free HBM after weights */
  uint32_t kv_block_tokens;         /* tokens per KV block (power of two); 0 = 64 */
  uint32_t max_sequences;           /* live sequence slots; 0 = 512 */
  uint32_t max_pass_rows;           /* rows per pass (prefill chunks + decode rows); 0 = 2048 */
} hllm_rocm_stage_config;

/* One request's share of a pass. */
typedef struct {
  uint32_t sequence;        /* handle from hllm_rocm_sequence_allocate */
  uint32_t query_tokens;    /* rows this item contributes (prefill chunk length, or 1) */
  uint64_t first_position;  /* must equal the sequence's current length */
  uint32_t flags;           /* HLLM_ITEM_* */
  uint32_t top_logprobs;    /* 0..5, with return_logprobs */
  double temperature;       /* runtime::SamplingOptions (cpp/include/hllm/runtime/sampling.hpp:10-17) */
  double top_p;
  uint64_t top_k;
  uint64_t seed;
  uint64_t generated_index; /* counter of the sequence's sampling RNG */
} hllm_rocm_item;

/* The final stage projects the item's last row and samples a token (otherwise the item
 * only extends the KV cache: PrefillProgress, cpp/src/cpu/stage.cpp:164). */
#define HLLM_ITEM_SAMPLE 1u
/* The item's single input token is the token its sequence sampled in its previous pass,
 * read on the device (no host round trip). Only on a stage that is both first and final,
 * and only when the sequence's previous pass sampled (HLLM_INVALID_REQUEST otherwise). */
#define HLLM_ITEM_TOKEN_FROM_DEVICE 2u
/* Return log-probabilities (runtime::SampledToken, cpp/src/sampling.cpp:65-89). */
#define HLLM_ITEM_LOGPROBS 4u

/* A ragged pass: any mix of prefill chunks and decode rows, rows packed in item order. */
typedef struct {
  uint32_t items;
  const hllm_rocm_item* item;
  const uint64_t* token_ids;     /* first stage: sum(query_tokens) IDs in item order */
  const uint16_t* boundary_in;   /* other stages: [sum(query_tokens), hidden] F16 LE */
  /* Optional. Checked before the pass is enqueued, before each layer is enqueued, and once
   * more when the pass completes (cpp/src/cuda/stage.cpp:357,396,456). Set before the
   * device runs the pass, nothing changes; set while it runs, the pass's results are
   * discarded, its sequences are failed (never resumed, cpp/src/cuda/stage.cpp:463-468)
   * and the call returns HLLM_CANCELLED. */
  const volatile int32_t* cancelled;
  /* outputs (host pointers; NULL = not wanted) */
  uint64_t* tokens;              /* final stage: [items]; items without SAMPLE get UINT64_MAX */
  /* For sampled items with HLLM_ITEM_LOGPROBS (runtime::SampledToken): the token's
   * log-probability, and the top_logprobs best tokens and theirs in entries item * 5 + r,
   * r < top_logprobs (later entries UINT64_MAX / NaN). Other items' entries are untouched. */
  double* logprobs;              /* [items] */
  uint64_t* top_ids;             /* [items * 5] */
  double* top_logprobs;          /* [items * 5] */
  uint16_t* boundary_out;        /* non-final: [sum(query_tokens), hidden] F16 LE */
  float* logits;                 /* final: [sampled items, vocabulary] F32, for tests */
  float* trace_hidden;           /* [owned layers, sum(query_tokens), hidden] F32, for tests */
  /* Optional, read at the same points as `cancelled`: cancel_poll(cancel_context) != 0 means
   * the pass is cancelled. For callers whose flag is not an int32_t (the reference's
   * `const std::atomic_bool& cancelled` of StageBackend::execute, stage_backend.hpp:86-89).
   * The context must stay valid until the pass's execute or wait call returns. */
  int32_t (*cancel_poll)(void* cancel_context);
  void* cancel_context;
} hllm_rocm_pass;

typedef struct {
  uint64_t host_bytes;
  uint64_t device_bytes;
  uint64_t pinned_host_bytes;
  uint64_t unified_bytes;
} hllm_rocm_memory;  /* runtime::MemoryAmounts (cpp/include/hllm/runtime/memory.hpp:11-17) */

/* BackendFactory::allocator_metrics (cpp/include/hllm/runtime/backend_factory.hpp:24-33):
 * device memory this library holds on `device`. Stages reserve every buffer when they are
 * created, straight from hipMalloc with no caching layer, so cached_bytes is always 0;
 * peak_bytes is the most held at once since the process started or the last reset. */
typedef struct {
  uint64_t active_bytes;
  uint64_t cached_bytes;
  uint64_t peak_bytes;
} hllm_rocm_allocator_metrics;

/* BackendFactory::profiling_device_info (cpp/include/hllm/runtime/profiling.hpp:8-15; the CUDA
 * worker's cpp/src/cuda/device.cpp:93-108): the device's identity (its UUID as hex digits:
 * 16 as ROCm reports them, or 32 for binary UUIDs), product name (the ISA name when the driver
 * reports none), ISA, HIP runtime and driver versions, compute units and free / total HBM. */
typedef struct {
  char identity[40];
  char name[64];
  char architecture[64];
  int32_t runtime_version;
  int32_t driver_version;
  uint32_t compute_units;
  uint64_t available_bytes;
  uint64_t total_bytes;
} hllm_rocm_device_info;

/* Thread-local message of the last failed call on this thread. */
const char* hllm_rocm_last_error(void);
uint32_t hllm_rocm_abi_version(void);

/* Stage construction, replacing the CUDA worker's CudaStage constructor
 * (cpp/src/cuda/stage.cpp:87-144) and the CPU loader (cpp/src/cpu/stage.cpp:207-255):
 * validate the configuration and reserve every device buffer up front. */
hllm_status hllm_rocm_stage_create(const hllm_rocm_stage_config* config, hllm_rocm_stage** out);
void hllm_rocm_stage_destroy(hllm_rocm_stage* stage);

/* Upload one checkpoint tensor (Safetensors name and row-major LE payload), replacing the
 * per-tensor read + upload of cpp/src/cuda/stage.cpp:123-143. Rejects unknown names,
 * wrong shapes, non-finite values (cpp/src/model/dense_source.cpp:151-153) and values
 * not representable as finite F16 for F16 residency (cpp/src/cuda/stage.cpp:126-133). */
hllm_status hllm_rocm_stage_load_tensor(hllm_rocm_stage* stage, const char* name, uint32_t dtype,
                                        const uint64_t* shape, uint32_t rank, const void* data,
                                        uint64_t bytes);
/* Fill one tensor with the seeded synthetic values (hllm_amd/synthetic.py) on the device. */
hllm_status hllm_rocm_stage_synthesize_tensor(hllm_rocm_stage* stage, const char* name,
                                              uint64_t seed, uint64_t tensor_id, float mean,
                                              float sigma, uint32_t source_dtype);
/* Verify that every owned tensor arrived; the stage accepts passes afterwards. */
hllm_status hllm_rocm_stage_finalize(hllm_rocm_stage* stage);

/* StageBackend::weight_memory / sequence_memory (stage_backend.hpp:72-83). With
 * rows = query_rows(tokens, maximum_query_tokens) (stage_backend.hpp:62-67) and bt the KV
 * block size: cache = {host: tokens * 24 + rows * hidden * 6 (request_transport_bytes,
 * stage_backend.hpp:36-40), device: ceil(tokens / bt) * bt * layers * 2 * kv_heads *
 * head_dim * (2 for F16 KV, 4 for F32 KV)}; workspace = {host: rows * hidden * 6 + 65536,
 * device: 0} (pass workspaces are reserved when the stage is created). tokens = 0 or above
 * maximum_sequence_length is HLLM_INVALID_REQUEST. */
hllm_status hllm_rocm_stage_weight_memory(const hllm_rocm_stage* stage, hllm_rocm_memory* out);
hllm_status hllm_rocm_stage_sequence_memory(const hllm_rocm_stage* stage, uint64_t tokens,
                                            uint64_t maximum_query_tokens,
                                            hllm_rocm_memory* cache, hllm_rocm_memory* workspace);

/* StageBackend::allocate_sequence (stage_backend.hpp:84-85): reserve paged KV for `tokens`
 * positions (HLLM_RESOURCE_EXHAUSTED when the block pool or the sequence slots run out).
 * Release is SequenceState destruction: the handle is invalid at once; when a submitted pass
 * still uses the sequence, its slot and blocks return to the pools when that pass completes. */
hllm_status hllm_rocm_sequence_allocate(hllm_rocm_stage* stage, uint64_t tokens, uint32_t* sequence);
hllm_status hllm_rocm_sequence_release(hllm_rocm_stage* stage, uint32_t sequence);
hllm_status hllm_rocm_sequence_length(const hllm_rocm_stage* stage, uint32_t sequence,
                                      uint64_t* length);

/* StageBackend::execute / execute_decode_batch (stage_backend.hpp:90-101), generalised to
 * ragged passes that mix prefill chunks with decode rows. Synchronous: outputs are on the
 * host when it returns. A pass that fails after touching the KV cache poisons its
 * sequences (cpp/src/cuda/stage.cpp:463-468). */
hllm_status hllm_rocm_stage_execute(hllm_rocm_stage* stage, const hllm_rocm_pass* pass);

/* The same pass, enqueued on the stage's stream without waiting; outputs are valid after
 * hllm_rocm_stage_wait. At most one pass is in flight per stage. */
hllm_status hllm_rocm_stage_submit(hllm_rocm_stage* stage, const hllm_rocm_pass* pass);
hllm_status hllm_rocm_stage_wait(hllm_rocm_stage* stage);

/* One timed phase of a profiled pass: runtime::ComponentTiming
 * (cpp/include/hllm/runtime/timing.hpp:11-15). Components, in pass order: "embedding" or
 * "from-wire", "layer" (layer = its model layer index) per owned layer, then "final_norm",
 * "lm_head" and "sampling" (final stage, when the pass samples) or "to-wire" (other
 * stages); layer is -1 except for "layer". */
typedef struct {
  char component[16];
  int32_t layer;
  double milliseconds;
} hllm_rocm_phase_time;

/* StageBackend::execute_profiled (stage_backend.hpp:103-106): hllm_rocm_stage_execute with
 * HIP events between phases on the stage's stream (no synchronisation inside the pass, so
 * the outputs equal hllm_rocm_stage_execute's bit for bit). Writes up to `capacity` phases
 * and their number to *count. */
hllm_status hllm_rocm_stage_execute_profiled(hllm_rocm_stage* stage, const hllm_rocm_pass* pass,
                                             hllm_rocm_phase_time* phases, uint32_t capacity,
                                             uint32_t* count);

/* runtime::sample_token (cpp/src/sampling.cpp:65-89) on the device for `rows` rows of
 * `vocabulary` F32 logits (host memory), each with the sampling fields of options[r]
 * (temperature, top_p, top_k, seed, generated_index; flags HLLM_ITEM_LOGPROBS and
 * top_logprobs). The stage's sampler, for callers that hold logits of their own. Errors as
 * the reference: invalid options are HLLM_INVALID_REQUEST, non-finite logits HLLM_INTERNAL.
 * Outputs (host) as hllm_rocm_pass's; logprobs / top_ids / top_logprobs may be NULL. */
hllm_status hllm_rocm_sample_logits(int32_t device, const float* logits, uint64_t rows,
                                    uint64_t vocabulary, const hllm_rocm_item* options,
                                    uint64_t* tokens, double* logprobs, uint64_t* top_ids,
                                    double* top_logprobs);

/* No counterpart in the reference: hllm_rocm_sample_logits for callers that cannot allocate
 * device memory (serving loops and harnesses that must not call hipMalloc). Same arguments,
 * results and errors; it allocates nothing (no device or host heap memory, no streams or
 * events): the rows are staged and sampled two at a time through one fixed area of device
 * memory in the library, HLLM_ROCM_NOALLOC_SCRATCH_BYTES per GPU, held from the first call
 * on that GPU until the process ends. Vocabularies above HLLM_ROCM_NOALLOC_MAX_VOCABULARY
 * are HLLM_RESOURCE_EXHAUSTED. Work runs on the device's null stream and the call returns
 * when it is done. Calls on one GPU share the area: the library runs one call at a time per
 * process (a lock), and each call clears what must start at zero; a caller that drives the
 * area's device from elsewhere while a call runs (another process aside) races with it. */
#define HLLM_ROCM_NOALLOC_MAX_VOCABULARY 262144u
#define HLLM_ROCM_NOALLOC_SCRATCH_BYTES 17320704u
hllm_status hllm_rocm_sample_logits_noalloc(int32_t device, const float* logits, uint64_t rows,
                                            uint64_t vocabulary, const hllm_rocm_item* options,
                                            uint64_t* tokens, double* logprobs, uint64_t* top_ids,
                                            double* top_logprobs);

/* Replay of repeated pass shapes (items, rows, sampled rows, sampler use, attention work
 * items) from captured HIP graphs, off by default: a shape's second pass is captured and
 * later ones replay it, with the same kernels and results as eager launches and less host
 * launch work. Passes that request logits, traces or profiling run eagerly. No counterpart
 * in the reference (its CUDA stage launches eagerly). Counters: shapes captured, passes
 * replayed from a graph. */
hllm_status hllm_rocm_stage_set_graphs(hllm_rocm_stage* stage, uint32_t enabled);
hllm_status hllm_rocm_stage_graph_stats(hllm_rocm_stage* stage, uint64_t* captured,
                                        uint64_t* replayed);

/* BackendFactory::allocator_metrics / profiling_reset_peak / profiling_device_info
 * (cpp/include/hllm/runtime/backend_factory.hpp:31-39; cpp/src/cuda/device.cpp:41-54,84-108).
 * reset_peak waits for the device's work to complete, then sets the peak to the bytes held. */
hllm_status hllm_rocm_device_allocator_metrics(int32_t device, hllm_rocm_allocator_metrics* out);
hllm_status hllm_rocm_device_reset_peak(int32_t device);
hllm_status hllm_rocm_device_query(int32_t device, hllm_rocm_device_info* out);

/* Diagnostics: the HBM read ceiling of `device`, measured as the best of five streaming
 * reads of `bytes` (at least 1 MiB, a multiple of 16) with a plain read kernel, in GB/s.
 * For comparing the stage's memory-bound rates with what the device delivers; no
 * counterpart in the reference. */
hllm_status hllm_rocm_measure_read_bandwidth(int32_t device, uint64_t bytes, double* gb_s);

/* Diagnostics: the F16 matrix-core rate of `device` in TFLOP/s with no memory traffic, for
 * v_mfma_f32_16x16x32_f16 (shape 16) or v_mfma_f32_32x32x16_f16 (shape 32): best of five
 * launches of eight workgroups of four waves per CU, each wave running eight independent
 * accumulation chains from registers. The measured ceiling the prefill GEMMs' MFMA fractions
 * are read against beside the 2.5 PFLOP/s dense F16 specification; no counterpart in the
 * reference. */
hllm_status hllm_rocm_measure_mfma_rate(int32_t device, uint32_t shape, double* tflops);

/* Tuning and test hook, process-wide: every later projection GEMM uses configuration
 * `config` of the kernel table (0 .. 18; 17: the decode kernel for every F16 projection of at
 * most 64 rows whose K splits are summed by the consumer or that applies SwiGLU) instead of the
 * choice by shape; -1 restores the
 * choice by shape. *previous (may be NULL) receives the value replaced. Results stay within
 * the execution mode's tolerance for every configuration; no counterpart in the reference.
 * HLLM_ROCM_GEMM_CONFIG gives the initial value. */
hllm_status hllm_rocm_set_gemm_config(int32_t config, int32_t* previous);

/* Diagnostics for parity tests, like the reference's traced execution
 * (cpp/include/hllm/cuda/stage.hpp:8-21): the last pass's device-built packing
 * (cu_seqlens [items + 1], per-row positions and KV slots [rows]), a sequence's physical
 * KV blocks (in logical order), and one layer's cached K and V as F32 [length, kv_heads,
 * head_dim] (the CPU cache order, cpp/src/cpu/llama.cpp:152-158). */
hllm_status hllm_rocm_stage_last_layout(hllm_rocm_stage* stage, uint32_t items, uint32_t rows,
                                        int32_t* cu_seqlens, int32_t* row_positions,
                                        int32_t* row_slots);
hllm_status hllm_rocm_sequence_blocks(hllm_rocm_stage* stage, uint32_t sequence, int32_t* blocks,
                                      uint32_t capacity, uint32_t* count, uint32_t* block_tokens);
/* One loaded tensor back as row-major F32 (hi + lo parts recombined), for loader tests. */
hllm_status hllm_rocm_stage_read_tensor(hllm_rocm_stage* stage, const char* name, float* out,
                                        uint64_t elements);
hllm_status hllm_rocm_sequence_read_kv(hllm_rocm_stage* stage, uint32_t sequence, uint32_t layer,
                                       float* keys, float* values);

/* Profiling hooks for benchmarks: HIP events on the stage's stream around every kernel
 * launched for the operation families named in `families` (';'-separated prefixes such
 * as "gemm_gate_up;attention"; "*" = all; "k:<kernel>" = that kernel only, whichever family
 * launches it; NULL or "" = off). Each family launch carries its
 * algorithmic HBM bytes and FLOPs. Records are kept per family (all kernels of the
 * family's launches), per kernel under "k:<kernel>" (the kernel as rocprofv3 names it,
 * with the bytes and FLOPs of the family launch attributed to its first kernel) and per
 * (family, kernel) pair under "<family>/<kernel>". Read back
 * as sums per record (a trailing '*' matches a prefix); `launches` counts family launches,
 * or kernel launches for "k:" records. */
hllm_status hllm_rocm_stage_profile(hllm_rocm_stage* stage, const char* families);
hllm_status hllm_rocm_stage_profile_read(hllm_rocm_stage* stage, const char* record,
                                         double* milliseconds, uint64_t* launches,
                                         uint64_t* bytes, double* flops);
/* Names of the records collected so far, newline-separated, NUL-terminated in `buffer`
 * (truncated to `capacity` bytes); `needed` receives the full length including the NUL. */
hllm_status hllm_rocm_stage_profile_records(hllm_rocm_stage* stage, char* buffer,
                                            uint64_t capacity, uint64_t* needed);

/* ------------------------------------------------------------ operators on device memory
 *
 * Rotary positions and an 8-bit paged KV cache for callers that hold their activations and
 * their cache in device memory of their own: the stage's rotation, K/V append and decode
 * attention in other forms (positions scaled for long contexts, neighbouring pairs, part of
 * a head; a cache of one byte a value). No counterpart in the reference.
 *
 * Every pointer inside these arguments is device memory of `device` unless it is a host
 * structure named by a type of this header; `stream` is a hipStream_t of that device (NULL:
 * its default stream). A call checks its arguments on the host (HLLM_INVALID_REQUEST, nothing
 * enqueued), enqueues its kernels on `stream` and returns without waiting; it allocates
 * nothing, keeps nothing between calls, leaves the thread's current device as it was and may
 * be captured into a graph. `rows` = 0 enqueues nothing; a call takes at most 2^20 rows, and of
 * very many heads no more than launches of less than 2^32 threads do. Positions, slots, page
 * tables and lengths are read by the device when the kernels run, so a captured call takes what
 * they hold at each replay. Calls may run at once on several streams; what they write must not
 * overlap, and neither may two outputs of one call, a cache's four buffers and a workspace among
 * them (refused where they start at one address). */

/* One tensor [rows][heads][head_dimension]: the last dimension is contiguous, strides are in
 * elements. `data` is 16-byte aligned and so is every head's vector (strides that are
 * multiples of 16 bytes). Inputs may repeat memory (strides of 0); the vectors of an output
 * may not overlap. */
typedef struct {
  void* data;
  uint32_t dtype;        /* HLLM_DTYPE_* */
  uint32_t heads;        /* 1 .. 1024 */
  uint64_t row_stride;
  uint64_t head_stride;
} hllm_rocm_tensor;

/* Which elements of a head's first `rotary_dimension` make the pairs that are rotated:
 * (i, i + rotary_dimension / 2), or (2 i, 2 i + 1). */
typedef enum { HLLM_ROPE_HALF = 0, HLLM_ROPE_INTERLEAVED = 1 } hllm_rope_layout;

/* How pair i's frequency f = theta^(-2 i / rotary_dimension) is changed for contexts longer
 * than the model was trained on:
 *   LINEAR  f / factor
 *   LLAMA3  f / factor for wavelengths 2 pi / f above original_length / low_frequency_factor,
 *           f below original_length / high_frequency_factor, mixed in between
 *   YARN    f / factor for pairs that turn less than `beta_slow` times over original_length, f
 *           for those that turn more than `beta_fast` times, a ramp over the pair indices in
 *           between; cos and sin times `magnitude` (0: 0.1 ln(factor) + 1) */
typedef enum {
  HLLM_ROPE_UNSCALED = 0,
  HLLM_ROPE_LINEAR = 1,
  HLLM_ROPE_LLAMA3 = 2,
  HLLM_ROPE_YARN = 3,
} hllm_rope_scaling;

typedef struct {
  uint32_t rotary_dimension;     /* even, 2 .. 256 */
  uint32_t layout;               /* hllm_rope_layout */
  uint32_t scaling;              /* hllm_rope_scaling; fields it does not use are not read */
  double theta;                  /* > 1 */
  double factor;                 /* >= 1 */
  double original_length;        /* LLAMA3, YARN: > 0 */
  double low_frequency_factor;   /* LLAMA3: > 0 */
  double high_frequency_factor;  /* LLAMA3: > low_frequency_factor */
  double beta_fast;              /* YARN: > beta_slow; 0 = 32 */
  double beta_slow;              /* YARN: > 0; 0 = 1 */
  double magnitude;              /* YARN: >= 0, and so in F32 */
} hllm_rocm_rope_config;

/* A rotation's plan, host memory filled by hllm_rocm_rope_plan and kept by the caller: each
 * pair's frequency in turns (angle / 2 pi) a position, as a 64-bit binary fraction. The
 * fraction of position x frequency is exact in 64-bit integers, of which the upper 32 are kept:
 * at every 32-bit position (negative ones too) angles are right to 2e-9 radians, and their sines
 * and cosines, in F32, to 5e-7. */
typedef struct {
  uint32_t rotary_dimension;
  uint32_t layout;
  float magnitude;
  uint32_t reserved;
  uint64_t turns[128];
} hllm_rocm_rope;

hllm_status hllm_rocm_rope_plan(const hllm_rocm_rope_config* config, hllm_rocm_rope* out);

/* q_out = q and k_out = k (NULL, both: none) rotated at `positions` [rows], computed in F32 and
 * rounded once; elements past the plan's rotary_dimension are copied. head_dimension is a
 * multiple of 16, at most 256 and at least rotary_dimension; all tensors have one dtype. An output
 * may be its own input (same data and strides), and otherwise overlaps no input. */
hllm_status hllm_rocm_rope_apply(int32_t device, void* stream, const hllm_rocm_rope* rope,
                                 const int32_t* positions, uint64_t rows, uint32_t head_dimension,
                                 const hllm_rocm_tensor* q, const hllm_rocm_tensor* q_out,
                                 const hllm_rocm_tensor* k, const hllm_rocm_tensor* k_out);

/* What an 8-bit cache holds of a vector x (a position's key or value of one head): codes and one
 * F32 scale, x ~= code * scale, with scale = max(|x|max, 2^-100) / c and code = x * (c /
 * max(|x|max, 2^-100)) rounded to nearest even: c = 448 for E4M3 (OCP, 8-bit floating point: relative
 * error at most 2^-4, the better for outliers) and 127 for INT8 (whole numbers: error at most
 * |x|max / 254, the smaller for even distributions). A vector with a value that is not finite
 * gets the scale NaN and codes 0: it reads back as NaN. */
typedef enum { HLLM_KV_E4M3 = 0, HLLM_KV_INT8 = 1 } hllm_kv_format;

/* A paged cache in device memory: codes at page * page_stride + position * token_stride + head *
 * head_stride (bytes, multiples of 16; page_stride below 2^32, token_stride at most 2^28; either of
 * positions and heads inside the other; vectors may not overlap) and scales [pages][kv_heads]
 * [page_tokens], for keys and values alike. A slot is page * page_tokens + position in the page. All
 * four pointers are 16-byte aligned. */
typedef struct {
  uint32_t format;          /* hllm_kv_format */
  uint32_t pages;           /* pages * page_tokens < 2^31 */
  uint32_t page_tokens;     /* a power of two, 8 .. 4096 */
  uint32_t kv_heads;        /* 1 .. 1024 */
  uint32_t head_dimension;  /* 64, 128 or 256 */
  uint64_t page_stride;
  uint64_t token_stride;
  uint64_t head_stride;
  void* keys;
  void* values;
  float* key_scales;
  float* value_scales;
} hllm_rocm_kv_pages;

/* Quantises rows of k and v [rows][kv_heads] into the cache at `slots` [rows]. With `rope`, k is rotated at
 * `positions` first (in F32, not rounded in between) and, with q (NULL, both: none), q_out = q
 * rotated, as hllm_rocm_rope_apply does; without `rope`, q must be NULL. A row whose slot is not
 * in [0, pages * page_tokens) is padding: nothing is written for it, q_out included. Slots of
 * other rows must differ: what is left in a slot that two rows name is not specified. */
hllm_status hllm_rocm_kv_append(int32_t device, void* stream, const hllm_rocm_kv_pages* pages,
                                const int32_t* slots, uint64_t rows, const hllm_rocm_tensor* k,
                                const hllm_rocm_tensor* v, const hllm_rocm_rope* rope,
                                const int32_t* positions, const hllm_rocm_tensor* q,
                                const hllm_rocm_tensor* q_out);

/* The cached vectors at `slots` [rows] (any order, repeats allowed) as k_out and v_out
 * [rows][kv_heads], code * scale in F32 rounded once. Rows whose slot is not in the cache are
 * padding and left as they were. */
hllm_status hllm_rocm_kv_read(int32_t device, void* stream, const hllm_rocm_kv_pages* pages,
                              const int32_t* slots, uint64_t rows, const hllm_rocm_tensor* k_out,
                              const hllm_rocm_tensor* v_out);

/* One new token's attention for each row, over a sequence in the cache: out = softmax(scale q
 * K^T) V with the keys and values of positions 0 .. lengths[row] - 1 of the row's pages; query
 * heads share KV heads in groups of q.heads / kv_heads. Scores, softmax and sums are F32; products
 * take codes exactly, and q and the weights as F16 (F16 and BF16 tensors, each vector's largest
 * weight scaled to 1) or as sums of two F16 values (F32 tensors). Weights below 2^-126 of a row's largest may be lost, scores past
 * 2^23 (times log2 e) are as F32 rounds them, and outputs may be off by 2^-115 besides.
 *
 * A row's length counts at most max_length and table_width * page_tokens positions; a length
 * of 0 gives zeros and a negative one marks a padding row, which is left as it was. Positions in
 * pages outside [0, pages) take no part, as if they were masked (a dropped page is -1); a row
 * with no other position gives zeros. NaN scores, and scores that are all -inf (an infinite query),
 * give NaN. What lies in a page behind a row's length is not used, NaN or not. */
typedef struct {
  uint64_t rows;
  const int32_t* page_table;  /* [rows][table_width], rows table_stride entries apart */
  uint64_t table_width;       /* table_width * page_tokens at most 2^30 */
  uint64_t table_stride;
  const int32_t* lengths;     /* [rows] */
  uint64_t max_length;        /* the host's bound of the lengths: work is split for it */
  float scale;
  hllm_rocm_tensor q;
  hllm_rocm_tensor out;       /* q's dtype and heads; not overlapping q */
  void* workspace;            /* 16-byte aligned; used while the call's kernels run, so calls that
                               * may run at once need one each; no contents are required */
  uint64_t workspace_bytes;   /* at least hllm_rocm_kv_attention_workspace */
} hllm_rocm_kv_attention_args;

hllm_status hllm_rocm_kv_attention(int32_t device, void* stream, const hllm_rocm_kv_pages* pages,
                                   const hllm_rocm_kv_attention_args* args);
/* ... with pages of its own for each KV head: head h of a row finds them table_head_stride * h entries after
 * the row's (0: every head the same), as a selection of pages by head leaves them. `lengths` counts the
 * positions of those pages, the same for all heads of a row. */
hllm_status hllm_rocm_kv_attention_by_head(int32_t device, void* stream, const hllm_rocm_kv_pages* pages,
                                           const hllm_rocm_kv_attention_args* args,
                                           uint64_t table_head_stride);
/* The workspace that does for a call with `rows` rows of `query_heads` heads and this max_length or a
 * smaller one (0: none, and `workspace` may be NULL). For this number of rows: of many rows none is cut, and fewer may need more, so
 * one workspace for batches of several sizes has the largest of their sizes. Needs no device. */
hllm_status hllm_rocm_kv_attention_workspace(const hllm_rocm_kv_pages* pages, uint64_t rows,
                                             uint32_t query_heads, uint64_t max_length,
                                             uint64_t* bytes);

/* What a 4-bit cache holds of 32 elements x that follow one another in a vector, a group: codes and one scale, x ~= value of
 * the code * scale. A group with an element that is not finite holds the scale NaN and reads back as NaN, its
 * vector's other groups as they are.
 *   E2M1  (OCP microscaling) codes of the numbers 0, 1/2, 1, 3/2, 2, 3, 4, 6, the fourth bit their sign; the scale is a
 *         power of two, the byte e + 127 (0: 2^-127; 255: NaN). Written with the smallest e that leaves max(|x|max, 2^-100)
 *         at most 7 * 2^e, but at most 125; x / 2^e is rounded to the nearest number, ties to the even code, 6 standing
 *         for all that is larger. Off by at most 2^e: 2/7 of |x|max (of the largest numbers more).
 *   INT4  codes -7 .. 7, held as code + 8; the scale is BF16 (the upper half of an F32 number; one that is not finite
 *         counts as NaN). Written with scale = max(|x|max, 2^-100) / 7 in F32, its lower half cut off, and code =
 *         x * (1 / scale) rounded to nearest even, at most 7: off by half a scale and 2^-7 |x|max at most.
 * Two codes lie in a byte, the lower four bits first. A key's codes lie in order: byte i holds elements 2 i and 2 i + 1. A
 * value's bytes go round its G = head_dimension / 32 groups: byte G c + g holds elements 32 g + 2 c and 32 g + 2 c + 1. */
typedef enum { HLLM_KV4_E2M1 = 0, HLLM_KV4_INT4 = 1 } hllm_kv4_format;

/* A paged 4-bit cache: as hllm_rocm_kv_pages, with head_dimension / 2 bytes a vector and
 * head_dimension / 32 scales, [pages][kv_heads][page_tokens][head_dimension / 32]. */
typedef struct {
  uint32_t format;          /* hllm_kv4_format */
  uint32_t pages;
  uint32_t page_tokens;
  uint32_t kv_heads;
  uint32_t head_dimension;  /* 64, 128 or 256 */
  uint64_t page_stride;     /* bytes, as in hllm_rocm_kv_pages */
  uint64_t token_stride;
  uint64_t head_stride;
  void* keys;
  void* values;
  void* key_scales;         /* E2M1: bytes; INT4: BF16 */
  void* value_scales;
} hllm_rocm_kv4_pages;

/* The 8-bit cache's operators over a 4-bit one, to the same rules. In attention E2M1 keys enter their products exactly, and an INT4
 * key's scale multiplies its group's part of the score in F32; a finite key's and query's products stay finite for
 * keys below 2^115. A value's scale enters its weight, which is F16 for 16-bit tensors (rounded once, beside INT4 values
 * twice; weights below 2^-25 of a wave's largest may be lost, and so may a group's scale below 2^-25 of the largest of its vector, an
 * INT4 one's last bits from 2^-17 down) and two F16 parts for F32 ones. Beside 16-bit tensors the values' scales, each
 * vector's largest one, lie within 2^180 of one another in a row (those of 0 apart): farther apart the output may be off by
 * more. `table_head_stride` as for hllm_rocm_kv_attention_by_head. */
hllm_status hllm_rocm_kv4_append(int32_t device, void* stream, const hllm_rocm_kv4_pages* pages,
                                 const int32_t* slots, uint64_t rows, const hllm_rocm_tensor* k,
                                 const hllm_rocm_tensor* v, const hllm_rocm_rope* rope,
                                 const int32_t* positions, const hllm_rocm_tensor* q,
                                 const hllm_rocm_tensor* q_out);
hllm_status hllm_rocm_kv4_read(int32_t device, void* stream, const hllm_rocm_kv4_pages* pages,
                               const int32_t* slots, uint64_t rows, const hllm_rocm_tensor* k_out,
                               const hllm_rocm_tensor* v_out);
hllm_status hllm_rocm_kv4_attention(int32_t device, void* stream, const hllm_rocm_kv4_pages* pages,
                                    const hllm_rocm_kv_attention_args* args, uint64_t table_head_stride);
hllm_status hllm_rocm_kv4_attention_workspace(const hllm_rocm_kv4_pages* pages, uint64_t rows,
                                              uint32_t query_heads, uint64_t max_length,
                                              uint64_t* bytes);

/* The bounds of a cache's pages, kept by the caller beside the cache: for each page and KV head the largest ([0]) and the
 * smallest ([1]) key element of each channel over the page's positions, as whole numbers times one power of two, the
 * smallest that leaves max(|x|max, 2^-100) of both at most 127 times it; x / scale is rounded to nearest even. Elements are
 * what reading back gives in F32. A page and head with an element that is not finite has codes of 0 and the
 * scale NaN. Both pointers are 16-byte aligned; sizes are the cache's. */
typedef struct {
  uint32_t pages;
  uint32_t page_tokens;
  uint32_t kv_heads;
  uint32_t head_dimension;
  int8_t* codes;            /* [pages][kv_heads][2][head_dimension] */
  float* scales;            /* [pages][kv_heads] */
} hllm_rocm_kv_bounds;

/* Makes the bounds of the pages that hold positions starts[row] .. lengths[row] - 1 of each row (a negative start counts as
 * 0), from all positions of those pages below lengths[row]: after a write of these positions. A row whose start is not
 * below its length, and pages outside the cache, have nothing made. Pages are made for max_new positions of a row from its start
 * on (and maybe the page behind them), within table_width pages: rows * these pages * kv_heads below 2^24. Rows may share a page if
 * their lengths agree on it. */
typedef struct {
  uint64_t rows;
  const int32_t* page_table;  /* [rows][table_width], rows table_stride entries apart */
  uint64_t table_width;
  uint64_t table_stride;
  const int32_t* starts;      /* [rows] */
  const int32_t* lengths;     /* [rows] */
  uint64_t max_new;           /* the host's bound of lengths - starts */
} hllm_rocm_kv_bounds_args;

hllm_status hllm_rocm_kv_bounds_update(int32_t device, void* stream, const hllm_rocm_kv_pages* pages,
                                       const hllm_rocm_kv_bounds* bounds,
                                       const hllm_rocm_kv_bounds_args* args);
hllm_status hllm_rocm_kv4_bounds_update(int32_t device, void* stream, const hllm_rocm_kv4_pages* pages,
                                        const hllm_rocm_kv_bounds* bounds,
                                        const hllm_rocm_kv_bounds_args* args);

/* Selects `keep` pages of each row for each KV head: its first `first` and last `last` pages (last at least 1, first + last at
 * most keep), and of the others those with the largest scores, of equal scores the first. A page's score is the largest,
 * over the KV head's query heads, of the sum over channels of max(q high, q low), with q as whole numbers times a power of
 * two by the bounds' rule: a sum of whole numbers below 2^24, times the query's scale and then the page's, in F32. That is exact
 * where it is in F32's normal range, so a selection depends on nothing but its row. A score that is NaN (a page or query that is not
 * finite) is above all others, a page outside the cache below them.
 *
 * selected [rows][kv_heads][keep] gets the selected entries of the row's page table in their order, -1 behind them
 * where the row has fewer pages, and selected_lengths [rows] the positions that they hold: what
 * hllm_rocm_kv_attention_by_head and hllm_rocm_kv4_attention take as a table of rows kv_heads * keep entries apart
 * and heads `keep` apart. A row's length counts at most max_length and table_width * page_tokens positions. A
 * negative length marks a padding row: it is passed on and the row's part of `selected` left as it was. rows * kv_heads is below
 * 2^24, where rows may have more than 512 pages below 2^22. */
typedef struct {
  uint64_t rows;
  const int32_t* page_table;
  uint64_t table_width;       /* table_width * page_tokens at most 2^30, keep * page_tokens too */
  uint64_t table_stride;
  const int32_t* lengths;
  uint64_t max_length;
  uint32_t keep;
  uint32_t first;
  uint32_t last;
  hllm_rocm_tensor q;         /* [rows][heads], heads a multiple of the cache's */
  int32_t* selected;
  int32_t* selected_lengths;
  void* workspace;            /* as in hllm_rocm_kv_attention_args, of hllm_rocm_kv_select_workspace bytes */
  uint64_t workspace_bytes;
} hllm_rocm_kv_select_args;

hllm_status hllm_rocm_kv_select(int32_t device, void* stream, const hllm_rocm_kv_bounds* bounds,
                                const hllm_rocm_kv_select_args* args);
/* The workspace that does for `rows` rows, this max_length or a smaller one and this `keep` or a larger one (0: none); fewer
 * rows may need more, as for hllm_rocm_kv_attention_workspace. Needs no device. */
hllm_status hllm_rocm_kv_select_workspace(const hllm_rocm_kv_bounds* bounds, uint64_t rows,
                                          uint64_t max_length, uint32_t keep, uint64_t* bytes);

#ifdef __cplusplus
}
#endif
#endif
