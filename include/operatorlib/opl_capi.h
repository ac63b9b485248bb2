#ifndef OPERATORLIB_OPL_CAPI_H_
#define OPERATORLIB_OPL_CAPI_H_

/* C-ABI of the B200 operator library (libopl_b200.so).
 *
 * Plain pointers, sizes and an opaque stream handle; no C++ or torch types,
 * so any FFI (ctypes, cffi, cgo, JNI) can bind it directly.  Each function
 * returns an int that is a cudaError_t value (0 == cudaSuccess,
 * 1 == cudaErrorInvalidValue for rejected arguments).  All pointers are
 * caller-owned device memory on the current device; outputs are
 * pre-allocated; work is only enqueued on `stream` (NULL = legacy default
 * stream) and nothing synchronises.  The C++ functions declared in
 * operatorlib/operators.h forward one-to-one to these entry points.
 *
 * Each entry point names the reference interface it replaces
 * (file:line in the reference project).
 */

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Same type as cudaStream_t (struct CUstream_st*), spelled without
 * including CUDA headers. */
typedef struct CUstream_st* opl_stream_t;

/* FP16 storage (IEEE binary16 bits), layout-compatible with __half. */
typedef uint16_t opl_half_t;

/* BF16 storage (bfloat16 bits), layout-compatible with __nv_bfloat16. */
typedef uint16_t opl_bf16_t;

/* Replaces operatorlib::reduce_sum_f32, include/operatorlib/operators.h:13-14
 * (implementation src/reduce.cu:54-69).  Sum of n floats, accumulated in
 * FP64 per block and combined in a fixed order: deterministic.  Uses a
 * stream-ordered workspace (cudaMallocAsync/cudaFreeAsync on `stream`). */
int opl_reduce_sum_f32(const float* input, float* output, size_t n,
                       opl_stream_t stream);

/* Multi-GPU building block with no single-call counterpart in the reference:
 * the same deterministic sum as opl_reduce_sum_f32 but written as one FP64
 * value, so per-GPU chunk partials can be all-reduced in FP64 before the
 * final cast (the reference combines block partials with a float atomicAdd,
 * src/reduce.cu:46). */
int opl_reduce_sum_partial_f64(const float* input, double* output, size_t n,
                               opl_stream_t stream);

/* No counterpart in the reference.  opl_reduce_sum_f32 without any
 * allocation, for callers that may not call cudaMalloc/cudaMallocAsync (code
 * inside allocator hooks or pool callbacks, frameworks that own all device
 * memory, fixed memory budgets).  Partial sums go to a fixed file-scope
 * device array of 4096 FP64 slots (32 KiB, held by every GPU that loads the
 * library until exit); the partial-sum grid never exceeds 4096 CTAs, so any
 * n fits.  The first call on each device looks the array up
 * (cudaGetSymbolAddress), caches the address and must come before any stream
 * capture; the cached address does not survive cudaDeviceReset.  All calls
 * share the array: calls that overlap on the GPU race; serialise them on one
 * stream.  Bit-identical result to opl_reduce_sum_f32. */
int opl_reduce_sum_f32_noalloc(const float* input, float* output, size_t n,
                               opl_stream_t stream);

/* Multi-GPU reduce fused with its all-reduce (no reference counterpart: the
 * reference is single-GPU; it replaces "per-GPU reduce + NCCL all-reduce").
 * A team is one rank per GPU of a node.  opl_team_create allocates this
 * GPU's team buffer and returns its CUDA IPC handle (64 bytes) to share with
 * the other ranks; opl_team_connect opens the peers' buffers from the
 * world * 64-byte array of all handles (rank order).  Every rank then calls
 * opl_team_reduce_sum_f32 on its own chunk, in the same order on all ranks:
 * each GPU sums its chunk, exchanges the FP64 partial with the peers over
 * NVLink and writes the identical total to *output.  A peer that does not
 * arrive within a bounded wait (about 2 s) yields NaN and the watchdog code.
 * A timeout is final for the team: every later call on that rank returns NaN
 * at once, the other ranks time out on their next call and do the same, and
 * the team has to be destroyed (opl_team_destroy) and created again. */
int opl_team_create(int rank, int world, void** team, void* ipc_handle_out);
int opl_team_connect(void* team, const void* all_ipc_handles);
int opl_team_reduce_sum_f32(void* team, const float* input, float* output, size_t n,
                            opl_stream_t stream);
int opl_team_destroy(void* team);

/* Replaces operatorlib::softmax_f32, operators.h:16-17 (src/softmax.cu:182-202). */
int opl_softmax_f32(const float* input, float* output, int rows, int cols,
                    opl_stream_t stream);

/* 16-bit I/O variants of softmax_f32 and rmsnorm_f32 (no counterpart in the
 * reference, whose launchers are FP32-only; it defers 16-bit I/O to a later
 * interface stage, docs/standalone_benchmark.md:14-16).  Inputs, weight and
 * outputs in FP16 or BF16; max / sums / normalisation in FP32; each result
 * rounded once to the storage type.  Same argument checks as the FP32
 * versions. */
int opl_softmax_f16(const opl_half_t* input, opl_half_t* output, int rows, int cols,
                    opl_stream_t stream);
int opl_softmax_bf16(const opl_bf16_t* input, opl_bf16_t* output, int rows, int cols,
                     opl_stream_t stream);
int opl_rmsnorm_f16(const opl_half_t* input, const opl_half_t* weight, opl_half_t* output,
                    int tokens, int hidden, float epsilon, opl_stream_t stream);
int opl_rmsnorm_bf16(const opl_bf16_t* input, const opl_bf16_t* weight, opl_bf16_t* output,
                     int tokens, int hidden, float epsilon, opl_stream_t stream);

/* Replaces operatorlib::transpose_f32, operators.h:19-20
 * (src/transpose.cu:38-47).  Bit-exact data movement. */
int opl_transpose_f32(const float* input, float* output, int rows, int cols,
                      opl_stream_t stream);

/* Replaces operatorlib::rmsnorm_f32, operators.h:22-24 (src/rmsnorm.cu:77-95).
 * epsilon <= 0 (or NaN) is rejected like the reference (src/rmsnorm.cu:80-82). */
int opl_rmsnorm_f32(const float* input, const float* weight, float* output,
                    int tokens, int hidden, float epsilon, opl_stream_t stream);

/* Replaces operatorlib::gemm_f32, operators.h:27-28 (src/gemm.cu:440-453).
 * Row-major C[M,N] = A[M,K] * B[K,N] on FP32 FFMA (no TF32 rounding). */
int opl_gemm_f32(const float* a, const float* b, float* c, int m, int n, int k,
                 opl_stream_t stream);

/* Replaces operatorlib::gemm_f16, operators.h:31-32 (src/gemm.cu:455-479).
 * FP16 A and B, tcgen05 tensor cores, FP32 accumulate and FP32 C.
 * Shapes whose row strides are not 16-byte multiples are staged through a
 * zero-padded stream-ordered workspace. */
int opl_gemm_f16(const opl_half_t* a, const opl_half_t* b, float* c, int m,
                 int n, int k, opl_stream_t stream);

/* Replaces operatorlib::attention_f32, operators.h:35-38
 * (src/attention.cu:445-484).  [B,H,S,D] contiguous, D <= 128, FP32 FFMA. */
int opl_attention_f32(const float* q, const float* k, const float* v,
                      float* output, int batch, int heads, int sequence,
                      int head_dim, int causal, opl_stream_t stream);

/* Replaces operatorlib::attention_f16, operators.h:41-44
 * (src/attention.cu:486-507).  FP16 Q/K/V, FP32 softmax state and output. */
int opl_attention_f16(const opl_half_t* q, const opl_half_t* k,
                      const opl_half_t* v, float* output, int batch, int heads,
                      int sequence, int head_dim, int causal,
                      opl_stream_t stream);

/* Decoding with a paged key-value cache (no counterpart in the reference,
 * whose attention takes whole contiguous [B,H,S,D] tensors): rotary positions,
 * appending to the cache, attention of one new token over it.  Tensors may
 * have any strides (in elements, not negative) as long as head_dim is
 * contiguous; head_dim is at most 256.  Addresses and strides that are multiples of 16 bytes take
 * the widest loads.  Indices that the device reads (slots, block table,
 * lengths) are checked there: a bad one is not followed, and its code is left
 * in the watchdog word (opl_read_and_clear_watchdog): 0x6b01 slot past the
 * cache, 0x6b02 block-table entry outside the cache, 0x6b03 length negative or
 * past the sequence's row of the block table. */

/* A rotary embedding.  Pair i of the rot_dim / 2 pairs (elements i and
 * i + rot_dim / 2, or 2i and 2i + 1 when `adjacent`) is turned by
 * positions[axis][token] * inv_freq[i]; the first sections[0] pairs belong to
 * axis 0, the next sections[1] to axis 1, and so on (video: time, height,
 * width).  `inverse` turns back: the transposed matrix, which is also the
 * gradient of the rotation.  rot_dim is even and at most head_dim; elements
 * past it are copied; 0 rotates nothing and needs no pointers.  Angles are
 * formed in FP64, the rotation in FP32, and each result is rounded once. */
typedef struct opl_rope_spec {
  const int64_t* positions; /* device, [axes][tokens] */
  const float* inv_freq;    /* device, [rot_dim / 2] */
  int rot_dim;
  int axes;                 /* 1 to 4 */
  int sections[4];          /* sum over the axes: rot_dim / 2 */
  int adjacent;
  int inverse;
} opl_rope_spec;

/* Keys and values in pages: token i of page p for key-value head h starts at
 * k + p * k_page + i * k_token + h * k_head (v alike). */
typedef struct opl_kv_cache {
  void* k;
  void* v;
  int64_t pages;
  int page_size;
  int kv_heads;
  int head_dim;
  int64_t k_page, k_token, k_head;
  int64_t v_page, v_token, v_head;
} opl_kv_cache;

/* out[t][h] = rotated x[t][h], [tokens, heads, head_dim].  out is x itself
 * (same strides) or does not overlap it. */
int opl_rope_f32(const float* x, float* out, int tokens, int heads, int head_dim,
                 int64_t x_token, int64_t x_head, int64_t out_token, int64_t out_head,
                 const opl_rope_spec* rope, opl_stream_t stream);
int opl_rope_f16(const opl_half_t* x, opl_half_t* out, int tokens, int heads, int head_dim,
                 int64_t x_token, int64_t x_head, int64_t out_token, int64_t out_head,
                 const opl_rope_spec* rope, opl_stream_t stream);
int opl_rope_bf16(const opl_bf16_t* x, opl_bf16_t* out, int tokens, int heads, int head_dim,
                  int64_t x_token, int64_t x_head, int64_t out_token, int64_t out_head,
                  const opl_rope_spec* rope, opl_stream_t stream);

/* Rotates the new tokens' queries into q_out and their keys into the cache,
 * and copies their values there: token t goes to token slots[t] % page_size
 * of page slots[t] / page_size.  A negative slot keeps the token out of the
 * cache (padding; its query is rotated all the same).  The slots that are not
 * negative have to be distinct: of two tokens with the same slot either may
 * win, element by element.  Nothing else of the cache is touched; its keys and
 * values share no memory.  q is [tokens, heads, head_dim]; k and v are
 * [tokens, kv_heads, head_dim]; none of them overlaps the cache (tokens are not
 * moved within it by this call); q_out is q itself or overlaps nothing. */
int opl_kv_append_f32(const float* q, int64_t q_token, int64_t q_head, const float* k,
                      int64_t k_token, int64_t k_head, const float* v, int64_t v_token,
                      int64_t v_head, float* q_out, int64_t out_token, int64_t out_head,
                      const opl_kv_cache* cache, const int64_t* slots, int tokens, int heads,
                      const opl_rope_spec* rope, opl_stream_t stream);
int opl_kv_append_f16(const opl_half_t* q, int64_t q_token, int64_t q_head, const opl_half_t* k,
                      int64_t k_token, int64_t k_head, const opl_half_t* v, int64_t v_token,
                      int64_t v_head, opl_half_t* q_out, int64_t out_token, int64_t out_head,
                      const opl_kv_cache* cache, const int64_t* slots, int tokens, int heads,
                      const opl_rope_spec* rope, opl_stream_t stream);
int opl_kv_append_bf16(const opl_bf16_t* q, int64_t q_token, int64_t q_head, const opl_bf16_t* k,
                       int64_t k_token, int64_t k_head, const opl_bf16_t* v, int64_t v_token,
                       int64_t v_head, opl_bf16_t* q_out, int64_t out_token, int64_t out_head,
                       const opl_kv_cache* cache, const int64_t* slots, int tokens, int heads,
                       const opl_rope_spec* rope, opl_stream_t stream);

/* Attention of one new token per sequence: q and out are [batch, heads,
 * head_dim] (out contiguous, overlapping nothing), query head h reads key-value head
 * h / (heads / kv_heads), and sequence b has seq_lens[b] keys, key j in page
 * block_table[b * table_row + j / page_size].  Softmax over scale * q.K in
 * FP32; the result is rounded once to the tensors' type.  Keys of a page outside
 * the cache are left out.  A sequence without keys (of length 0, or with all of
 * its pages outside) gives zeros.  Table entries past a sequence's pages are not
 * read.  A page's tokens past its length may be fetched together with those in
 * front of them, but what they hold, or what is being written there, does not
 * matter.  max_pages * page_size is at most 2^30, and batch times that at most
 * 2^34.
 * `workspace` is 16-byte aligned device memory of at least the size that
 * opl_paged_attention_workspace gives; its contents do not matter and need not
 * be kept, but two calls that may overlap on the GPU need one each. */
int opl_paged_attention_workspace(int heads, int kv_heads, int head_dim, size_t* bytes);
int opl_paged_attention_f32(const float* q, int64_t q_batch, int64_t q_head,
                            const opl_kv_cache* cache, const int* block_table, int64_t table_row,
                            int max_pages, const int* seq_lens, float* out, int batch, int heads,
                            float scale, void* workspace, size_t workspace_bytes,
                            opl_stream_t stream);
int opl_paged_attention_f16(const opl_half_t* q, int64_t q_batch, int64_t q_head,
                            const opl_kv_cache* cache, const int* block_table, int64_t table_row,
                            int max_pages, const int* seq_lens, opl_half_t* out, int batch,
                            int heads, float scale, void* workspace, size_t workspace_bytes,
                            opl_stream_t stream);
int opl_paged_attention_bf16(const opl_bf16_t* q, int64_t q_batch, int64_t q_head,
                             const opl_kv_cache* cache, const int* block_table, int64_t table_row,
                             int max_pages, const int* seq_lens, opl_bf16_t* out, int batch,
                             int heads, float scale, void* workspace, size_t workspace_bytes,
                             opl_stream_t stream);

/* Library utilities (no reference counterpart). */

/* cudaGetErrorString of an error code returned above. */
const char* opl_error_string(int error);

/* Reads and clears the per-device watchdog word of the current device.
 * Kernels whose pipelines wait on mbarriers give up after a bounded number
 * of polls, record a non-zero code here and exit instead of hanging the
 * GPU.  Synchronises the current device (diagnostics only). */
int opl_read_and_clear_watchdog(int* code);

/* Library version, e.g. "opl-b200 0.1.0 sm_100a". */
const char* opl_version(void);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* OPERATORLIB_OPL_CAPI_H_ */
