/*
 * kvfx.h - C ABI of the B200 (sm_100a) paged-KV data path.
 *
 * Plain pointers and sizes only: no C++ or torch types cross this boundary, so
 * any FFI (ctypes, cgo, JNI, N-API) can bind it. Every entry point is
 * stream-ordered: it enqueues work on `stream` (a cudaStream_t; NULL is the
 * legacy default stream) and returns without synchronising. Device arrays
 * must be resident on `cache->device`. Return value: KVFX_OK or an error code;
 * kvfx_last_error() gives a message for the calling thread's last failure.
 *
 * The cache layout is the reference's single-layer paged layout
 * (src/v2/paged_kv_layout.cpp:27-68 in KVFlux):
 *     K[num_blocks][num_kv_heads][block_size][head_size], then V alike,
 * and a slot id is physical_block * block_size + offset_in_block
 * (src/v2/slot_mapping.cpp:29).
 *
 * These entry points trust the tables they are given only as far as memory
 * safety: a slot or block id at or beyond the cache is skipped (writes) or
 * read as nothing, and sets KVFX_FLAG_BAD_INDEX in the device status word
 * (kvfx_device_status). The C++ API in include/kvflux/v2 validates everything
 * on the host first and raises the reference's exception types.
 */
#ifndef KVFX_H
#define KVFX_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Return codes. */
#define KVFX_OK 0
#define KVFX_EINVAL 1       /* bad argument: null pointer, bad shape or dtype   */
#define KVFX_ERANGE 2       /* index outside the cache                           */
#define KVFX_EOVERFLOW 3    /* size arithmetic overflow                          */
#define KVFX_ECUDA 4        /* CUDA runtime error (message in kvfx_last_error)   */
#define KVFX_ETIMEOUT 5     /* a bounded device-side wait gave up                */
#define KVFX_ENOSPACE 6     /* workspace smaller than the *_workspace_bytes size */

/* Cache element types (same order as kvflux::DType). */
#define KVFX_F16 0
#define KVFX_BF16 1
#define KVFX_F32 2

/* Most layers one kvfx_write_layers / kvfx_gather_layers call takes. */
#define KVFX_MAX_LAYERS 128u

/* Most sequences one kvfx_attention_batch call takes. */
#define KVFX_MAX_PREFILL_SEQS 32u

/* Most groups one kvfx_decode_shared call takes. */
#define KVFX_MAX_PREFIX_GROUPS 32u

/* Slot of a padding token (kvfx_write_rotated): nothing is written for it. */
#define KVFX_NO_SLOT UINT64_MAX

/* Bits of the per-device status word. */
#define KVFX_FLAG_BAD_INDEX 1u  /* a slot/block id beyond the cache was skipped */
#define KVFX_FLAG_TIMEOUT 2u    /* a bounded wait inside a kernel expired        */

typedef struct kvfx_cache {
    void* k_base;            /* device address of K[0][0][0][0]                  */
    void* v_base;            /* device address of V[0][0][0][0]                  */
    uint64_t num_blocks;     /* physical pages                                   */
    uint32_t num_kv_heads;
    uint32_t block_size;     /* tokens per page                                  */
    uint32_t head_size;
    uint32_t dtype;          /* KVFX_F16 / KVFX_BF16 / KVFX_F32                  */
    int32_t device;          /* CUDA ordinal holding the cache                   */
    uint32_t reserved;       /* must be 0                                        */
} kvfx_cache;

/*
 * Paged KV write: for token i, K[slot_i / bs][h][slot_i % bs][:] = k_new[i][h][:]
 * and the same for V, for all h. k_new/v_new: [num_tokens][num_kv_heads][head_size]
 * in the cache dtype; slots: device uint64[num_tokens], pairwise distinct.
 * Replaces the kernel launch of write_paged_kv (KVFlux src/v2/paged_kv_write.cu:86-97).
 */
int kvfx_write(const kvfx_cache* cache, const void* k_new, const void* v_new,
               const uint64_t* slots, uint64_t num_tokens, void* stream);

/*
 * Gather of one sequence: k_out[t][h][:] = K[blocks[t / bs]][h][t % bs][:] for
 * t < num_tokens (V alike). blocks: device uint64[ceil(num_tokens / bs)].
 * Outputs must not overlap each other or the cache. Rows that are 16-byte
 * multiples of at most 256 elements, with 16-byte aligned bases, move by TMA
 * tensor copies (one load and one store per page and KV head); other shapes
 * by vector loads and stores.
 * Replaces the kernel launch of read_paged_kv (KVFlux src/v2/paged_kv_read.cu:90-102).
 */
int kvfx_gather(const kvfx_cache* cache, const uint64_t* blocks, uint64_t num_tokens,
                void* k_out, void* v_out, void* stream);

/*
 * Batched gather: sequence b has seq_lens[b] tokens, pages in row b of the
 * row-major table blocks[batch][max_blocks_per_seq], and outputs k_out[b] /
 * v_out[b] (device arrays of device pointers). One launch for the whole batch.
 * No counterpart in the reference, which gathers one sequence per call.
 */
int kvfx_gather_batch(const kvfx_cache* cache, const uint64_t* blocks,
                      const uint64_t* seq_lens, uint64_t batch, uint64_t max_blocks_per_seq,
                      void* const* k_out, void* const* v_out, void* stream);

/*
 * Layer batches. A model keeps one cache per layer, all with one shape and
 * one page pool (the reference's multi-layer plan: one PagedKVStorage per
 * layer over one PhysicalBlockPool, docs/v2_paged_kv_storage.md:19), so a
 * slot or a page id means the same place in every layer. These two calls
 * move one step's rows (or a batch of sequences) for every layer in one
 * launch, e.g. the whole KV of a request arriving from a prefill instance or
 * leaving for host memory. caches: host array of num_layers (<=
 * KVFX_MAX_LAYERS) descriptors equal in all fields but k_base and v_base.
 * No counterpart in the reference, which writes and reads one layer per call.
 */

/* kvfx_write on every layer: layer l's rows are k_new/v_new + l * layer_stride_bytes
 * ([num_tokens][num_kv_heads][head_size] each; layer_stride_bytes >= that size). */
int kvfx_write_layers(const kvfx_cache* caches, uint32_t num_layers, const void* k_new,
                      const void* v_new, uint64_t layer_stride_bytes, const uint64_t* slots,
                      uint64_t num_tokens, void* stream);

/* kvfx_gather_batch on every layer: sequence b's layer l goes to
 * k_out[b] + l * out_layer_stride_bytes (and v_out alike). */
int kvfx_gather_layers(const kvfx_cache* caches, uint32_t num_layers, const uint64_t* blocks,
                       const uint64_t* seq_lens, uint64_t batch, uint64_t max_blocks_per_seq,
                       void* const* k_out, void* const* v_out, uint64_t out_layer_stride_bytes,
                       void* stream);

/*
 * Whole-page copy of K and V from src_block to dst_block (byte-exact).
 * Replaces the two cudaMemcpyAsync of PagedKVStorage::copy_block
 * (KVFlux src/v2/paged_kv_storage.cpp:70-93).
 */
int kvfx_copy_page(const kvfx_cache* cache, uint64_t src_block, uint64_t dst_block,
                   void* stream);

/*
 * Copies inside the caches of a layer batch (caches, num_layers as for
 * kvfx_write_layers), one launch for all layers, byte-exact.
 *   kvfx_copy_pages: page dst_pages[i] = page src_pages[i], i < num_pages, in K
 *     and V of every layer (the private last pages of a batch of forks).
 *   kvfx_copy_slots: the rows of slot dst_slots[i] = those of slot
 *     src_slots[i], every head, K and V of every layer (the kept tokens of an
 *     eviction, moved together into fresh pages).
 * The id arrays are device uint64. A source may appear several times; each
 * destination may appear once, and no destination may be a source of the same
 * call (what a violation leaves in those pages or slots is undefined). An id
 * outside the cache is skipped and sets KVFX_FLAG_BAD_INDEX.
 * No counterpart in the reference, which copies one page of one layer per
 * call (src/v2/paged_kv_storage.cpp:70-93) and never moves tokens.
 */
int kvfx_copy_pages(const kvfx_cache* caches, uint32_t num_layers, const uint64_t* src_pages,
                    const uint64_t* dst_pages, uint64_t num_pages, void* stream);
int kvfx_copy_slots(const kvfx_cache* caches, uint32_t num_layers, const uint64_t* src_slots,
                    const uint64_t* dst_slots, uint64_t num_slots, void* stream);

/*
 * Rotary positions and the per-head norms of Q and K, as kvfx_write_rotated
 * applies them. A head's first rotary_dim dimensions are turned in pairs by
 * the angles of the token's position: pair i is dimensions (i, i +
 * rotary_dim / 2), or (2i, 2i + 1) when interleaved is 1. Row p of cos_sin
 * holds position p's rotary_dim / 2 cosines, then its sines.
 */
typedef struct kvfx_rotary {
    const float* cos_sin;    /* device [max_positions][rotary_dim]                 */
    uint64_t max_positions;
    uint32_t rotary_dim;     /* even, 2 .. head_size                                */
    uint32_t interleaved;    /* 0 or 1                                              */
    const float* q_weight;   /* device [head_size], or NULL: Q heads are not normed */
    const float* k_weight;   /* device [head_size], or NULL: K heads are not normed */
    float eps;               /* added to the mean square, >= 0                      */
    uint32_t reserved;       /* must be 0                                           */
} kvfx_rotary;

/*
 * Fills a cos_sin table: angle i of position p is
 * p * position_scale * base^(-2i / rotary_dim), computed in FP64.
 * base > 0, position_scale finite.
 */
int kvfx_rotary_table(float* cos_sin, uint64_t max_positions, uint32_t rotary_dim, double base,
                      double position_scale, int device, void* stream);

/*
 * New tokens' Q, K and V in one pass: K and Q heads are normed (y = x /
 * sqrt(mean(x^2) + eps) * weight, where weights are given) and rotated, K and
 * V go to their cache slots as in kvfx_write, and Q goes out in FP32 as the
 * attention entry points take it. Computed in FP32; K is rounded once.
 *   q, k, v   : device, the cache's dtype; token t's heads are contiguous
 *               rows of head_size from q + t * q_stride on (strides in
 *               elements, at least heads * head_size, so the three may be
 *               slices of one projection's output); must not overlap the
 *               cache or q_out
 *   positions : device uint64[num_tokens], each < max_positions
 *   slots     : device uint64[num_tokens], pairwise distinct; KVFX_NO_SLOT
 *               marks a padding token: nothing is written for it, and
 *               its position, q, k and v may hold anything
 *   q_out     : device float[num_tokens][q_heads][head_size]
 * q_heads may be 0 (q and q_out are then not looked at). A token whose slot
 * or position is out of range is skipped and sets KVFX_FLAG_BAD_INDEX.
 * Rows of 32, 64, 128 or 256 elements with 16-byte aligned bases and strides
 * (q_out: 32-byte), and a rotary_dim that is a multiple of 16 (8 interleaved),
 * take a kernel of 16-byte vectors; other shapes an element-wise one.
 * No counterpart in the reference, whose write takes K and V as they are
 * (src/v2/paged_kv_write.cu:101-139).
 */
int kvfx_write_rotated(const kvfx_cache* cache, const kvfx_rotary* rotary, const void* q, const void* k,
                       const void* v, uint64_t q_stride, uint64_t k_stride, uint64_t v_stride,
                       uint32_t q_heads, const uint64_t* positions, const uint64_t* slots,
                       uint64_t num_tokens, float* q_out, void* stream);

/*
 * Batch decode PagedAttention: one last-position query per sequence.
 *   q, o         : device float[batch][q_heads][head_size]
 *   block_table  : device uint64[batch][max_blocks_per_seq], row b holds the
 *                  pages of sequence b (entries past its length are not read)
 *   seq_lens     : device uint64[batch], each in [1, max_seq_len]
 *   max_seq_len  : host-side upper bound of seq_lens (sizes the grid)
 *   pages_per_split: split-K chunk in pages; 0 chooses one from the shape
 *   workspace    : device scratch of kvfx_decode_workspace_bytes(...) bytes,
 *                  zero-filled (cudaMemset) before its first use. Its start
 *                  holds the split counters, which every launch leaves at
 *                  zero again, so it stays ready for the next launch of any
 *                  batch, lengths or split size on caches with the same
 *                  num_kv_heads (zero it again before using it with a cache
 *                  of another head count). Launches that share a workspace
 *                  must not overlap on the GPU.
 * q_heads must be a multiple of num_kv_heads; Q head j uses KV head
 * j / (q_heads / num_kv_heads). Scale 1/sqrt(head_size).
 * Replaces paged_attention_batch's launch (KVFlux src/v2/paged_attention.cu:248-313).
 */
uint64_t kvfx_decode_workspace_bytes(const kvfx_cache* cache, uint64_t batch,
                                     uint32_t q_heads, uint64_t max_seq_len,
                                     uint32_t pages_per_split);
uint32_t kvfx_decode_pages_per_split(const kvfx_cache* cache, uint64_t batch,
                                     uint32_t q_heads, uint64_t max_seq_len,
                                     uint64_t total_tokens);
int kvfx_decode(const kvfx_cache* cache, const float* q, float* o,
                const uint64_t* block_table, const uint64_t* seq_lens, uint64_t batch,
                uint64_t max_blocks_per_seq, uint32_t q_heads, uint64_t max_seq_len,
                uint32_t pages_per_split, void* workspace, uint64_t workspace_bytes,
                void* stream);

/*
 * Batch decode over groups of rows that share a prefix: the attention of
 * kvfx_decode, with each group's shared pages read once for all of its rows
 * instead of once per row. Group g is the next groups[g].rows rows of the
 * batch, whose first groups[g].prefix_tokens positions (whole pages) are the
 * same pages: those of the group's first row, whose table entries are read
 * for them (also where that row is padding); every row's table still holds all
 * of its pages. The batch is the
 * groups' rows in order (at most 65535), num_groups at most
 * KVFX_MAX_PREFIX_GROUPS, prefix_tokens a multiple of block_size, at most
 * max_seq_len, and 0 where rows share nothing. groups is a host array, read
 * before the call returns.
 *   seq_lens  : device uint64[batch], each 0 or in [prefix_tokens of its
 *               group, max_seq_len]; a row of length 0 is padding: its output
 *               stays as it was. A row outside its bounds is refused the same
 *               way and sets KVFX_FLAG_BAD_INDEX.
 *   workspace : device scratch of kvfx_decode_shared_workspace_bytes(...)
 *               bytes, 16-byte aligned; nothing is kept in it from call to
 *               call. Calls that share one must not overlap on the GPU.
 * The other arguments as for kvfx_decode. 16-bit caches with head_size 64 or
 * 128 and block_size 16, with 16-byte aligned bases, q and o, read the prefix on
 * the tensor cores (at the FP32-class accuracy of the other attention entry
 * points), unless the rows are so short that reading them one by one is
 * faster; other shapes run row by row, each reading all of its pages.
 * Where a wait inside a kernel runs out (KVFX_FLAG_TIMEOUT), the rows that
 * depend on it become NaN or stay as they were.
 * No counterpart in the reference, whose batch attention re-reads shared pages
 * for every row (src/v2/paged_attention.cu:248-313).
 */
typedef struct kvfx_prefix_group {
    uint64_t rows;           /* >= 1 */
    uint64_t prefix_tokens;
} kvfx_prefix_group;
uint64_t kvfx_decode_shared_workspace_bytes(const kvfx_cache* cache, const kvfx_prefix_group* groups,
                                            uint32_t num_groups, uint32_t q_heads, uint64_t max_seq_len);
int kvfx_decode_shared(const kvfx_cache* cache, const float* q, float* o, const uint64_t* block_table,
                       const uint64_t* seq_lens, const kvfx_prefix_group* groups, uint32_t num_groups,
                       uint64_t max_blocks_per_seq, uint32_t q_heads, uint64_t max_seq_len,
                       void* workspace, uint64_t workspace_bytes, void* stream);

/*
 * One batch decode step fused with its paged KV write. Row b's new token is
 * position seq_lens[b] - 1 (seq_lens already count it); its K/V rows are
 * k_new/v_new[b][num_kv_heads][head_size] in the cache dtype and its slot is
 * new_slots[b] (device uint64[batch]), whose offset in its page must equal
 * (seq_lens[b] - 1) % block_size. The launch writes those rows into the cache,
 * stores the slot's page into block_table[b][(seq_lens[b] - 1) / block_size]
 * (block_table is device memory that stays resident between steps; entries
 * before that column are read as they are), and computes the same attention
 * as kvfx_decode over the updated rows; q, o, workspace and the other
 * arguments as for kvfx_decode. A slot outside the cache or at the wrong
 * offset is not written and sets KVFX_FLAG_BAD_INDEX. Each new slot must lie
 * in a page that no other row of the launch reads (copy a shared last page on
 * write first, as append_token_cow does); rows' slots must be distinct.
 * Replaces, for a batch, the write_paged_kv + paged_attention pair of the
 * reference's decode step (KVFlux src/v2/sequence_lifecycle.cpp:53-73), with
 * the block table kept on the device instead of uploaded per call
 * (src/v2/paged_attention.cu:287-292).
 */
int kvfx_decode_append(const kvfx_cache* cache, const void* k_new, const void* v_new,
                       const uint64_t* new_slots, const float* q, float* o, uint64_t* block_table,
                       const uint64_t* seq_lens, uint64_t batch, uint64_t max_blocks_per_seq,
                       uint32_t q_heads, uint64_t max_seq_len, uint32_t pages_per_split,
                       void* workspace, uint64_t workspace_bytes, void* stream);

/*
 * Batch decode that allocates nothing: the same computation and arguments as
 * kvfx_decode without pages_per_split and the workspace. No counterpart in
 * the reference. For callers that cannot call cudaMalloc: engines that hand
 * all device memory to their KV pool at start-up, loops that cannot take
 * cudaMalloc/cudaFree's implicit synchronisation, and embedders whose
 * allocator policy forbids device allocations outside their own allocator.
 * Its scratch (split-K partials + counters) is a static 16 MiB device array
 * held by every GPU that loads this code until the process exits; the split
 * size is chosen so the scratch fits, and a batch whose batch x num_kv_heads
 * cannot fit even with one split per sequence is rejected with KVFX_ENOSPACE.
 * The first call on a device looks up the array's address (make it before
 * any stream capture; a device reset invalidates it, so do not call this on
 * a device after resetting it). All calls share the array: calls that
 * overlap on the GPU race. The split counters return to zero at the end of
 * every launch; the first call on a device, and a call whose cache has
 * another num_kv_heads than the previous call's, clears them on `stream`
 * first. Device-side flags (an out-of-range page id, a bounded wait that
 * gave up) are kept in a device variable that kvfx_device_status reads
 * together with the other kernels' flags.
 */
int kvfx_decode_noalloc(const kvfx_cache* cache, const float* q, float* o,
                        const uint64_t* block_table, const uint64_t* seq_lens, uint64_t batch,
                        uint64_t max_blocks_per_seq, uint32_t q_heads, uint64_t max_seq_len,
                        void* stream);

/*
 * Single-sequence causal PagedAttention with query_tokens queries aligned to
 * the end of the kv_tokens-long sequence (query i sees positions
 * <= kv_tokens - query_tokens + i). q, o: device float[query_tokens][q_heads][head_size];
 * blocks: device uint64[ceil(kv_tokens / bs)]. workspace: as for kvfx_decode
 * (zero-filled before its first use; query_tokens == 1 runs the decode
 * kernel, the only case that needs one).
 * Replaces paged_attention's launch (KVFlux src/v2/paged_attention.cu:193-246).
 */
uint64_t kvfx_attention_workspace_bytes(const kvfx_cache* cache, uint64_t query_tokens,
                                        uint64_t kv_tokens, uint32_t q_heads);
int kvfx_attention(const kvfx_cache* cache, const float* q, float* o, const uint64_t* blocks,
                   uint64_t query_tokens, uint64_t kv_tokens, uint32_t q_heads,
                   void* workspace, uint64_t workspace_bytes, void* stream);

/*
 * kvfx_attention over num_seqs (<= KVFX_MAX_PREFILL_SEQS) sequences of one
 * cache in one call: sequence i has query_tokens[i] queries aligned to the
 * end of its kv_tokens[i] tokens, Q and O at the device addresses q[i] and
 * o[i] (float[query_tokens[i]][q_heads][head_size]) and its pages in row i of
 * the device table block_table[num_seqs][max_blocks_per_seq]. q, o,
 * query_tokens and kv_tokens are host arrays of num_seqs entries. Each
 * output equals what kvfx_attention gives for that sequence alone (bit for
 * bit); the sequences of tensor-core prefill shapes run as one persistent
 * launch that deals the query tiles of all of them, heaviest first, over the
 * SMs, the others as one kvfx_attention each after it. The workspace is the largest
 * kvfx_attention_workspace_bytes of the sequences. Sequences with no queries
 * are skipped. Replaces the per-sequence loop over paged_attention's launch
 * (KVFlux src/v2/paged_attention.cu:193-246) that a batched prefill makes.
 */
int kvfx_attention_batch(const kvfx_cache* cache, uint32_t num_seqs, const float* const* q, float* const* o,
                         const uint64_t* block_table, uint64_t max_blocks_per_seq,
                         const uint64_t* query_tokens, const uint64_t* kv_tokens, uint32_t q_heads,
                         void* workspace, uint64_t workspace_bytes, void* stream);

/* Message of the calling thread's last failed call ("" if none). */
const char* kvfx_last_error(void);

/*
 * Reads the status word of `device` (KVFX_FLAG_* bits set by kernels since
 * the last clear, kvfx_decode_noalloc's included) after the caller has
 * synchronised the work in question; clears it when `clear` is non-zero.
 */
int kvfx_device_status(int device, uint32_t* flags, int clear);

/*
 * Self-test of device-side failure detection. Every kernel here that waits on
 * a shared-memory barrier (TMA arrivals, tensor-core commits) bounds the wait
 * (2 s): a wait that runs out raises KVFX_FLAG_TIMEOUT in the status word and
 * the kernel returns instead of hanging; the C++ API then throws
 * std::runtime_error. This call runs those waits (inline and out-of-line
 * forms) on `device` on a barrier that nothing completes and nothing is in
 * flight on, synchronously (~2 s). Returns KVFX_ETIMEOUT when both waits gave
 * up and reported it (the expected outcome; the context stays usable),
 * KVFX_EINVAL if a wait did not report it, KVFX_ECUDA on a CUDA error. The
 * status word is left as it was (run no other work on the device meanwhile,
 * or its timeout flag may be folded into the test's). No counterpart in the reference, whose
 * kernels do not wait on barriers.
 */
int kvfx_selftest_wait_timeout(int device);

/*
 * kvfx_decode_shared as it ends when every wait of its prefix kernel has run
 * out, without the waits: that kernel's pieces are given up by the code that
 * the waits' end reaches, and the rest of the call joins them. Rows behind a
 * prefix become NaN, whatever the workspace held; rows without one, and calls
 * that launch no prefix kernel, are computed as ever. No flag is raised.
 */
int kvfx_selftest_lost_prefix(const kvfx_cache* cache, const float* q, float* o, const uint64_t* block_table,
                              const uint64_t* seq_lens, const kvfx_prefix_group* groups, uint32_t num_groups,
                              uint64_t max_blocks_per_seq, uint32_t q_heads, uint64_t max_seq_len,
                              void* workspace, uint64_t workspace_bytes, void* stream);

/* Library version, e.g. "kvflux-b200 0.1.0 sm_100a". */
const char* kvfx_version(void);

#ifdef __cplusplus
}
#endif

#endif /* KVFX_H */
