/* libgtok C ABI: text -> token ids for byte-level BPE tokenizers on one B200.
 *
 * The first thirteen entry points are the reference's own C ABI
 * (src/gtok_shim.cc:133-399, exported through src/gtok.map:4-7) with the same
 * names, argument meaning and return codes, so that its ctypes / dlopen callers
 * (python/gpu_bpe_tokenizer/vllm.py:87-121, integrations/dynamo) bind unchanged.
 * The gtok_x_* entry points are additions for measurement and diagnostics.
 *
 * Ownership: the caller owns every input and output buffer; a handle owns its
 * device and pinned memory.  No exception crosses this boundary: failures are
 * negative return codes (or NULL).  A tokenizer handle is not thread-safe; a
 * dispatcher handle is.
 *
 * This library has no CPU route: gtok_cpu_backend() is always "off" (a state the
 * reference also has, src/cpu_route.cc:68-74) and every encode runs on the GPU;
 * creation fails when no sm_100 device is present.
 */
#ifndef GTOK_H
#define GTOK_H
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

/* src/gtok_shim.cc:138-155.  Loads an HF tokenizer.json; max_bytes is the largest
 * input a call may carry (raised to 4096).  GPU contexts are built on first use.
 * NULL on failure (see gtok_x_last_error). */
void* gtok_create(const char* vocab_json_path, uint32_t max_bytes);

/* src/gtok_shim.cc:160-202.  Returns the token count, -1 on error, -2 if `out` is too
 * small, -3 if the (normalised) input exceeds the handle's byte cap. */
int32_t gtok_encode(void* handle, const uint8_t* text, uint32_t len, uint32_t* out, uint32_t max_out);

/* src/gtok_shim.cc:209-236.  As gtok_encode, ids copied device-to-device into out_dev, which they are in
 * when the call returns.  No queued work may still use out_dev (or see gtok_x_result_stream). */
int32_t gtok_encode_to_device(void* handle, const uint8_t* text, uint32_t len, void* out_dev, uint32_t max_out);

/* src/gtok_shim.cc:246-318.  n_docs documents concatenated in concat_bytes with
 * n_docs+1 byte offsets; one graph replay; result equals per-document gtok_encode
 * concatenated.  out_doc_offsets gets n_docs+1 running token counts.  Returns the
 * total, -1 error, -2 out_tokens too small, -3 bytes exceed the cap, -4 document
 * capacity could not grow. */
int32_t gtok_encode_batch(void* handle, const uint8_t* concat_bytes, const uint32_t* doc_byte_offsets, uint32_t n_docs,
                          uint32_t* out_tokens, uint32_t out_cap, uint32_t* out_doc_offsets);

/* src/gtok_shim.cc:325-335.  CPU-route controls; the route does not exist here:
 * the limit reads 0, setting it is accepted and ignored, the backend is "off". */
uint32_t gtok_cpu_max_bytes(void* handle);
void gtok_set_cpu_max_bytes(void* handle, uint32_t max_bytes);
const char* gtok_cpu_backend(void* handle);

/* src/gtok_shim.cc:346-390.  One dispatcher is shared by all request threads;
 * gtok_dispatch_encode is thread-safe and blocking.  policy: 0 adaptive, 1 GPU,
 * 2 CPU (accepted; every request still runs on the GPU).  Stats: [cpu_requests,
 * gpu_requests, gpu_batches, gpu_large, gpu_batch_ns]. */
void* gtok_dispatcher_create(const char* vocab_json_path, uint32_t cpu_workers, uint32_t max_batch_bytes,
                             uint32_t max_batch_docs, uint32_t policy);
int32_t gtok_dispatch_encode(void* dispatcher, const uint8_t* text, uint32_t len, uint32_t* out, uint32_t max_out);
void gtok_dispatcher_stats(void* dispatcher, uint64_t* out5);
void gtok_dispatcher_destroy(void* dispatcher);

/* src/gtok_shim.cc:392-399. */
uint32_t gtok_vocab_size(void* handle);
void gtok_destroy(void* handle);

/* ---- additions (no counterpart in the reference's C ABI) -------------------- */

/* Last failure message of this thread's most recent failing call ("" if none). */
const char* gtok_x_last_error(void);
/* 0 GPT-2, 1 Llama-3, 2 Qwen2.5; bit 8 set when the vocabulary asks for NFC. */
uint32_t gtok_x_family(void* handle);
/* Measurement, after the reference's stage_input / launch_graph_sync / read_staged_batch
 * (src/tokenizer.cuh:252-279): copy the input to the device once, then time graph
 * replays on their own.  doc_byte_offsets may be NULL for a single document.
 * gtok_x_replay returns the token count and writes the CUDA-event time of the replay. */
int32_t gtok_x_stage(void* handle, const uint8_t* bytes, uint32_t len, const uint32_t* doc_byte_offsets, uint32_t n_docs);
int32_t gtok_x_replay(void* handle, float* ms_out);
int32_t gtok_x_read(void* handle, uint32_t* out_tokens, uint32_t out_cap, uint32_t* out_doc_offsets);
/* Boundary bits of the staged input after a replay: bit i of the stream is set where a
 * pre-token starts at byte i.  Writes (len + 31) / 32 words; returns that count. */
int32_t gtok_x_read_boundaries(void* handle, uint32_t* out_words, uint32_t max_words);
/* The staged input once more, launched kernel by kernel with CUDA events between:
 * ms_out6 = {pre-tokenization, words, miss, assemble kernel, whole sequence, what runs before
 * pre-tokenization (normalisation and document-bit kernels)}. */
int32_t gtok_x_profile(void* handle, float* ms_out6);
/* Diagnostics: when the environment variable GTOK_PHASE_CLOCKS was set as the staged
 * context was created, SM cycles spent in each phase of the two kernels, summed over
 * thread blocks since the last reset (slots 0-6 pre-tokenization, 8-11 words, 12-15 assemble,
 * 16-20 miss, 24-26 normalisation).  -1 if off. */
int32_t gtok_x_phase_clocks(void* handle, uint64_t* out32, int32_t reset);
/* Diagnostics, same switch: when each thread block of the last replay's four kernels started,
 * finished, and finished its first six work items, as stamps of the GPU's nanosecond timer:
 * out[(kernel * 1280 + block) * 8 + slot], slot 0 = start, 1 = end, 2.. = work items; kernel 0
 * pre-tokenization, 1 words, 2 miss, 3 assemble.  Returns the words written (at most 40960),
 * -1 if off.  The record is cleared by the call. */
int32_t gtok_x_timeline(void* handle, uint64_t* out, uint32_t max_words);
/* gtok_encode_batch with the ids and the n_docs + 1 token offsets left in device memory (device-to-
 * device copies), as gtok_encode_to_device does for one document: what the reference's Python
 * Tokenizer.encode_batch_to_device returns (src/python_bindings.cc:410-507); its C ABI has no such entry. */
int32_t gtok_x_encode_batch_to_device(void* handle, const uint8_t* concat_bytes, const uint32_t* doc_byte_offsets, uint32_t n_docs,
                                      void* out_tokens_dev, uint32_t out_cap, void* out_doc_offsets_dev);
/* What the next encoding call on this handle writes to device memory (gtok_encode_to_device,
 * gtok_x_encode_batch_to_device, gtok_x_encode_measured) is written behind the work that is queued on
 * `cuda_stream` (a cudaStream_t of the current device, NULL = its default stream; it must live until that
 * call returns): a handle works on a stream of its own, so a buffer that queued work still reads or writes,
 * such as one that an allocator working in stream order has just handed out again, has to be announced so.
 * The encoding does not wait, only the copies do.  Ignored while the stream is being captured.  0 or -1. */
int32_t gtok_x_result_stream(void* handle, void* cuda_stream);
/* Raises the handle's byte cap (the limit behind return code -3) without re-creating the handle:
 * vocabulary and tables stay, the GPU context grows at the next call that needs it.  The reference
 * has callers re-create a bigger handle (src/gtok_shim.cc:160-202), which reloads the vocabulary.
 * Returns the cap now in force (never lowered). */
uint32_t gtok_x_set_max_bytes(void* handle, uint32_t max_bytes);
/* What the last replay of the staged input handed from kernel to kernel, for byte accounting:
 * out6 = {pre-tokens, pre-tokens of 2..64 bytes the whole-word table did not know, their bytes,
 * pre-tokens longer than 64 bytes, their bytes, ids written by the miss kernel}.  Counted on the
 * host from the lists and boundary bits in device memory (a debugging-speed call).  0 or -1. */
int32_t gtok_x_work_stats(void* handle, uint64_t* out6);
/* Sizes in bytes of the merge table, the whole-word table and the remaining tables. */
void gtok_x_table_bytes(void* handle, uint64_t* out3);
/* Kernel launches one graph replay performs (single document / batch). */
int32_t gtok_x_launches_per_replay(void* handle, int32_t batch);

/* Pre-token boundaries for callers that must not allocate.  No counterpart in the
 * reference.  Some hosts of this library cannot call cudaMalloc when they need an
 * answer: a serving process whose framework has claimed the whole device for its own
 * memory pool, or a plug-in that was handed a fixed set of buffers and nothing else.  For
 * them this entry point runs the pre-tokenization kernel with all of its working memory
 * taken from an array that is part of the library's device image (about 0.5 MB, held on
 * every GPU that loads the library until the process exits), and calls no cudaMalloc,
 * cudaFree or any other allocating routine.  That fixed array is also the limit: inputs
 * above 4 MiB (4,194,304 bytes) are refused with -3 and a message in gtok_x_last_error.
 *   text_dev      device pointer, 16-byte aligned, one document of `len` bytes; the
 *                 buffer must be readable up to `len` rounded up to 16
 *   out_bits_dev  device pointer to ((len + 4095) / 4096) * 128 uint32; bit i of the
 *                 stream is set where a pre-token starts at byte i (same bits as
 *                 gtok_x_read_boundaries)
 *   cuda_stream   a cudaStream_t (NULL = default stream); the work is queued on it and
 *                 the call waits for it (cudaStreamSynchronize) before it returns
 * The handle (created earlier, when allocation was still possible) supplies the
 * vocabulary tables; its device is made current for the call and the caller's current
 * device is put back before returning.  The first call on a device looks up the array's
 * device address: make that first call before any stream capture begins.  All calls share
 * the one array, which keeps the previous call's contents (the parts that must start at
 * zero are cleared on the stream each time): two calls that overlap on the GPU race, so
 * serialise them.  Returns 0; -1 on error, which includes error bits raised by the kernel
 * itself (a wait on an earlier tile that gave up, as overlapping calls can cause); -3 when
 * `len` exceeds the limit. */
int32_t gtok_x_boundaries_noalloc(void* handle, const void* text_dev, uint32_t len, void* out_bits_dev, void* cuda_stream);

/* Raw bytes of token `id` (the spelling the ids decode to); returns the length, -1 for an
 * id outside the vocabulary.  Nothing is written when `cap` is too small. */
int32_t gtok_x_token_bytes(void* handle, uint32_t id, uint8_t* out, uint32_t cap);

/* Decoding on the device: `n` token ids -> the bytes they spell, one pass (lengths, scan,
 * gather) in a captured graph of its own.  Replaces the reference's TokenizerCtx::decode
 * (src/tokenizer.cu:5499-5573, kernels :5225-5275) behind Tokenizer.decode / decode_bytes
 * (src/python_bindings.cc:558-600); the reference's C ABI has no decode entry.  Host buffers.
 * Returns the byte count; -1 on error (an id outside the vocabulary included); -2 when
 * `max_out` is too small (out = NULL with max_out = 0 asks for the size).  `need_out` (may be NULL)
 * receives the byte count in both cases,
 * `kernel_ms` (may be NULL) the CUDA-event time of the graph. */
int64_t gtok_x_decode(void* handle, const uint32_t* ids, uint32_t n, uint8_t* out, uint64_t max_out, uint64_t* need_out, float* kernel_ms);

/* The encode and decode calls in steps, for bindings that hold text in pieces (a list of strings) and make
 * the result's memory themselves once its size is known.  A handle takes one call at a time: measure, encode
 * and take belong together; any other call that encodes, stages or replays on the handle ends them, and the
 * step that would have come next answers -1.
 *   gtok_x_measure         UTF-8 bytes of the pieces, which are the documents of a batch or the parts of one
 *                          text; -1 where a character has no UTF-8 form (a surrogate)
 *   gtok_x_encode_measured encodes them (they must still be in place) and returns the id count; return codes as
 *                          gtok_encode / gtok_encode_batch.  `bytes` is what gtok_x_measure returned (-1 for anything
 *                          else); after -2 the same text may follow with more room, else once.  With out_dev the ids (and with out_doc_dev the
 *                          n_pieces + 1 token offsets of a batch) go to device memory, else gtok_x_take_ids
 *                          copies them to host memory (directly where that is page-locked)
 *   gtok_x_decode_room     a page-locked buffer for n ids; ids put there need no further copy.  Optional; the
 *                          buffer is the handle's, until its next decoding call
 *   gtok_x_decode_run      ids -> bytes, which gtok_x_take_bytes copies to host memory; returns their number
 */
typedef struct {
    const void* data;
    uint64_t units;      /* bytes (kind 1) or characters */
    uint32_t kind;       /* 1 bytes as they are (UTF-8 or whatever the text is); characters of 2 or 4 bytes: 2, 4; of one byte (Latin-1): 3 */
} gtok_x_piece;
int64_t gtok_x_measure(void* handle, const gtok_x_piece* pieces, uint32_t n_pieces, int32_t batch);
int64_t gtok_x_encode_measured(void* handle, int64_t bytes, void* out_dev, uint64_t out_cap, void* out_doc_dev);
int32_t gtok_x_take_ids(void* handle, uint32_t* out, uint32_t* out_doc_offsets);
uint32_t* gtok_x_decode_room(void* handle, uint32_t n);
int64_t gtok_x_decode_run(void* handle, const uint32_t* ids, uint32_t n);
int32_t gtok_x_take_bytes(void* handle, uint8_t* out);

/* Partitioning over the GPUs of one box (no counterpart in the reference, which is
 * single-GPU).  gtok_x_plan_chunks cuts one document into n_parts pieces at
 * positions where a pre-token starts whatever precedes it (letter | space letter),
 * so that the pieces' ids concatenate to the ids of the whole; out_offsets gets
 * n_parts+1 byte offsets.  gtok_x_plan_documents cuts a batch into n_parts
 * contiguous document ranges of about equal bytes; out_doc_index gets n_parts+1
 * document indices.  Each part is then encoded by one GPU with gtok_encode /
 * gtok_encode_batch; only the parts' token counts cross GPUs. */
int32_t gtok_x_plan_chunks(void* handle, const uint8_t* text, uint64_t len, uint32_t n_parts, uint64_t* out_offsets);
int32_t gtok_x_plan_documents(const uint32_t* doc_byte_offsets, uint32_t n_docs, uint32_t n_parts, uint32_t* out_doc_index);

/* ---- between token ids and a model -----------------------------------------------
 * No counterpart in the reference.  What a model does with token ids at its two ends that are as wide as the
 * vocabulary: rows of the embedding table are looked up by id, and the hidden states of each position are
 * compared with the id that follows there.  These entries work on device memory only, need no handle and no
 * vocabulary file, allocate nothing, wait for nothing and read nothing back: the work is queued on `cuda_stream` (a
 * cudaStream_t of the current device, NULL = its default stream), may be captured into a graph, and calls on different
 * streams may overlap as long as each has a workspace of its own.  A workspace is device memory of at least the size
 * that the _workspace entry answers, aligned to 256 bytes; nothing in it outlives the call's work.
 * 0 or -1 (see gtok_x_last_error); sizes, types, strides and addresses are checked before anything is queued.
 * Results do not depend on how the GPU schedules the work.  Sums are in fp32, rounded once to the output's type
 * unless a comment says otherwise.  Outputs must not overlap inputs. */
typedef struct {
    void* data;              /* device memory */
    int64_t rows, cols;
    int64_t stride;          /* elements from a row to the next; elements of a row follow one another */
    int32_t type;            /* 0 fp32, 1 bf16, 2 fp16 */
} gtok_x_matrix;

/* out[t, :] = scale * table[ids[t], :] for n ids of `id_bits` (32 or 64) bits.  A negative id gives a row of zeros,
 * an id beyond the table a row of NaN. */
int32_t gtok_x_embed(const void* ids, int32_t id_bits, int64_t n, const gtok_x_matrix* table, float scale, const gtok_x_matrix* out, void* cuda_stream);
/* Its gradient: out[v, :] = scale * (sum of grad[t, :] over the t with ids[t] = v), summed in the order of the ids; rows that no
 * id asks for become 0.  With `accumulate` the sums are added to what `out` holds (rounded once more) and other rows stay.
 * Ids outside the table are left out. */
int64_t gtok_x_embed_grad_workspace(int64_t n, int64_t vocab, int64_t width);
int32_t gtok_x_embed_grad(const void* ids, int32_t id_bits, int64_t n, const gtok_x_matrix* grad, float scale, const gtok_x_matrix* out, int32_t accumulate,
                          void* workspace, uint64_t workspace_bytes, void* cuda_stream);
/* Targets of packed documents, as gtok_x_encode_batch_to_device leaves them: out[i] = ids[i + 1] where i and i + 1 lie in the
 * same document, else `ignore`; `ignore` also where loss_mask (may be NULL) is 0 and outside of all documents.
 * doc_offsets: n_docs + 1 ascending places. */
int32_t gtok_x_next_targets(const int32_t* ids, int64_t n, const int32_t* doc_offsets, int64_t n_docs, const uint8_t* loss_mask, int32_t ignore, int32_t* out,
                            void* cuda_stream);

/* Losses over the vocabulary from hidden states H [n, width] and an output table W [vocab, width] (both bf16 or both fp16),
 * with logits Z = H W^T that are never held as a whole.  Beside copies of the rows (and of a table whose rows are no whole 16 bytes) a forward pass
 * takes a workspace of 8 bytes for each of the n rows and 128 ids of the vocabulary (4.7 KB a row at least), a backward pass one of at most 512 MiB (or 512
 * bytes a row, where that is more) and the fp32 sums of d_hidden (for few rows in several parts, up to 155 MB).  Tensor-core sums are cut off rather than rounded; logits are scaled by 1 + 2^-26 for each 16 elements of the width, what that
 * takes from them on average, which is also how far they are off where nothing is cut off.
 *   entries == 0   cross entropy: losses[i] = lse(z_i / T) - z_i[targets[i]] / T.  A negative target and `ignore` are no loss
 *   entries > 0    distillation from a teacher's `entries` (at most 1024) top logits a row: ids in `targets` (rows
 *                  `target_stride` apart; a negative id is no entry), logits of any type in teacher_logits.  With q the softmax of a row's
 *                  logits / T, losses[i] = sum_k q_k (log q_k - z_i[id_k] / T + lse(z_i / T)); an id that comes twice counts twice.
 *                  A row without entries, or with logits of -infinity only, is no loss
 * Rows without a loss get 0 and leave no trace in any gradient, whatever H holds there; a target or entry beyond the vocabulary gives
 * NaN as that row's loss and no gradient.  No factor T^2 is applied.
 *   forward    writes losses[n], lse[n] (natural logarithm, of z / T) and, where `total` is given, the sum of the losses or,
 *              with `mean`, their mean over the rows that have a loss (0 where none has)
 *   backward   reads lse, and grad: the gradient of each loss (grad_stride elements apart, 0 for one that all share), or with
 *              `mean` that of the mean.  Writes d_hidden and d_weight (either may have data = NULL).  dZ is rounded to the tables' type on its way
 *              into the two products, in one scale for all rows: by the largest finite row gradient, so that fp16's range does, and in distillation
 *              by what the teacher's probabilities in the call's first 2,048 entries round best at.  In fp16, rows whose gradient is far below the largest
 *              keep fewer bits: dZ of less than 2^-29 of it lies among the numbers below the normal ones, of less than 2^-40 becomes 0.  A gradient that is
 *              not finite makes its row of d_hidden, and all of d_weight, not finite, and leaves other rows of d_hidden as they are
 * `kept` (may be NULL; gtok_x_vocab_loss_kept bytes, aligned to 256) is where a forward pass leaves its copy of the rows with a loss and their
 * targets; a backward pass that is given it does not look at `hidden`'s, `targets`' and `teacher_logits`' values again.  It must come from a
 * forward pass of the same sizes, `entries` and temperature, may be used any number of times, and is only read. */
typedef struct {
    gtok_x_matrix hidden, weight;
    const void* targets;
    int64_t target_stride;
    int32_t target_bits;     /* 32 or 64 */
    int32_t entries;
    gtok_x_matrix teacher_logits;
    int64_t ignore;
    float temperature;       /* T: at least 2^-126 */
    int32_t mean;
    float* losses;
    float* lse;
    float* total;
    const float* grad;
    int64_t grad_stride;
    gtok_x_matrix d_hidden, d_weight;
    void* kept;
    uint64_t kept_bytes;
    void* workspace;
    uint64_t workspace_bytes;
    void* cuda_stream;
} gtok_x_vocab_loss;
int64_t gtok_x_vocab_loss_workspace(const gtok_x_vocab_loss* args, int32_t backward);   /* of the addresses it goes by weight's alignment and by whether `kept` is given */
int64_t gtok_x_vocab_loss_kept(const gtok_x_vocab_loss* args);
int32_t gtok_x_vocab_loss_forward(const gtok_x_vocab_loss* args);
int32_t gtok_x_vocab_loss_backward(const gtok_x_vocab_loss* args);

/* ---- from hidden states to the next ids ---------------------------------------------
 * No counterpart in the reference.  The last steps of a model that answers: products of some hidden states with an output table that is
 * held in 4 bits, changes to the logits, and the draw of an id for each row.  As for the entries above: device memory only, no handle, nothing is allocated or
 * waited for, calls on different streams may overlap and may be captured.  They need no workspace.
 *
 * A table of `vocab` rows and `width` columns: codes q of 4 bits, and for every `group` columns of a row (32, or a multiple of 64; the last group may be shorter) a scale s
 * in 16 bits and, with `zeros`, a zero b of 4 bits (8 for all where there are none).  The value of an element is s * (q - b).  It lies in one piece of memory of
 * gtok_x_table4_bytes, aligned to 256 bytes, in an order of its own.
 *   pack       from codes (a byte each, of which the low four bits count; rows `codes_stride` apart), scales [vocab, groups of a row] of the table's type, and zeros likewise
 *   quantize   from weights of any type: without zeros s = max |w| / 7, q = round(w / s) + 8; with zeros s = (max(w, 0) - min(w, 0)) / 15, b = round(-min(w, 0) / s),
 *              q = round(w / s) + b; s is rounded to the table's type first, ties go to even, q is held to 0 to 15.  A group with a NaN or an
 *              infinity, or whose scale would be infinite in the table's type, has NaN for a scale
 *   logits     out[i, v] = sum over the groups of s * (sum over the group's columns of (q - b) * hidden[i, k]), for hidden states of the table's type; out is fp32 or of
 *              that type.  Products are exact and summed in fp32, in an order that depends on the sizes alone.  A row's hidden states touch no other row */
typedef struct {
    void* data;
    uint64_t bytes;
    int64_t vocab, width, group;
    int32_t type;            /* of scales and hidden states: 1 bf16, 2 fp16 */
    int32_t zeros;           /* 0 or 1 */
} gtok_x_table4;
int64_t gtok_x_table4_bytes(int64_t vocab, int64_t width, int64_t group, int32_t zeros);
int32_t gtok_x_table4_pack(const gtok_x_table4* table, const uint8_t* codes, int64_t codes_stride, const gtok_x_matrix* scales, const uint8_t* zeros, int64_t zeros_stride,
                           void* cuda_stream);
int32_t gtok_x_table4_quantize(const gtok_x_table4* table, const gtok_x_matrix* weight, void* cuda_stream);
int32_t gtok_x_table4_logits(const gtok_x_matrix* hidden, const gtok_x_table4* table, const gtok_x_matrix* out, void* cuda_stream);

/* Changes to logits [n, vocab], in fp32 and rounded once; `out` has their type and is their memory, with the same stride, or apart from it; it is apart from all else.  In this order:
 *   ids of the row's history: l > 0 becomes l / repetition, others l * repetition; then, for ids that come `count` > 0 times behind the row's first
 *     prompt_lengths (all of them without it), l - frequency * count - presence.  Row i's history is ids[offsets[i]] to ids[offsets[i + 1] - 1] (of `n_ids` in all; `offsets` NULL: none); ids
 *     outside the vocabulary are left out
 *   l + the sum, in the order of the list, of the row's biases for that id: `entries` (at most 1024) ids and values a row, `bias_stride` apart (0: one list for all).  A negative id is no entry
 *   -infinity, whatever stood there, where bit id % 32 of word id / 32 of the row's mask is 0.  Masks are `allowed_stride` words apart; row i has mask allowed_rows[i], or
 *     mask i without it.  A negative number is no mask, one of allowed_count or more allows nothing
 * repetition, presence and frequency: a value for each row or, where NULL, the one_ value for all. */
typedef struct {
    gtok_x_matrix logits, out;
    const void* ids;
    int64_t n_ids;
    int32_t id_bits;         /* 32 or 64 */
    int32_t entries;
    const int32_t* offsets;
    const int32_t* prompt_lengths;
    const float *repetition, *presence, *frequency;
    float one_repetition, one_presence, one_frequency;
    int32_t reserved;
    const int32_t* bias_ids;
    const float* bias;
    int64_t bias_stride;
    const int32_t* allowed;
    const int32_t* allowed_rows;
    int64_t allowed_count, allowed_stride;
    void* cuda_stream;
} gtok_x_adjustment;
int32_t gtok_x_adjust_logits(const gtok_x_adjustment* args);

/* An id for each row of logits [n, vocab] (vocab at most 2^24).  With m = exp((l - max) / temperature), ids go in order of falling logits, equal ones in order of rising ids.  The first top_k
 * are kept (all, where it is 0 or less); of these the fewest whose m make up at least top_p of theirs (all, where it is 1 or more; one, where it is 0 or less); of these the ones with m >= min_p;
 * the first in any case.  ids[i] is the first id, in the order of ids, at which the running sum of the kept m exceeds u[i] times their sum (u from 0, below 1); logprobs[i] is
 * the logarithm of its share of all m, kept or not, and never above 0.  Temperature 0 gives the first id and logprob 0.  Sums of masses are exact sums of whole
 * numbers, whatever the order and the number of rows; a mass is off by 2^-43 relative, and rounding it to a whole number takes 2^-25 of a row's total at most from all masses together (2^-29 for
 * 128,256 ids).
 * -infinity is never drawn; a row of nothing else gives id -1 and logprob -infinity.  A row with a NaN, or whose temperature is negative or not finite, whose u is outside its range
 * or whose top_p or min_p is NaN gives id -1 and logprob NaN.  Parameters: a value for each row or, where NULL, the one_ value for all. */
typedef struct {
    gtok_x_matrix logits;
    const void* u;           /* n numbers */
    int32_t u_bits;          /* fp32 or fp64: 32 or 64 */
    int32_t one_top_k;
    const float* temperature;
    const int32_t* top_k;
    const float *top_p, *min_p;
    float one_temperature, one_top_p, one_min_p;
    int32_t reserved;
    int32_t* ids;
    float* logprobs;
    void* cuda_stream;
} gtok_x_draw;
int32_t gtok_x_sample(const gtok_x_draw* args);

#ifdef __cplusplus
}
#endif
#endif
