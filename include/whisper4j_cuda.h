/*
 * whisper4j_cuda.h — C ABI of libwhisper4j_cuda.so, the B200 (sm_100a) Whisper
 * text-decoder token loop.
 *
 * The library replaces the reference's decoder hot path
 * (com.sparrowlogic.whisper4j.nn.WhisperDecoder and the nn/tensor code under it)
 * behind plain C types, so a Java host binds it with java.lang.foreign downcalls
 * and any C/C++/Python host with its own FFI.  All entry points return an int
 * status (W4J_OK = 0, negative on error); w4j_last_error() gives the message of
 * the calling thread's last failure.  A context is bound to one CUDA device;
 * calls on one context are serialised internally, separate contexts run
 * concurrently.
 *
 * Reference interfaces each entry point replaces are cited as file:line within
 * sparrowlogic/whisper4j (W4J = src/main/java/com/sparrowlogic/whisper4j).
 */
#ifndef WHISPER4J_CUDA_H
#define WHISPER4J_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define W4J_OK 0
#define W4J_ERR_ARG -1       /* IllegalArgumentException in the reference */
#define W4J_ERR_STATE -2     /* IllegalStateException (e.g. weights missing, closed) */
#define W4J_ERR_CUDA -3      /* CUDA runtime or kernel failure */
#define W4J_ERR_OOM -4       /* device allocation failed */
#define W4J_ERR_CANCELLED -5 /* w4j_cancel() observed between steps */

/* GGML tensor types (W4J/model/GgmlLoader.java:30-36). */
#define W4J_GGML_F32 0
#define W4J_GGML_F16 1
#define W4J_GGML_Q8_0 8
#define W4J_GGML_BF16 30 /* operands of the paged cache and of the 8-bit integer products only */

/* W4J/model/ModelDimensions.java:6-17, same field order. */
typedef struct w4j_dims {
    int32_t n_mels, n_audio_ctx, n_audio_state, n_audio_head, n_audio_layer;
    int32_t n_vocab, n_text_ctx, n_text_state, n_text_head, n_text_layer;
} w4j_dims;

typedef struct w4j_ctx w4j_ctx;

/* Last error message of the calling thread ("" if none). */
const char *w4j_last_error(void);

/* Library version string. */
const char *w4j_version(void);

/*
 * Create a decoder context on `device` (replaces `new WhisperDecoder(weights, dims)`,
 * W4J/nn/WhisperDecoder.java:36-56, called at W4J/WhisperModel.java:160).
 * max_streams: independent audio chunks decoded together by one call;
 * max_beam: largest beam size used (1 for greedy only).  Device memory for the
 * KV caches is sized from these and n_text_ctx / n_audio_ctx.
 */
int w4j_ctx_create(const w4j_dims *dims, int device, int max_streams, int max_beam, w4j_ctx **out);
int w4j_ctx_destroy(w4j_ctx *ctx);

/*
 * Upload one decoder tensor straight from the GGML file's bytes (the hook next
 * to GgmlLoader.dequantize, W4J/model/GgmlLoader.java:185-202).  `ne` is the
 * GGML shape (fastest dimension first), `data` the raw payload: F32, F16 or
 * Q8_0 (34-byte blocks).  Encoder tensors ("encoder.*") are kept on the same
 * device for w4j_encoder_forward (F16 / F32 matrices; a Q8_0 encoder matrix is
 * skipped with return 1).  Other names return 1.  Unknown decoder or encoder
 * tensor names, wrong shapes and unsupported types are errors.
 */
int w4j_upload_tensor(w4j_ctx *ctx, const char *name, int ggml_type, const int64_t *ne, int n_dims,
                      const void *data, size_t nbytes);

/* Check that every decoder tensor is present (WeightStore.get, W4J/model/WeightStore.java:28-34). */
int w4j_finalize(w4j_ctx *ctx);

/*
 * Set the encoder output xa (n_audio_ctx x n_audio_state f32, row-major, host
 * memory) of stream `slot` and project the cross-attention K/V of every layer
 * into the device cache (the first-call branch of MultiHeadAttention.forward,
 * W4J/nn/MultiHeadAttention.java:65-75).  The _device variant takes a device
 * pointer on the context's device.
 */
int w4j_set_encoder_output(w4j_ctx *ctx, int slot, const float *xa, int n_audio_ctx);
int w4j_set_encoder_output_device(w4j_ctx *ctx, int slot, const float *xa_device, int n_audio_ctx);

/*
 * Run the audio encoder on the device (replaces WhisperEncoder.forward, W4J/nn/WhisperEncoder.java:42-76,
 * with Conv1d.forward, W4J/nn/Conv1d.java:38-80): mel is the log-mel spectrogram, n_mels x n_frames f32
 * row-major host memory (the reference's (1, n_mels, n_ctx) tensor), n_frames = 2 * n_audio_ctx.  The
 * encoder weights ("encoder.*") come through w4j_upload_tensor like the decoder's, F16 or F32
 * matrices.  xa_out (host, n_audio_ctx x n_audio_state f32) receives the encoder output when not
 * NULL; slot >= 0 also sets that stream's encoder output on the device (as
 * w4j_set_encoder_output_device, no host round trip), which needs a finalized decoder.
 */
int w4j_encoder_forward(w4j_ctx *ctx, const float *mel, int n_frames, float *xa_out, int slot);

/*
 * The log-mel front end on the device (replaces FeatureExtractor.extract + padOrTrim,
 * W4J/audio/FeatureExtractor.java:68-160, with the model's filters as the
 * FeatureExtractor(nMels, melFilterData, nFftBins) constructor takes them, :44-55).
 * w4j_upload_mel_filters: the GGML file's mel filters, n_mels x n_bins f32 (n_fft = 2 (n_bins - 1)).
 * w4j_log_mel: 16 kHz mono samples -> n_mels x (2 n_audio_ctx) log-mel (host, when mel_out is not NULL).
 * w4j_encode_audio: the same spectrogram straight into the encoder (w4j_encoder_forward's outputs:
 * xa_out on the host, and / or stream `slot`'s cross K/V on the device) — one chunk of
 * WhisperModel.transcribe's feature + encoder stage (W4J/WhisperModel.java:361-366).
 */
int w4j_upload_mel_filters(w4j_ctx *ctx, const float *filters, int n_mels, int n_bins);
int w4j_log_mel(w4j_ctx *ctx, const float *audio, int n_samples, float *mel_out);
int w4j_encode_audio(w4j_ctx *ctx, const float *audio, int n_samples, float *xa_out, int slot);

/*
 * The chunked transcription loop (replaces WhisperModel.transcribeChunked, W4J/WhisperModel.java:334-427,
 * with parseTimestampSegments / findLastTimestampPos / buildPromptWithContext, :430-530): the whole
 * recording (16 kHz mono f32, host) is copied to the device once; per 30 s window at the seek
 * position the library runs the log-mel, the encoder, the cross K/V projection into stream 0 and
 * decodeWithFallback, retries without the previous-text context when it made the average
 * log-probability drop below -1, skips no-speech windows, cuts the tokens into timestamped
 * segments and advances the seek from the last timestamp.  Token ids only: the host's tokenizer
 * turns them into text.  A segment is kept when it has at least one text token (the reference keeps
 * it when the decoded text is not blank; the host drops segments whose text is blank).
 */
typedef struct w4j_transcribe_opts {
    const int32_t *sot;          /* tokenizer.sotSequence() (the prompt before the no-timestamps token) */
    int32_t n_sot;
    int32_t eot, no_speech;      /* token ids (tokenizer.eot(), tokenizer.noSpeech()) */
    int32_t no_timestamps;       /* appended to the prompt when ts_begin < 0 (buildPrompt, :573-582) */
    int32_t sot_prev;            /* the previous-text marker of buildPromptWithContext (:522-524) */
    int32_t ts_begin;            /* tokenizer.timestampBegin() with timestamps, -1 without */
    const int32_t *suppress;     /* buildSuppressTokens() */
    int32_t n_suppress;
    int32_t beam_size;           /* 1: greedy */
    int32_t condition_on_previous;
    uint64_t seed;               /* temperature-fallback sampling */
} w4j_transcribe_opts;

typedef struct w4j_segment {
    float start, end;            /* seconds */
    int32_t token_begin, n_tokens;  /* the segment's tokens: w4j_transcript.tokens[token_begin ..] */
} w4j_segment;

typedef struct w4j_transcript {
    int32_t *tokens;             /* caller's buffer: every segment's tokens, in order */
    int32_t tokens_cap;
    w4j_segment *segments;       /* caller's buffer */
    int32_t segments_cap;
    int32_t n_tokens, n_segments, n_windows;  /* out: used entries, 30 s windows decoded */
} w4j_transcript;

int w4j_transcribe(w4j_ctx *ctx, const float *audio, int n_samples, const w4j_transcribe_opts *opts,
                   w4j_transcript *out);

/*
 * WhisperDecoder.forward(tokens, xa, kvCache) (W4J/nn/WhisperDecoder.java:59-104)
 * for stream `slot`.  use_cache=1 appends the tokens to the slot's self-attention
 * cache (the kvCache map); use_cache=0 runs with an empty private cache and leaves
 * the slot's cache unchanged (kvCache == null, as detectLanguage does at
 * W4J/WhisperModel.java:548).  out_logits receives n_tokens x n_vocab f32.
 */
int w4j_forward(w4j_ctx *ctx, int slot, const int32_t *tokens, int n_tokens, int use_cache, float *out_logits);

/* Empty the self-attention cache of a stream (a fresh kvCache map). */
int w4j_reset_cache(w4j_ctx *ctx, int slot);

/*
 * Decode result per stream (WhisperDecoder.DecodeResult, W4J/nn/WhisperDecoder.java:672-673):
 * out_tokens[s * max_tokens .. + out_lens[s]) are the generated ids; sum/avg
 * log-probabilities, compression ratio and no-speech probability per stream.
 */
typedef struct w4j_result {
    int32_t *tokens;         /* n_streams * max_tokens */
    int32_t *lens;           /* n_streams */
    double *sum_logprob;     /* n_streams */
    float *avg_logprob;      /* n_streams */
    float *compression;      /* n_streams (zlib ratio, WhisperDecoder.java:628-647) */
    float *no_speech_prob;   /* n_streams */
} w4j_result;

/*
 * Greedy (temperature 0) or sampled decode of n_streams independent streams
 * (slots[i] names the stream whose encoder output was set), each starting from
 * its own prompt of n_prompt tokens (prompts: n_streams x n_prompt).  Mirrors
 * WhisperDecoder.decode (W4J/nn/WhisperDecoder.java:161-204) including the
 * logit processors (:450-564) and no-speech probability (:442-448).  ts_begin
 * <= 0 disables timestamp rules.  seed drives temperature sampling.
 */
int w4j_decode(w4j_ctx *ctx, const int32_t *slots, int n_streams, const int32_t *prompts, int n_prompt,
               int32_t eot, int max_tokens, const int32_t *suppress, int n_suppress, int32_t no_speech,
               float temperature, int32_t ts_begin, uint64_t seed, w4j_result *out);

/* Beam search (WhisperDecoder.decodeBeam, W4J/nn/WhisperDecoder.java:214-394). */
int w4j_decode_beam(w4j_ctx *ctx, const int32_t *slots, int n_streams, const int32_t *prompts, int n_prompt,
                    int32_t eot, int max_tokens, const int32_t *suppress, int n_suppress, int32_t no_speech,
                    int32_t ts_begin, int beam, w4j_result *out);

/*
 * Temperature-fallback policy (WhisperDecoder.decodeWithFallback,
 * W4J/nn/WhisperDecoder.java:119-149): beam search (beam > 1) or greedy at
 * t = 0, then sampling at 0.2 .. 1.0 while needsFallback (:435-440) holds.
 * out_temperature receives the temperature of the returned result per stream.
 */
int w4j_decode_with_fallback(w4j_ctx *ctx, const int32_t *slots, int n_streams, const int32_t *prompts,
                             int n_prompt, int32_t eot, int max_tokens, const int32_t *suppress, int n_suppress,
                             int32_t no_speech, int32_t ts_begin, int beam, uint64_t seed, w4j_result *out,
                             float *out_temperature);

/* Ask a running decode on this context to stop at its next step boundary
 * (TranscriptionHandle cancellation, W4J/WhisperModel.java:620-633). */
int w4j_cancel(w4j_ctx *ctx);

/* Host-side helpers of the policy (no device work). */
float w4j_compression_ratio(const int32_t *tokens, int n);                            /* :628-647 */
int w4j_needs_fallback(float compression_ratio, float avg_logprob, float no_speech);  /* :435-440 */

/*
 * Timing of the last decode call on this context: device milliseconds from the
 * first prompt kernel to the end of the result gather (the cross K/V projection
 * of w4j_set_encoder_output excluded), the number of graph-replayed steps after
 * the prompt, and the number of kernels launched.
 */
int w4j_last_timing(w4j_ctx *ctx, double *loop_ms, int *steps, long long *kernel_launches);

/*
 * In-chain kernel timing (measurement; no counterpart in the reference).  With a kernel class
 * set, the step graphs of later decode calls are captured with CUDA event records around every
 * launch of that class, and each step is waited for, so w4j_kernel_timing returns the summed
 * device milliseconds and the number of those launches over the graph-replayed steps of the last
 * decode call.  The events cost each timed launch its overlap with the launch before it, so use
 * this for a separate profiling call, not for the timed throughput.  Classes: 0 off,
 * 1 projections, 2 self-attention, 3 cross-attention, 4 vocabulary logits, 5 token selection.
 */
#define W4J_KC_PROJ 1
#define W4J_KC_SELF_ATTN 2
#define W4J_KC_CROSS_ATTN 3
#define W4J_KC_LOGITS 4
#define W4J_KC_SELECT 5
int w4j_set_kernel_timing(w4j_ctx *ctx, int kernel_class);
int w4j_kernel_timing(w4j_ctx *ctx, double *ms, long long *launches);

/* ---------------------------------------------------------------------------
 * Op-level entry points on device buffers (plain pointers on the context's
 * device, stream 0 of the calling thread unless `stream` is given).  They run
 * single kernels of the step for tests and for hosts that drive their own loop.
 * ------------------------------------------------------------------------- */

/*
 * y = LN?(x) . W^T + b for M rows (Linear.forward, W4J/nn/Linear.java:23-26,
 * optionally preceded by LayerNorm.forward, W4J/nn/LayerNorm.java:28-30).
 * W is a GGML F16 or Q8_0 payload already on the device: F16 (N x K halves), or
 * Q8_0 repacked by w4j_q8_0_repack.  ln_g/ln_b may be NULL (no LayerNorm).
 * epilogue: 0 = store, 1 = GELU (Tensor.geluInPlace), 2 = residual y += ...
 */
int w4j_op_linear(w4j_ctx *ctx, const float *x, int M, int K, const void *W, int w_type, int N,
                  const float *bias, const float *ln_g, const float *ln_b, int epilogue, float *y, void *stream);

/* Split a GGML Q8_0 payload (N*K/32 blocks of 34 bytes, device) into the
 * device layout: int8 quants (N x K) then f16 scales (N x K/32). dst holds N*K + N*K/16 bytes. */
int w4j_q8_0_repack(const void *src_device, int N, int K, void *dst_device, void *stream);

/*
 * logits = LN(x) . E^T over the vocabulary followed by argmax and log-softmax
 * of the chosen id, for M rows (WhisperDecoder.java:102-103 then argmax :566-574
 * and logSoftmax :614-626).  x: M x d f32, E: V x d f16, ln: d f32 each;
 * outputs token ids (M) and log-probabilities (M, double).  Scratch memory for
 * the per-block partial results is taken from the context (1 <= M <= max(max_streams *
 * max_beam, n_text_ctx)).  If a bounded wait inside the kernels ran out, every out_token of
 * that call is -1 and every out_logprob NaN (the context's error word for this op is cleared
 * for the next call).  Asynchronous on `stream`.
 */
int w4j_op_logits_argmax(w4j_ctx *ctx, const float *x, int M, const void *E, int V, const float *ln_g,
                         const float *ln_b, int32_t *out_token, double *out_logprob, void *stream);

/*
 * w4j_op_logits_argmax_noalloc — no counterpart in the reference.
 *
 * The computation of w4j_op_logits_argmax (same kernels, same results) for callers that
 * cannot let the library allocate device memory: a host that has handed the whole device to
 * its own arena or caching allocator (so a cudaMalloc would fail or fragment it), a process
 * under a fixed device-memory budget, or code that only needs this one op and holds no
 * decoder context (creating one allocates the weights, caches and scratch of a whole model).
 * It takes no context and never calls cudaMalloc, cudaFree or an allocating library routine.
 *
 * Scratch: the per-block partial results live in a file-scope device array of the library
 * (W4J_NOALLOC_MAX_ROWS x W4J_NOALLOC_MAX_PARTS records of 144 bytes = 360 KiB per device),
 * found with cudaGetSymbolAddress on the first call for each device.  That first call also
 * sets kernel attributes; make it before any stream capture begins on that device.
 * Nothing in the partials has to start at zero (each call writes every record it reads).
 * One device error word must be zero when a call starts: it is zero when the library loads,
 * and each call clears it at the end.
 *
 * Limits: 1 <= M <= W4J_NOALLOC_MAX_ROWS; d a multiple of 64 in [64, 1280]; x, E, ln_g and
 * ln_b 16-byte aligned; min(SM count, V) <= W4J_NOALLOC_MAX_PARTS.  Outside them the call
 * returns W4J_ERR_ARG with the reason in w4j_last_error() and launches nothing.
 *
 * Concurrency: calls on one device share the scratch.  Two calls whose executions overlap on
 * the device (different streams without an event between them, or different host threads)
 * race and return wrong ids; order them on one stream, or with events.
 *
 * device: the GPU holding every pointer (made current on the calling thread).  x: M x d f32,
 * E: V x d f16, ln_g/ln_b: d f32; out_token (M int32) and out_logprob (M double) on the device.
 * If a bounded wait inside the kernels ran out, every out_token of that call is -1 and every
 * out_logprob NaN.  Asynchronous on `stream` (NULL = legacy default stream).
 */
/*
 * Test hook (no counterpart in the reference): the next n_launches tcgen05 vocabulary passes of
 * w4j_op_logits_argmax / w4j_op_logits_argmax_noalloc issue none of their weight copies, so
 * every bounded wait inside them runs out (about a second) and the call reports it through its
 * error word (token -1, NaN log-probability).  Lets a test exercise that path without faulting
 * the GPU.  0 turns it off.
 */
int w4j_test_withhold_logits_copies(int n_launches);

#define W4J_NOALLOC_MAX_ROWS 16
#define W4J_NOALLOC_MAX_PARTS 160
int w4j_op_logits_argmax_noalloc(int device, const float *x, int M, int d, const void *E, int V,
                                 const float *ln_g, const float *ln_b, int32_t *out_token, double *out_logprob,
                                 void *stream);

/* ---------------------------------------------------------------------------
 * A paged key/value cache for hosts that drive their own loop (no counterpart in the reference, whose
 * kvCache map copies and concatenates, W4J/nn/MultiHeadAttention.java:140-164).  Rows (sequences) hold
 * pages of page_tokens tokens; a page may be held by many rows, so beams of a stream and re-decodes of a
 * window keep their common prompt once.  All memory is the caller's, on `device`:
 *
 *   pool    [2 n_layer][n_pages][n_kv_head][page_tokens][head_dim], F16 or BF16, 16-byte aligned; plane 2 l
 *           holds the keys of layer l, plane 2 l + 1 its values
 *   ref     [n_pages] rows that hold each page (0: free)
 *   table   [n_rows][table_width] page of each run of page_tokens tokens; entries behind a row's length
 *           are neither read nor written
 *   len     [n_rows] tokens of each row
 *   status  [1] what calls could not do, W4J_PAGES_* bits, added up until the caller clears it
 *   work    w4j_op_pages_workspace's bytes of scratch that belong to this cache for as long as it lives and that
 *           all of its calls share, captured ones too: it keeps which rows' last extension was refused
 *
 * A new cache is ref, len, status and work set to zero.  A last page that is not full belongs to one row alone:
 * every call here keeps that so, and a caller that builds tables of its own has to.
 *
 * The calls are asynchronous on `stream` and change the cache in stream order; calls on one cache that
 * may run at the same time (several streams without an event between them) are the caller's to order, and
 * so are replays of graphs that hold them.  The integer arguments (rows, start, dst, src) are device arrays
 * that must stay as they are until the call has run.  Each call but a write is all or nothing: where a row is
 * out of range or named twice, a length does not fit or the free pages do not suffice, it changes nothing but
 * `status`.  New pages are the lowest free ones in the order of the call's rows; pages that a call lets go
 * of are free for the next call.  page_tokens is a multiple of 8 up to 1024, head_dim 64 or 128.
 * ------------------------------------------------------------------------- */
#define W4J_PAGES_BAD_ROW 1   /* a row out of range, or named twice by one call */
#define W4J_PAGES_FULL 2      /* too few free pages */
#define W4J_PAGES_TOO_LONG 4  /* a row would outgrow its table */
#define W4J_PAGES_BAD_START 8 /* start does not begin at 0, does not ascend or does not fit the row lengths */
#define W4J_PAGES_BAD_PAGE 16 /* a table entry out of range, or in fork, free and compact one whose page nobody holds */

typedef struct w4j_pages {
    int32_t device;
    int32_t type;                /* of the pool: W4J_GGML_F16 or W4J_GGML_BF16 */
    int32_t n_layer, n_kv_head, head_dim, page_tokens, n_pages, n_rows, table_width;
    void *pool;
    int32_t *ref, *table, *len, *status;
    void *work;
    size_t work_bytes;
} w4j_pages;

/* Bytes of scratch (16-byte aligned) that a cache of these sizes needs (its pointers are not looked at). */
int w4j_op_pages_workspace(const w4j_pages *cache, size_t *bytes);

/* Row rows[i] grows by start[i + 1] - start[i] tokens (start: n + 1 ascending numbers from 0), whose keys
 * and values w4j_op_pages_write brings layer by layer. */
int w4j_op_pages_extend(const w4j_pages *cache, const int32_t *rows, const int32_t *start, int n, void *stream);

/* Keys and values of the last start[i + 1] - start[i] tokens of row rows[i], as tokens start[i] ..
 * start[i + 1] - 1 of k and v (n_tokens = start[n] tokens of [n_kv_head][head_dim], k_stride and v_stride
 * elements apart, multiples of 8, both 16-byte aligned: the K and V parts of a fused projection can stay in
 * place).  After w4j_op_pages_extend of the same rows and start.  A row whose last extension was refused takes no
 * tokens until one succeeds (its length has not grown: theirs would be the places of its last ones): they are left
 * out and raise that refusal's status bits again.  Tokens whose row or page is out of range, and tokens that start
 * deals to no row, are left out and raise their status bit.  So are those of a row that is named twice, but for the index
 * that it has in its last extension's rows. */
int w4j_op_pages_write(const w4j_pages *cache, int layer, const int32_t *rows, const int32_t *start, int n,
                       const void *k, int64_t k_stride, const void *v, int64_t v_stride, int n_tokens, void *stream);

/* Row dst[i] becomes what row src[i] was before the call, for all i at once (a beam reorder, or new
 * beams off one row); src[i] = -1 empties dst[i].  Full pages are shared.  A last page that is not full stays
 * with one holder (the source row if it goes on, else the lowest i that takes it over) and is copied, as far
 * as it is filled, to a new page for every other. */
int w4j_op_pages_fork(const w4j_pages *cache, const int32_t *dst, const int32_t *src, int n, void *stream);

/* The rows become empty; pages that nobody else holds become free. */
int w4j_op_pages_free(const w4j_pages *cache, const int32_t *rows, int n, void *stream);

/* Moves the held pages to the front of the pool: with n of them held, the i-th lowest free page below n
 * takes over the i-th lowest held page from n on, in the tables of all rows too.  n_live (device, may be
 * NULL) gets n: pages n .. n_pages - 1 are free afterwards and may be cut off. */
int w4j_op_pages_compact(const w4j_pages *cache, int32_t *n_live, void *stream);

/*
 * Attention of one layer over a paged cache, for a batch whose groups share their first tokens (the
 * softmax(q k^T) v of W4J/nn/MultiHeadAttention.java:77-132 for many sequences at once).
 *
 * Sequence i (0 <= i < n_seq) is row rows[i] of the cache; group g is sequences group_start[g] ..
 * group_start[g + 1] - 1 (n_group + 1 ascending numbers from 0 to n_seq).  All sequences of group g hold the
 * same first shared[g] tokens, on the same pages or on copies of them: their keys and values are read
 * once for the whole group, through the table of its first sequence.  Query t (0 <= t < n_query) of a
 * sequence sees the first len - n_query + t + 1 tokens of its row: the last n_query tokens are the queries'
 * own, already written.  A query that sees no token, or none that scores more than -inf, gets zeros.  What lies
 * behind a row's length, and what a query does not see, may be anything, NaN included.
 *
 *   q, out  [n_seq n_query] tokens of [n_head][head_dim] of the cache's type, q_stride and out_stride
 *           elements apart (multiples of 8, 16-byte aligned); query head h reads key/value head h / (n_head / n_kv_head)
 *   shared[g] may be at most max_shared, and at most len - n_query + 1 (or 0) of each of its rows.  max_shared and
 *           max_own (an upper bound of len - shared over the rows) size the launch; only max_shared is a limit
 *   work    w4j_op_attn_shared_workspace's bytes, 16-byte aligned, for this call alone until it has run
 *
 * Scores, the softmax and all sums are held in 32 bits; the softmax's weights are rounded to the cache's
 * type before they meet the values.  A sequence whose row, group or shared length is bad, or whose table names a
 * page that is not there, gets NaN, and the cache's status its bit; so do the sequences that a wait inside the
 * kernels concerns, if it runs out.  Asynchronous on `stream`; results do not depend on the order in which blocks run.
 */
#define W4J_PAGES_BAD_SHARED 32 /* a shared length over max_shared, or over what a row's queries all see */
#define W4J_PAGES_TIMEOUT 64    /* a bounded wait inside a kernel ran out */

typedef struct w4j_attn_shared {
    const w4j_pages *cache;
    int32_t layer, n_head, n_query, n_seq, n_group, max_shared, max_own;
    float scale;
    const void *q;
    void *out;
    int64_t q_stride, out_stride;
    const int32_t *rows, *group_start, *shared;
    void *work;
    size_t work_bytes;
} w4j_attn_shared;

/* Bytes of scratch a call of these sizes needs, 0 for a few rows that are not very long (pointers and strides are not looked at). */
int w4j_op_attn_shared_workspace(const w4j_attn_shared *args, size_t *bytes);
int w4j_op_attn_shared(const w4j_attn_shared *args, void *stream);

/*
 * Test hook: in the next n_calls of w4j_op_attn_shared every wait for keys and values counts on 16 bytes more than
 * are copied, so that it runs out (a second or two) and the call reports W4J_PAGES_TIMEOUT.  0 turns it off.
 */
int w4j_test_attn_shared_waits_run_out(int n_calls);

/* ---------------------------------------------------------------------------
 * A Linear layer in 8-bit integers with a scale for each row of activations and each output channel (the
 * product of W4J/nn/Linear.java:23-26 with both operands quantised; w4j_op_linear keeps the activations).
 * ------------------------------------------------------------------------- */

/*
 * q = round(x / s), s = max |x| (1 / 127), 1 / 127 as a 32-bit float and the product rounded to one, for each of M rows
 * of K elements (ldx elements apart, of type
 * x_type: F32, F16 or BF16), optionally behind a LayerNorm (ln_g and ln_b, K floats each, or both NULL).  The
 * quotient is rounded as if exact, ties to even, and kept within +-127.  q has rows ldq bytes apart (a multiple of 16 of at least
 * K, 16-byte aligned); columns K up to the next multiple of 16 get zeros.  A row of zeros gets scale 0, a row with
 * an infinity or a NaN zeros and scale NaN, which a product hands on to all of the row's outputs.  The weights of
 * a layer are quantised by the same call, a row being an output channel.
 */
int w4j_op_quantize_rows(int device, const void *x, int x_type, int M, int K, int64_t ldx, const float *ln_g,
                         const float *ln_b, int8_t *q, int64_t ldq, float *scale, void *stream);

/*
 * y[m][n] = x_scale[m] w_scale[n] sum_k x[m][k] w[n][k] + bias[n] (bias may be NULL), the sum exact in 32-bit
 * integers, the rest in 32-bit floats, rounded once to y_type (F32, F16 or BF16).  x: M rows, w: N rows,
 * ldx and ldw bytes apart (multiples of 16), 16-byte aligned, columns K up to the next multiple of 16 zero (as
 * w4j_op_quantize_rows leaves them).  K at most 131056.  y: rows ldy elements apart, at least N.  epilogue: 0 =
 * store, 1 = GELU (tanh form in 32 bits; w4j_op_linear looks the same function up by the f16 of its argument),
 * 2 = residual y += ....  y may not overlap the inputs.  If a bounded wait inside the kernels runs out, the outputs that
 * it concerns are NaN (there is no status word to say so).
 */
int w4j_op_linear_i8(int device, const int8_t *x, int64_t ldx, const float *x_scale, int M, int K, const int8_t *w,
                     int64_t ldw, const float *w_scale, int N, const float *bias, int epilogue, void *y, int y_type,
                     int64_t ldy, void *stream);

/*
 * The two in one call, x in floats (as w4j_op_quantize_rows) and y as w4j_op_linear_i8 makes it: up to 4 rows that fit
 * 1536 bytes as integers take one launch.  Behind a LayerNorm its sums may run in another order there, so that a quotient
 * next to a half may fall to its other side.  work: w4j_op_linear_i8_layer_workspace's bytes (0 for those few rows),
 * 16-byte aligned, for this call alone until it has run.
 */
int w4j_op_linear_i8_layer_workspace(int M, int K, size_t *bytes);
int w4j_op_linear_i8_layer(int device, const void *x, int x_type, int64_t ldx, const float *ln_g, const float *ln_b, int M,
                           int K, const int8_t *w, int64_t ldw, const float *w_scale, int N, const float *bias,
                           int epilogue, void *y, int y_type, int64_t ldy, void *work, size_t work_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* WHISPER4J_CUDA_H */
