/*
 * mitok.h — C ABI of the MI355X token loop for the rustCrates transformer.
 *
 * The reference crate (src/neural_networks/..., Rust, CPU-only) has no
 * foreign-function boundary on this path except the OpenBLAS `zgemm_` it
 * calls (utils/matrix.rs:13-15).  This header is the boundary a Rust FFI crate
 * binds instead: each entry point names the Rust item it replaces.  The Rust
 * declarations of this header are bindings/rust/mitok-sys/src/lib.rs.
 *
 * Conventions
 *  - Complex<f64> (num-complex 0.4.6, #[repr(C)] {re, im}) crosses the ABI as
 *    two interleaved doubles; a [rows][cols] complex matrix is rows*cols*2
 *    doubles, row-major, exactly Vec<Vec<Complex<f64>>> flattened.
 *  - Weight layouts are the reference's: Linear/Dense weights [in][out]
 *    (linear_layer.rs:38, layer.rs:268), attention heads [heads][dim][head_dim]
 *    (masked_attention_head.rs:64-75), bias_pos [heads][max_ctx][max_ctx].
 *  - A NULL tensor leaves the device tensor zeroed (fill it with
 *    mitok_init_seeded); NULL gamma/beta/biases take the reference's initial
 *    values (gamma 1, beta 0: norm_layer.rs:45-50; biases 1+0i: layer.rs:269,
 *    linear_layer.rs:39).
 *  - Every call returns 0 or a MITOK_ERR_* code and never aborts; the message
 *    is in mitok_last_error() (thread-local).  Where the reference panics
 *    (NaN in GELU, non-finite FFN output, unknown token id, NaN logits), the
 *    call returns MITOK_ERR_NAN / MITOK_ERR_ARG instead.
 *  - A network is used by one thread at a time (the reference takes
 *    &mut NeuralNetwork); calls are synchronous on return.
 */
#ifndef MITOK_H
#define MITOK_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MITOK_OK 0
#define MITOK_ERR_ARG 1
#define MITOK_ERR_HIP 2
#define MITOK_ERR_STATE 3
#define MITOK_ERR_NAN 4
#define MITOK_ERR_NOMEM 5

/* OperationMode (network_types/neural_network_generic.rs:17-20) */
#define MITOK_TRAINING 0
#define MITOK_PRODUCTION 1

/* mitok_set_learning_rate: every layer; mitok_get_learning_rate: the
 * network's own rate (NeuralNetwork::learning_rate) */
#define MITOK_ALL_LAYERS 0xFFFFFFFFu
#define MITOK_NETWORK_RATE 0xFFFFFFFFu

/* operators of a serving loop: a drafted token without a parent among the
 * drafted ones (or a sequence without one); no token (an unused entry, or no
 * answer); no cached row; no page of a paged cache; continuations kept of a group
 * of beams at most */
#define MITOK_NO_PARENT 0xFFFFFFFFu
#define MITOK_NO_TOKEN 0xFFFFFFFFu
#define MITOK_NO_ROW 0xFFFFFFFFu
#define MITOK_NO_PAGE 0xFFFFFFFFu
#define MITOK_TREE_MAX_NODES 256
#define MITOK_BEAM_MAX_KEEP 64

/* kernel classes for mitok_timing_enable */
#define MITOK_TIME_VOCAB 1       /* the vocab Linear (the Linear before Softmax) */
#define MITOK_TIME_LAYER_GEMM 2  /* Q/K/V and FFN projections of one-row (decode) calls */
#define MITOK_TIME_ATTENTION 3   /* attention kernels */
#define MITOK_TIME_STEP 4        /* one whole decode step (one token for every sequence) */
#define MITOK_TIME_PREFILL_GEMM 5 /* Q/K/V and FFN projections of calls with several rows per sequence */

typedef struct mitok_network mitok_network; /* NeuralNetwork (neural_network_generic.rs:23-31) */

int mitok_version(void);
const char* mitok_last_error(void);
int mitok_device_count(int* count);

/* create(...) (neural_network_generic.rs:76-88): an empty layer list on `device`. */
int mitok_network_create(int device, mitok_network** out);
void mitok_network_destroy(mitok_network* net);
int mitok_num_layers(const mitok_network* net);

/* ---- LayerEnum variants, appended in order (network_components/layer.rs:75-88) ---- */
/* EmbeddingLayer (embedding_layer.rs:24-36, forward :158-211); table [vocab][dim] */
int mitok_add_embedding(mitok_network* net, uint32_t vocab, uint32_t dim, const double* table);
/* PositionalEncodingLayer (positional_encoding_layer.rs:15-32, forward :35-99) */
int mitok_add_positional_encoding(mitok_network* net, uint32_t dim, double base);
/* NormalNormLayer (norm_layer.rs:17-62, forward :84-130) */
int mitok_add_norm(mitok_network* net, uint32_t dim, double eps, const double* gamma, const double* beta);
/* SelfAttentionLayer of `heads` MaskedAttentionHeads plus its NormalNormLayer
 * (self_attention_layer.rs:29-50, forward :55-133; masked_attention_head.rs:64-106,
 * forward :122-220).  max_ctx sizes bias_pos (the reference fixes it at 512,
 * transformer_network.rs:32) and the KV cache. */
int mitok_add_self_attention(mitok_network* net, uint32_t heads, uint32_t dim, uint32_t max_ctx, double eps,
                             const double* wq, const double* wk, const double* wv, const double* bias_pos,
                             const double* gamma, const double* beta);
/* FeedForwardLayer = Dense(GELU) -> Linear (feedforward_layer.rs:30-48, forward :56-138) */
int mitok_add_feed_forward(mitok_network* net, uint32_t dim, uint32_t hidden, const double* w1, const double* b1,
                           const double* w2, const double* b2);
/* LinearLayer (linear_layer.rs:37-54, forward :55-75); w [in][out] */
int mitok_add_linear(mitok_network* net, uint32_t in, uint32_t out, const double* w, const double* b);
/* SoftmaxLayer (softmax_output_layer.rs:30-65) */
int mitok_add_softmax(mitok_network* net, int operation_mode);
/* DiscreteWaveletLayer (network_types/wavelet_discrete_layer.rs:46-161), partial
 * mode, over rows of `dim` features.  At a prompt pass (and a stateless one)
 * it replaces each sequence's S rows by the low half of dwt_1d along the
 * sequence of every feature (wavelet_transform/dwt.rs:36-90), and the padding
 * mask by its thresholded low half (:297-313); later layers and the KV cache
 * see S' = mitok_seq_out_len rows.  A cached step's row passes through, and
 * its RoPE position still counts the uncompressed prompt (time_step,
 * transformer_network.rs:300-304).  wavelet: DiscreteWaletetType index (0 DB1,
 * 1 DB2); mode: WaveletMode index (0 ZERO, 1 CONSTANT, 2 SYMMETRIC,
 * 3 ANTISYMMETRIC, 4 REFLECT, 6 PERIODIC); is_full_mode must be 0.  Others
 * are MITOK_ERR_ARG. */
int mitok_add_discrete_wavelet(mitok_network* net, uint32_t dim, uint32_t wavelet, uint32_t mode, int is_full_mode);
/* Rows per sequence that layers [first, last) leave of a prompt pass of `seq`
 * rows (the wavelet layers compress them): the row count of mitok_predict's
 * and mitok_forward_layers' outputs. */
int mitok_seq_out_len(const mitok_network* net, uint32_t first, uint32_t last, uint32_t seq, uint32_t* out);

/* Seeded Xavier-uniform weights (initialize_weights_complex, utils/weights_initializer.rs:73-89),
 * computed on the device from a counter generator: the CPU checker holds the same values. */
int mitok_init_seeded(mitok_network* net, uint64_t seed);
/* EmbeddingLayer::new's embeddings (embedding_layer.rs:40-77) for the
 * Embedding at `layer`: for every token id, create_embedding draws src_dim
 * values uniform in [-0.4, 0.5) (here the counter generator on stream
 * (layer << 12) | 0xFFF, index id * src_dim + k, where the reference draws
 * from the unseeded rand::rng()), decomposes them with
 * decompose_in_wavelet_2d_default (network_types/wavelet_network.rs:42-135:
 * 5 levels of DB1/SYMMETRIC dwt_2d_full keeping the LL quadrant, then the
 * CMOR CWT at scales 2, 8, 16, 32) and keeps the first scale's row.  src_dim:
 * a power of two up to 4096 (512 in create_transformer) whose decomposed
 * width is the layer's dim (16 for 512). */
int mitok_init_embedding_wavelet(mitok_network* net, uint32_t layer, uint64_t seed, uint32_t src_dim);
/* Reads a weight tensor back (slots as in oracle/oracle.h; slot 3 = Re(bias_pos), n doubles). */
int mitok_get_tensor(mitok_network* net, uint32_t layer, uint32_t slot, double* out, uint64_t n);
/* Drops every KV cache (k_cache = v_cache = None, masked_attention_head.rs:54-57). */
int mitok_reset(mitok_network* net);

/* predict (transformer_network.rs:315-504).  ids [batch][seq], right-padded:
 * entries at or beyond lens[b] become PAD=1 (embedding_layer.rs:112-155).
 * time_steps [batch] or NULL: RoPE position when forward_only && > 0.
 * forward_only: KV-cache semantics (masked_attention_head.rs:135-178) and
 *   out = Re(logits) (convert_c_to_f64_3d); otherwise stateless and out = the
 *   SoftmaxLayer output for its OperationMode.
 * last_row_only: out is [batch][vocab] from each sequence's last row, else
 *   [batch][seq'][vocab] with seq' = mitok_seq_out_len (seq without wavelet layers).
 * out_padding_mask [batch][seq'] or NULL (the mask the last layer saw). */
int mitok_predict(mitok_network* net, const uint32_t* ids, const uint32_t* lens, uint32_t batch, uint32_t seq,
                  const uint32_t* time_steps, int forward_only, int last_row_only, double* out,
                  uint32_t* out_padding_mask);
/* The training pass of train (transformer_network.rs:73-79): mitok_predict with
 * forward_only = 0 when each sequence's last target_rows ids are its targets
 * (LayerInput's target_batch_ids).  Only the DiscreteWavelet layer reads them:
 * it compresses each sequence's first seq - target_rows rows and passes the
 * target rows on (wavelet_discrete_layer.rs:102-134, separate_input_target
 * :233-279), so seq' = mitok_seq_out_len(seq - target_rows) + target_rows per
 * wavelet layer.  With a wavelet layer and target_rows > 0 every sequence
 * must be unpadded (lens[b] == seq; the reference panics otherwise).
 * out_probs [batch][seq'][vocab] or NULL: the softmax output then stays on the
 * device, where mitok_cross_entropy_loss and mitok_backward read it. */
int mitok_predict_targets(mitok_network* net, const uint32_t* ids, const uint32_t* lens, uint32_t batch, uint32_t seq,
                          uint32_t target_rows, double* out_probs, uint32_t* out_padding_mask);
/* cross_entropy_loss_batch (transformer_network.rs:662-711), which train
 * (:81) computes on predict's softmax output, computed on the device from the
 * output the last stateless predict left there, so the [batch][seq'][vocab]
 * probabilities need not cross PCIe.  targets [batch][max_t] (target_lens[b]
 * used of each row, max_t <= 8192), the same arrays mitok_backward takes.
 * out_loss[2] = the complex loss (re, im): per sequence the mean of
 * -ln(p + 1e-15) over its non-PAD targets (p at row seq' - len - 1 + t),
 * then the mean over the batch.  MITOK_ERR_ARG where the reference would
 * panic (a target id >= vocab, fewer than len + 1 rows); the forward pass
 * stays valid for mitok_backward. */
int mitok_cross_entropy_loss(mitok_network* net, const uint32_t* targets, const uint32_t* target_lens, uint32_t batch,
                             uint32_t max_t, double* out_loss);

/* Layers [first, last) on hidden states: in [batch][seq][dim_in] complex,
 * out [batch][seq][dim_out] complex; padding_mask [batch][seq] or NULL (all 1).
 * This is each layer's forward(&LayerInput) -> LayerOutput chained. */
int mitok_forward_layers(mitok_network* net, uint32_t first, uint32_t last, const double* in,
                         const uint32_t* padding_mask, uint32_t batch, uint32_t seq, const uint32_t* time_steps,
                         int forward_only, double* out);
/* mitok_forward_layers on device buffers (the per-layer drop-in for a caller
 * whose hidden states stay on the GPU): d_in and d_out are device memory of the
 * network's GPU (hipMalloc), d_out [batch][seq'][dim_out] with
 * seq' = mitok_seq_out_len.  padding_mask and time_steps stay host arrays.  A
 * pointer that is not device memory of that GPU, or an allocation too small
 * for the shape, is MITOK_ERR_ARG. */
int mitok_forward_layers_device(mitok_network* net, uint32_t first, uint32_t last, const double* d_in,
                                const uint32_t* padding_mask, uint32_t batch, uint32_t seq,
                                const uint32_t* time_steps, int forward_only, double* d_out);

/* Greedy token loop on ids (predict_token_by_token, transformer_network.rs:165-313,
 * without the text tokenizer): resets the caches, runs the prompt, then feeds
 * each greedy id back for n_new tokens in total.  Sequence b of a batch is an
 * independent batch-1 run.  Only token ids cross PCIe per step.
 * out_ids [batch][n_new]; out_logits [n_new][batch][vocab] or NULL. */
int mitok_generate(mitok_network* net, const uint32_t* prompt, const uint32_t* lens, uint32_t batch, uint32_t seq,
                   uint32_t n_new, uint32_t* out_ids, double* out_logits);

/* The token loop one step at a time, for a host loop that inspects every id
 * (predict_token_by_token, transformer_network.rs:225-304: the prompt at t = 0,
 * then one fed token per step, the "<eos>" check and the print per token on the
 * host).  Only ids cross PCIe: 4 B per sequence per step.
 * mitok_prefill: resets the caches (k_cache = None) and runs the prompt
 *   (ids [batch][seq] right-padded as for mitok_predict); out_ids [batch] = the
 *   greedy id of each sequence's last prompt row; out_logits [batch][vocab]
 *   Re-logits of that row, or NULL.
 * mitok_decode_step: feeds ids [batch] (NULL: the ids the previous prefill or
 *   step returned, already on the device; MITOK_ERR_STATE where a mitok_predict
 *   used the caches last) at position = each sequence's KV length, appends to
 *   the caches; out_ids [batch] = the next greedy ids; out_logits
 *   [batch][vocab] or NULL.  batch must equal the prefill's.
 * On error the caches are dropped (prefill again). */
int mitok_prefill(mitok_network* net, const uint32_t* prompt, const uint32_t* lens, uint32_t batch, uint32_t seq,
                  uint32_t* out_ids, double* out_logits);
int mitok_decode_step(mitok_network* net, const uint32_t* ids, uint32_t batch, uint32_t* out_ids, double* out_logits);

/* The output head's training step: backward (transformer_network.rs:506-636)
 * through the Softmax and the vocab Linear of the last stateless predict
 * (forward_only = 0; any other call in between is MITOK_ERR_STATE).
 * SoftmaxLayer::backward (softmax_output_layer.rs:67-145): targets [batch][T],
 * tlens[b] of them used; the cross-entropy gradient of the softmax output
 * rows that predict them.  LinearLayer::backward (linear_layer.rs:77-128):
 * dW = conj(X)^T G, db = column sums, and out_grad_input [batch][seq'][d_in]
 * (complex) = G conj(W)^T, or NULL.  update_params: LinearLayer::
 * update_parameters (linear_layer.rs:130-175) at learning_rate: the layer's
 * first update descends by the clipped gradient / batch, later ones run
 * AdamW (utils/adam_w.rs:9-103) at time_step.  The weights stay on the
 * device (mitok_get_tensor reads them).  The layers below the vocab Linear
 * are not differentiated. */
int mitok_backward_head(mitok_network* net, const uint32_t* targets, const uint32_t* tlens, uint32_t batch, uint32_t T,
                        int update_params, double learning_rate, uint32_t time_step, double* out_grad_input);
/* The same reverse walk (transformer_network.rs:506-636) through n_layers
 * layers below the Softmax: 1 = the vocab Linear (mitok_backward_head), up to
 * every layer the stateless predict ran.  Each layer's backward and, with
 * update_params, its update_parameters where the walk calls it:
 *  - Linear: as above, at time_step;
 *  - FeedForward (feedforward_layer.rs:140-186, 219-250): its Linear at
 *    time_step, then its Dense with the GELU derivative of
 *    utils/derivative.rs:48-84 at step 1 (Layer::time_step is never set,
 *    layer.rs:111,285);
 *  - SelfAttention (self_attention_layer.rs:135-196, 260-273): its Norm's
 *    backward (norm_layer.rs:132-209), then every head
 *    (masked_attention_head.rs:222-345); updates the Norm's gamma and beta,
 *    wq / wk / wv and Re(bias_pos) on the pass's S x S slice;
 *  - Norm (backward only), PositionalEncoding (positional_encoding_layer.rs:
 *    101-144);
 *  - Embedding: passes the gradient on; with update_params
 *    EmbeddingLayer::update_parameters (embedding_layer.rs:223-264) moves and
 *    renormalizes the table rows of the target ids.
 *  - DiscreteWavelet (wavelet_discrete_layer.rs:163-207): the gradient of
 *    the compressed rows through decompress_partial (grad_dwt_1d_trend) and
 *    align_gradient_rows_complex, the target rows' gradient passed through.
 * out_grad_input: the gradient of the lowest walked layer's input
 * [batch][rows of that layer's input][its d_in], or NULL. */
int mitok_backward(mitok_network* net, const uint32_t* targets, const uint32_t* tlens, uint32_t batch, uint32_t T,
                   uint32_t n_layers, int update_params, double learning_rate, uint32_t time_step,
                   double* out_grad_input);

/* backward(transformer_network, target_ids, update_params) as train calls it
 * (transformer_network.rs:129, 506-636): the whole reverse walk over every
 * layer the last stateless predict ran, each layer updated at its own
 * learning rate (mitok_set_learning_rate) and the Embedding at the network's
 * (transformer_network.rs:520, mitok_set_network_learning_rate); otherwise as
 * mitok_backward. */
int mitok_backward_walk(mitok_network* net, const uint32_t* targets, const uint32_t* tlens, uint32_t batch, uint32_t T,
                        int update_params, uint32_t time_step, double* out_grad_input);

/* Learning rates (neural_network_generic.rs:57-73, 115-186).  Every layer
 * starts at 0.01 (create_transformer's rate, transformer_builder.rs:16), the
 * network too.  mitok_set_learning_rate(net, MITOK_ALL_LAYERS, lr) is
 * update_learning_rate (what update_step_lr_scheduler calls); with a layer
 * index it sets that layer's field (a SelfAttention's heads and Norm, a
 * FeedForward's Dense and Linear together).  mitok_set_network_learning_rate
 * sets NeuralNetwork::learning_rate, which decay_learning_rate halves and the
 * Embedding's update reads; mitok_get_learning_rate(net, MITOK_NETWORK_RATE)
 * reads it back. */
int mitok_set_learning_rate(mitok_network* net, uint32_t layer, double learning_rate);
int mitok_get_learning_rate(const mitok_network* net, uint32_t layer, double* out);
int mitok_set_network_learning_rate(mitok_network* net, double learning_rate);
/* reset_previous_gradient (neural_network_generic.rs:188-242), which train
 * calls when the loss keeps rising (transformer_network.rs:147-151): the next
 * update of every Linear, FeedForward sublayer and attention head is the
 * clipped descent again, and the AdamW after it starts from zero moments.  An
 * attention layer's Norm keeps its moments, as in the reference. */
int mitok_reset_previous_gradient(mitok_network* net);

/* greedy_decoding (src/utils/sampling_methods.rs:5-18) on the device for host
 * logits [rows][vocab]: last index among equal maxima; NaN -> MITOK_ERR_NAN. */
int mitok_greedy_decoding(mitok_network* net, const double* logits, uint32_t rows, uint32_t vocab, uint32_t* out_ids);
/* greedy_decoding on device buffers: d_logits [rows][vocab] f64 and d_out_ids
 * [rows] are device memory of the network's GPU, checked as for
 * mitok_forward_layers_device. */
int mitok_greedy_decoding_device(mitok_network* net, const double* d_logits, uint32_t rows, uint32_t vocab,
                                 uint32_t* d_out_ids);

/* mitok_greedy_decoding without any device allocation.  No counterpart in the
 * reference: it is for callers that cannot allocate device memory (tight
 * serving loops, harnesses that forbid hipMalloc).  It copies the host logits
 * in and synchronises the network's stream before it returns, so it must not
 * be called while that stream is being captured into a graph, and it is not
 * recorded into a capture on another stream.  The logits and ids are staged in a
 * fixed per-GPU array of the library (8 MiB + 16 KiB, held by every GPU the
 * library runs on until the process ends): rows * vocab <= 1048576 and
 * rows <= 4096, else MITOK_ERR_ARG.  All calls on one GPU share that array, so
 * calls that overlap on one GPU (two networks on one device used from two
 * threads) race; calls through one network are serialised by its stream. */
int mitok_greedy_decoding_noalloc(mitok_network* net, const double* logits, uint32_t rows, uint32_t vocab,
                                  uint32_t* out_ids);

/* ---- operators of a serving loop (no reference counterpart) ----
 * Drafted tokens checked several at a time, rows evicted from the cache by the
 * attention they received, and rules that turn logits into a token.  The
 * *_device entry points work on device arrays of the network's GPU (checked:
 * in one allocation, aligned to 16 bytes for complex arrays and to their
 * elements otherwise; outputs overlap nothing but where in place is allowed).
 * They run on the network's stream, behind everything queued on the device's
 * default stream before the call (work on other streams has to be finished),
 * and are complete on return; so they cannot be captured into a graph.
 * Lengths, parents and paths are host arrays. */

/* Attention of a tree of drafted tokens over a KV cache.  Sequence b has
 * kv_lens[b] committed rows and counts[b] <= nodes drafted ones (counts NULL:
 * nodes of each; at most MITOK_TREE_MAX_NODES), whose keys and values already
 * lie behind them: node i in slot kv_lens[b] + i.  parents[b][i] < i, or
 * MITOK_NO_PARENT.  Node i attends over the committed rows, its ancestors and
 * itself:
 *   score(i, t) = Re(sum_e q_i[e] k_t[e]) / (1e-8 + sqrt(head_dim)) + bias[h][column(t)]
 *   column(t) = t for a committed row, kv_lens[b] + depth for a drafted one
 *   out_i = sum_t softmax(score(i, .))_t v_t
 * (scale_attention_scores and bias row 0, masked_attention_head.rs:184-208,
 * 453-465), so a chain of nodes gives what decode steps one by one give.  A
 * row that a node does not see has no part in its output, finite or not; rows
 * past counts[b] are zero.
 *   d_q, d_out [batch][nodes][heads * head_dim] complex
 *   d_k_cache, d_v_cache [batch][heads][max_ctx][head_dim] complex, head_dim <= 256, max_ctx <= 2^30,
 *     batch * heads <= 2^18 (here and in an eviction)
 *   d_bias [heads] rows of real numbers, bias_stride apart, or NULL
 *   d_weights [batch][heads][max_ctx] or NULL: the softmax weights that the
 *     first weigh_nodes nodes give each slot are summed; committed slots are
 *     added to, the drafted ones set. */
int mitok_tree_attention_device(mitok_network* net, const double* d_q, const double* d_k_cache,
                                const double* d_v_cache, const double* d_bias, uint64_t bias_stride,
                                const uint32_t* kv_lens, const uint32_t* parents, const uint32_t* counts,
                                uint32_t batch, uint32_t nodes, uint32_t heads, uint32_t head_dim, uint32_t max_ctx,
                                uint32_t weigh_nodes, double* d_weights, double* d_out);
/* A tree of drafted tokens through the whole stack, on the caches that
 * mitok_prefill (or a forward_only mitok_predict) left: ids, parents
 * [batch][nodes], counts as above.  A node's output is what decode steps along
 * its path would give (RoPE position and bias column by its depth).
 * out_ids [batch][nodes] or NULL: the greedy id after each node (MITOK_NO_TOKEN
 * past counts[b]); out_logits [batch][nodes][vocab] or NULL: its Re-logits.
 * weigh_nodes > 0: the attention that the first weigh_nodes nodes pay is kept
 * per layer, head and cached row, for mitok_evict_rows (1: the root, a token
 * already decided).  The step itself adds it, whether its nodes are committed
 * or not: a step repeated, or one whose tree is dropped, has weighed all the
 * same (such a step weighs once if the others pass 0).  The caches' committed
 * rows stay as they are: mitok_tree_accept
 * commits nodes, any other call on the caches drops them.  Every sequence
 * needs room for `nodes` rows.  On an error of the pass the caches are dropped. */
int mitok_tree_step(mitok_network* net, const uint32_t* ids, const uint32_t* parents, const uint32_t* counts,
                    uint32_t batch, uint32_t nodes, uint32_t weigh_nodes, uint32_t* out_ids, double* out_logits);
/* mitok_tree_step with the logits [batch][nodes][vocab] left in device memory,
 * where mitok_process_logits_device reads them (rows past counts[b] have no
 * meaning). */
int mitok_tree_step_device(mitok_network* net, const uint32_t* ids, const uint32_t* parents, const uint32_t* counts,
                           uint32_t batch, uint32_t nodes, uint32_t weigh_nodes, double* d_logits);
/* Commits the nodes path[b][0 .. path_lens[b]) of the last mitok_tree_step, a
 * chain from a node without a parent downwards (path [batch][max_path]; 0
 * nodes: none): their rows become the cache's next ones.  A following
 * mitok_decode_step(NULL) feeds the greedy id after the last of them.  Where
 * the runtime fails once rows move (here and in mitok_evict_rows) the caches
 * are dropped. */
int mitok_tree_accept(mitok_network* net, const uint32_t* path, const uint32_t* path_lens, uint32_t batch,
                      uint32_t max_path);

/* Eviction from a cache by accumulated attention weight.  A sequence of more
 * than `keep` rows keeps, in every head, its first `sinks`, its last `recent`
 * (sinks + recent <= keep) and of the others those of largest weight (equal
 * weights, and NaN, which counts as less than any number: the lowest slot
 * first); others keep all.  The kept rows of keys, values and weights go, in
 * order, to slots 0, 1, ... of the output arrays [batch][heads][out_ctx]...;
 * slots behind them stay as they were.  In place: d_k_out == d_k_cache,
 * d_v_out == d_v_cache, d_weights_out == d_weights and out_ctx == max_ctx.
 * d_kept [batch][heads][keep] (keep <= 2^30) or NULL: the slots kept, then MITOK_NO_ROW.
 * out_lens (host) [batch]: rows kept. */
int mitok_evict_rows_device(mitok_network* net, const double* d_k_cache, const double* d_v_cache,
                            const double* d_weights, const uint32_t* kv_lens, uint32_t batch, uint32_t heads,
                            uint32_t head_dim, uint32_t max_ctx, uint32_t keep, uint32_t sinks, uint32_t recent,
                            double* d_k_out, double* d_v_out, double* d_weights_out, uint32_t out_ctx,
                            uint32_t* d_kept, uint32_t* out_lens);
/* The same in place on every attention layer's cache, by the weights that
 * mitok_tree_step(weigh_nodes > 0) kept since the prompt (rows that other
 * calls appended weigh 0; MITOK_ERR_STATE if no step weighed).  Later tokens
 * keep their RoPE positions; a bias column goes by the row's place in the
 * cache.  out_lens [batch] or NULL: rows left.  Drops an uncommitted tree. */
int mitok_evict_rows(mitok_network* net, uint32_t batch, uint32_t keep, uint32_t sinks, uint32_t recent,
                     uint32_t* out_lens);

/* Rules on rows of logits, then the greedy id.  For token t of row r, seen
 * c > 0 times in the row's history: x = x > 0 ? x / repetition : x * repetition,
 * then x -= frequency * c + presence; then x += its bias; a token whose bit
 * is 0 in `allowed` becomes -inf (whatever it was).
 *   d_history [rows][max_history], d_penalties [rows][3] (repetition > 0,
 *     presence, frequency); max_history 0: neither is read
 *   d_bias_ids, d_bias [rows][max_bias]: of equal ids the last entry counts
 *   d_allowed [rows][(vocab + 31) / 32] bits (t at bit t % 32 of word t / 32) or NULL
 *   each size at most 2^30
 * MITOK_NO_TOKEN entries of the history and the ids are skipped; another id
 * >= vocab is MITOK_ERR_ARG.  d_out [rows][vocab] or NULL: the logits after
 * the rules (d_logits itself: in place).  d_out_ids [rows] or NULL: the last
 * index of the largest one, MITOK_NO_TOKEN if none is above -inf.  A NaN that
 * is allowed is MITOK_ERR_NAN, as in greedy_decoding (sampling_methods.rs:5-18).
 * On an error the outputs have no meaning; logits in place are as they were
 * where ids or penalties are refused, and changed on MITOK_ERR_NAN. */
int mitok_process_logits_device(mitok_network* net, const double* d_logits, uint32_t rows, uint32_t vocab,
                                const uint32_t* d_history, uint32_t max_history, const double* d_penalties,
                                const uint32_t* d_bias_ids, const double* d_bias, uint32_t max_bias,
                                const uint32_t* d_allowed, double* d_out, uint32_t* d_out_ids);
/* The same on host arrays. */
int mitok_process_logits(mitok_network* net, const double* logits, uint32_t rows, uint32_t vocab,
                         const uint32_t* history, uint32_t max_history, const double* penalties,
                         const uint32_t* bias_ids, const double* bias, uint32_t max_bias, const uint32_t* allowed,
                         double* out, uint32_t* out_ids);

/* ---- beams on a paged cache (no reference counterpart) ----
 * Several hypotheses per prompt, which share the cached rows that they have in
 * common.  A cache of pages holds a sequence's slot t in row t % page_rows of page
 * table[sequence][t / page_rows]; a pool has [pages][heads][page_rows][head_dim]
 * complex keys, and as many values.  page_rows: a multiple of 16 up to 1024;
 * head_dim <= 256; pages <= 2^24, each of at most 2^30 complex keys; at most
 * 65535 sequences, sequences * max_pages <= 2^28, max_pages * page_rows <= 2^30.
 * Streams, checks and completion are those of the operators above. */

/* Attention of a chunk of new tokens: sequence b holds kv_lens[b] rows, and its
 * counts[b] <= rows new ones (counts NULL: rows of each; rows <= 65536) are stored
 * behind them and attend, new row i over the slots up to its own:
 *   score(i, t) = Re(sum_e q_i[e] k_t[e]) / (1e-8 + sqrt(head_dim)) + bias[h][t],  t <= kv_lens[b] + i
 *   out_i = sum_t softmax(score(i, .))_t v_t
 * With bias_row_stride > 0 a head's biases are a table of rows so far apart, of
 * which new row i takes row kv_lens[b] + i: a prompt's pass, in one chunk or
 * several (masked_attention_head.rs:184-208); 0 is a decode step's.  Slots that a
 * row does not see have no part in its output, finite or not; rows past
 * counts[b] are zero.
 *   d_q, d_k_new, d_v_new, d_out [batch][rows][heads * head_dim] complex
 *   d_table [batch][max_pages]: entries of the slots in use, the new rows' too;
 *     entries behind them are not read
 *   d_bias [heads] of bias_stride apart, or NULL
 * batch * heads <= 2^18, and at most 2^20 groups of 16 new rows (counted from `rows`)
 * and 2^23 blocks of work, of up to 64 rows of a head each: MITOK_ERR_ARG.
 * An entry in use that is >= pages is MITOK_ERR_ARG, and so are two pages of a call
 * that store new rows to one page of the pool.  A page that is stored to may be
 * in no other sequence's use (mitok_fork_pages_device sees to that): the rows read
 * of it would depend on the order.  On an error the outputs have no meaning. */
int mitok_paged_attention_device(mitok_network* net, const double* d_q, const double* d_k_new, const double* d_v_new,
                                 double* d_k_pages, double* d_v_pages, const uint32_t* d_table, const double* d_bias,
                                 uint64_t bias_stride, uint64_t bias_row_stride, const uint32_t* kv_lens,
                                 const uint32_t* counts, uint32_t batch, uint32_t rows, uint32_t heads,
                                 uint32_t head_dim, uint32_t page_rows, uint32_t max_pages, uint32_t pages,
                                 double* d_out);
/* Sequences that take other sequences' rows.  New sequence i (of new_sequences)
 * has the rows of d_parents[i] (MITOK_NO_PARENT: none) and room for d_grow[i] more
 * (d_grow NULL or no parent: 0).  Rows are shared by sharing pages; a page that is
 * part filled, last of a sequence that grows, and held by another new sequence
 * too, is copied (its used rows, in every layer), except for the first of its
 * holders where all of them grow from it.  Pages that no new sequence holds are
 * free; copies and room take them in ascending order, sequence by sequence, a
 * copy before the room.
 *   d_k_pages, d_v_pages: `layers` <= 16384 pools one behind the other, of one table
 *   d_table [sequences][max_pages], d_lens [sequences] rows
 *   d_table_out [new_sequences][max_pages]: MITOK_NO_PAGE behind a sequence's last
 *     page; d_lens_out [new_sequences]: its rows, without the room
 * d_table_out may be d_table and d_lens_out d_lens.  MITOK_ERR_ARG: a parent or a
 * page that is none, rows and room past max_pages; MITOK_ERR_NOMEM: fewer free pages
 * than needed.  Either leaves every array as it was. */
int mitok_fork_pages_device(mitok_network* net, double* d_k_pages, double* d_v_pages, uint32_t layers, uint32_t pages,
                            uint32_t heads, uint32_t page_rows, uint32_t head_dim, const uint32_t* d_table,
                            const uint32_t* d_lens, uint32_t sequences, uint32_t max_pages, const uint32_t* d_parents,
                            const uint32_t* d_grow, uint32_t new_sequences, uint32_t* d_table_out,
                            uint32_t* d_lens_out);
/* The best continuations of each group of beams (batch groups of `beams` <= 1024
 * rows): of all (row r, token t) the `keep` <= MITOK_BEAM_MAX_KEEP of largest rank,
 *   score(r, t) = scores[r] + logits[r][t] - log sum_u exp(logits[r][u])
 *   rank(r, t) = score(r, t) * scale[r]
 * the best first; in a row the larger logit is first, of equal ones the lower
 * token, between rows of equal rank the lower row.  A row with done[r] != 0 has
 * one continuation, itself (score scores[r], no token); one of score -inf has
 * none, and a logit of -inf is none (nor is one whose score or rank passes the
 * doubles to -inf; finite masks down to the lowest double are logits like others).
 * The logits of both kinds of row are not read.
 * At most 2^30 logits of a group, 2^23 rows and 2^23 pieces of 1024 logits in all.
 *   d_logits [batch * beams][vocab], d_scores, d_scale [batch * beams] (scale NULL: 1;
 *     else finite and above 0), d_done [batch * beams] or NULL
 *   d_parents [batch][keep]: the row, counted over all groups, d_tokens,
 *     d_scores_out; where there are no more continuations MITOK_NO_ROW,
 *     MITOK_NO_TOKEN and -inf (the row alone: an ended one's own)
 * A score or a live row's logit that is NaN or +infinity is MITOK_ERR_NAN.  On an error
 * the outputs have no meaning. */
int mitok_beam_select_device(mitok_network* net, const double* d_logits, const double* d_scores, const uint32_t* d_done,
                             const double* d_scale, uint32_t batch, uint32_t beams, uint32_t vocab, uint32_t keep,
                             uint32_t* d_parents, uint32_t* d_tokens, double* d_scores_out);
/* The same on host arrays. */
int mitok_beam_select(mitok_network* net, const double* logits, const double* scores, const uint32_t* done,
                      const double* scale, uint32_t batch, uint32_t beams, uint32_t vocab, uint32_t keep,
                      uint32_t* parents, uint32_t* tokens, double* scores_out);
/* predict_token_by_token's loop with `beams` <= MITOK_BEAM_MAX_KEEP hypotheses per
 * prompt (transformer_network.rs:165-313 keeps one): up to n_new tokens each, one
 * that chooses end_id ends there (MITOK_NO_TOKEN: none does).  A hypothesis is ranked
 * by its score, the sum of its tokens' log probabilities, over its number of
 * tokens to the power length_power (0: by the score; within [-16, 16]).  The prompt
 * runs once and its rows are shared; one beam without an end gives
 * mitok_generate's ids.  Drops the caches, as mitok_generate does, and leaves none.
 * At most 65535 hypotheses, hypotheses * heads <= 2^18, 2^26 tokens of all of them.
 *   prompt [batch][seq], lens [batch] as for mitok_generate
 *   out_ids [batch][beams][n_new], the best hypothesis first, MITOK_NO_TOKEN behind its
 *     tokens; out_lens [batch][beams] tokens (the end among them);
 *     out_scores [batch][beams], -inf where there are fewer hypotheses than beams */
int mitok_beam_search(mitok_network* net, const uint32_t* prompt, const uint32_t* lens, uint32_t batch, uint32_t seq,
                      uint32_t beams, uint32_t n_new, uint32_t end_id, double length_power, uint32_t* out_ids,
                      uint32_t* out_lens, double* out_scores);

/* ---- measurement (no reference counterpart: the reference prints wall
 * clock only, transformer_network.rs:307-310) ---- */
/* Wall time of the last mitok_generate on the device stream, in ms:
 * t[0] prefill (prompt forward + first id), t[1] all decode steps, t[2] how
 * the decode steps ran: 0 direct launches, 1 a replayed HIP graph, 2 the
 * resident loop. */
int mitok_last_timings(mitok_network* net, double* t3);
/* HIP-event timing of one kernel class during the following calls (0 disables;
 * decode steps then run without graph replay so each launch is bracketed). */
int mitok_timing_enable(mitok_network* net, int kernel_class);
/* Accumulated since enable: total ms, launches, and the algorithmic HBM bytes
 * and real flops of those launches (any pointer may be NULL). */
int mitok_timing_read(mitok_network* net, double* total_ms, uint64_t* launches, double* alg_bytes, double* alg_flops);
/* hipDeviceSynchronize on `device` (bench brackets its timed region with it). */
int mitok_device_synchronize(int device);
/* 0 = replay decode steps as HIP graphs (default), 1 = launch kernels directly. */
int mitok_set_graph_mode(mitok_network* net, int direct_launch);
/* 3 = generate's decode loop for up to 8 sequences runs as one resident
 *     cooperative launch (one block per CU; how its blocks exchange values:
 *     mitok_resident_exchange);
 * 2 = the resident loop for 1 and 2 sequences (1 if the polling exchange is
 *     off or a RoPE layer rules it out), plan 1 above (default);
 * 1 = decode steps of up to 64 sequences run the fused plan (up to 8: GEMV
 *     products with the row transforms in their prologues; 9 to 64: skinny
 *     MFMA products after a row-transform launch), replayed as a graph;
 * 0 = one launch per reference operation and one query row per attention block.
 * Plans 1 to 3 run prefill attention on the tiled kernel.
 * No counterpart in the reference (a scheduling choice; results agree to the
 * parity tolerance). */
int mitok_set_decode_plan(mitok_network* net, int plan);
/* Whether a stateless predict keeps each FeedForward's and attention layer's
 * forward products (16 bytes of a row times 2 hidden, or 3 width) for
 * backward.  1 (default): yes, where the device has room; they give way to any
 * other allocation of the network, and a pass that needs as much as once had
 * to give way keeps none (this call forgets that).  0: backward forms them
 * again.  No counterpart in the reference; the results are the same bits. */
int mitok_set_product_saving(mitok_network* net, int keep);
/* Per-operation profile of the resident decode loop (plan 2).  enable = 1:
 * later launches record block 0's clock after every grid barrier.  Then, if
 * nops is not NULL, reports the last launch's operations (at most max_ops):
 * kinds[i] (0 product, 1 attention chunks with their combine, 2 row transform) and
 * us[i], the microseconds from the previous barrier to the one after op i,
 * averaged over the steps.  No counterpart in the reference (instrumentation). */
int mitok_resident_profile(mitok_network* net, int enable, int max_ops, int* nops, int* kinds, double* us);
/* How the blocks of the resident decode loop hand values to each other.
 * mode 1 (default): polling -- every exchanged value starts a step as a
 * sentinel and its reader re-reads it until written, one grid barrier per
 * step -- where the program allows it (no RoPE); mode 0: a grid barrier
 * after every operation.  mode -1 leaves it unchanged.  *polled (if not
 * NULL): whether the last resident launch polled.  No counterpart in the
 * reference (a scheduling choice; the arithmetic is the same either way). */
int mitok_resident_exchange(mitok_network* net, int mode, int* polled);

#ifdef __cplusplus
}
#endif
#endif
