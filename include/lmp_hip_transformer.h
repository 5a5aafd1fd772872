/*
 * lmp_hip_transformer.h -- C ABI of the transformer-training operators of
 * liblmp_hip.so: layer normalisation, the AdamW step, packed attention, rotary
 * positions, dropout, gated linear layers and cross entropy over a vocabulary.
 *
 * The reference has none of these; they follow the conventions of lmp_hip.h:
 * every entry point returns an lmp_status and leaves its message in
 * lmp_rt_last_error(), device pointers are HIP device allocations of the
 * current device, all work goes in order to lmp_rt_stream() without
 * synchronising, and scratch memory comes from the library's pool, so calls may
 * be recorded between lmp_rt_graph_begin and lmp_rt_graph_end.  Arguments are
 * checked before anything is written.  Leading dimensions (ld*, *_ld) are in
 * elements.  Sums are formed in a fixed order: equal calls give equal bits.
 */
#ifndef LMP_HIP_TRANSFORMER_H_
#define LMP_HIP_TRANSFORMER_H_

#include "lmp_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------- layer norm */

/* y = (x - mean) * rstd * w + b over each row's `cols` values, with mean and
 * rstd = 1 / sqrt(var + eps) (var biased, formed from the differences to the
 * mean) written per row.  dtype is LMP_FLOAT32 or LMP_FLOAT64 for every buffer;
 * statistics are held in that type.  w and b (cols values) may be null, for 1
 * and 0; mean and rstd (rows values) may be null where no backward pass
 * follows.  y may be x.  cols must be positive. */
int lmp_k_layer_norm(int dtype, size_t rows, size_t cols, const void* x, size_t ldx, const void* w,
                     const void* b, double eps, void* y, size_t ldy, void* mean, void* rstd);

/* The gradients of lmp_k_layer_norm from its output gradient g and the mean and
 * rstd it wrote: with z = (x - mean) * rstd and u = g * w,
 *   dx = rstd * (u - avg(u) - z * avg(u z)),  dw = sum_rows g z,  db = sum_rows g.
 * w may be null (1); each of dx, dw and db may be null where it is not wanted.
 * dx may be g or x. */
int lmp_k_layer_norm_backward(int dtype, size_t rows, size_t cols, const void* g, size_t ldg,
                              const void* x, size_t ldx, const void* w, const void* mean,
                              const void* rstd, void* dx, size_t lddx, void* dw, void* db);

/* ------------------------------------------------------------------ AdamW */

#define LMP_ADAMW_BLOCK 256 /* values that share one scale of an 8-bit state */

/* One tensor of an AdamW step: n float32 parameters p and gradients g.  With
 * states of 32 bits m and v are n floats and the scales are null; with states
 * of 8 bits m is n int8 codes, v n uint8 codes, and the scales are
 * ceil(n / LMP_ADAMW_BLOCK) floats each. */
typedef struct {
  float* p;
  const float* g;
  void* m;
  void* v;
  float* m_scale;
  float* v_scale;
  uint64_t n;
  double decay;
} lmp_adamw_tensor;

/* One step over `count` tensors (a host array, read before the call returns):
 *   m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g g,
 *   p = p (1 - lr decay) - lr m^ / (sqrt(v^) + eps),
 * m^ = m / (1 - beta1^t) and v^ = v / (1 - beta2^t).  `step` is two int64 on the
 * device: step[0] the steps done so far (t = step[0] + 1; the call adds one),
 * step[1] the library's, 0 before the first call.  Keeping the count on the
 * device lets a recorded step be replayed.  State bits are 32 or 8.  The buffers that
 * a step writes (p, m, v and the scales of every tensor) do not overlap each other.
 * 8 bits: per block of values of one tensor, the largest magnitude M as a
 * float and per value a code c for sign(c) (|c| / Q)^2 M, Q = 127 for m and 255
 * for v, rounded up or down at random with the value as its expectation; a v
 * above zero never becomes zero.  M below 1e-30 is stored as 0, an infinite or
 * NaN M as NaN.  The 16 random bits of each code come from MurmurHash3's 32-bit
 * finalizer over (seed, t, the tensor's place in the list, the value's place):
 * the low half for m, the high half for v.  Equal calls give equal codes.  With states
 * of 8 bits the parameter's root and quotient are formed to a unit in their last places
 * (correctly rounded with states of 32, and where eps is below 2^-39 / sqrt(1 - beta2)). */
int lmp_k_adamw_f32(int bits, size_t count, const lmp_adamw_tensor* tensors, double lr,
                    double beta1, double beta2, double eps, uint64_t seed, int64_t* step);

/* The n values of 8-bit codes: signed_codes != 0 for m's int8, 0 for v's. */
int lmp_k_adamw_decode(int signed_codes, const void* codes, const float* scales, size_t n,
                       float* out);

/* -------------------------------------------------------------- attention */

/* A packed batch: `sequences` pairs of lengths (host arrays, each length may be
 * 0), their queries one after another in the rows of q and o, their keys in the
 * rows of k and v.  Row i holds `heads` (q, o) or `kv_heads` (k, v) vectors of
 * head_dim values one after another; heads is a multiple of kv_heads, and head
 * h reads key head h / (heads / kv_heads).  causal != 0: query i of a sequence
 * with Lq queries and Lk keys sees keys 0 .. i + Lk - Lq, so the last query
 * sees every key.  head_dim is at most LMP_ATTENTION_MAX_DIM.
 * The plan holds the batch's work lists on the device; making one copies them
 * there and waits, so it fails during a graph capture.  It is read by the calls
 * that use it and must outlive them and any graph that records them. */
#define LMP_ATTENTION_MAX_DIM 256
int lmp_k_attention_plan_create(void** plan, size_t sequences, const int64_t* q_lengths,
                                const int64_t* k_lengths, size_t heads, size_t kv_heads,
                                size_t head_dim, int causal);
int lmp_k_attention_plan_destroy(void* plan);

/* o = softmax(scale q k^T + mask) v, and lse [rows of q, heads] the logarithm of
 * each softmax's sum (null where no backward pass follows).  A query that sees
 * no key gives o = 0 and lse = -inf.  What masked places hold, infinities and NaN
 * too, reaches no result.  Outputs do not overlap operands, here and below (dq, dk
 * and dv may be slices of the same rows).
 * Short batches, single tokens and a head_dim above 128 run on the fp32 matrix cores.
 * Long batches run on the fp16 matrix cores with every operand split into two fp16 parts that share a
 * power of two per 32 rows of one head: a product then errs by at most 2^-21 of
 * itself (2^-23.5 rms) and by 2^-40 of the largest one among its 32 rows.  Softmax
 * weights, and gradients of scores, are split against the largest that their query (for
 * dk and dv their key) has met so far, each times its tile's power of two and faded as
 * the softmax goes on: what they multiply errs by 2^-37 of the largest such product.
 * Rows that lie further apart than 2^12, infinities, NaN and largest values outside
 * [2^-60, 2^41) send their sequence's key head, the whole of it, to the fp32 kernels:
 * one such row of g makes the backward pass of 2048 positions, 16 heads of 128 on 4, five
 * times as long (325 us and 1.7 ms), of 8192 seven times. */
int lmp_k_attention_f32(const void* plan, const float* q, size_t q_ld, const float* k, size_t k_ld,
                        const float* v, size_t v_ld, double scale, float* o, size_t o_ld,
                        float* lse);

/* dq, dk and dv from the output gradient g and the o and lse of
 * lmp_k_attention_f32; all three are written.  The weights are formed again from lse, so
 * that besides the errors above each is off by about |lse| 2^-23 of itself: 1e-5 where
 * scores are some 100, and no digit is left where they pass 2^23. */
int lmp_k_attention_backward_f32(const void* plan, const float* q, size_t q_ld, const float* k,
                                 size_t k_ld, const float* v, size_t v_ld, double scale,
                                 const float* o, size_t o_ld, const float* lse, const float* g,
                                 size_t g_ld, float* dq, size_t dq_ld, float* dk, size_t dk_ld,
                                 float* dv, size_t dv_ld);

/* ------------------------------------------------------- rotary positions */

/* y = x with the pairs of its first `heads` vectors of each row turned by the row's
 * position.  A row has `cols` values: the vectors of head_dim values one after another,
 * then what is copied as it is (the values of a projection to queries, keys and values).
 * Of each vector the first rotary_dim values (even, head_dim at most) turn and the others
 * are copied: pair j, at values (j, j + rotary_dim / 2) or with interleaved != 0 at
 * (2 j, 2 j + 1), becomes
 *   scale (u cos a - v sin a, v cos a + u sin a),  a = positions[row] * frequencies[j],
 * with inverse != 0 by -a: the gradient of the same call.  dtype is LMP_FLOAT32 or
 * LMP_FLOAT64 for x and y; positions (int64) and frequencies (float64, rotary_dim / 2
 * radians per position) are on the device.  Angles are formed in 64 bits: for float32 a
 * turned value errs by 2^-20 of its pair's larger one, and besides by |a| 2^-51 of both.
 * y may be x with the same leading dimension, or rows beside x's; another overlap is
 * refused. */
int lmp_k_rotary(int dtype, size_t rows, size_t cols, size_t heads, size_t head_dim,
                 size_t rotary_dim, int interleaved, const void* x, size_t ldx,
                 const int64_t* positions, const double* frequencies, double scale, int inverse,
                 void* y, size_t ldy);

/* ---------------------------------------------------------------- dropout */

/* y = residual + (kept ? x / (1 - rate) : 0) over n contiguous values (residual null: 0),
 * rate in [0, 1].  What is kept comes from Philox4x32-10 with the seed's halves as its key
 * and (place / 4, number of the call), low halves first, as its counter: value i takes word
 * i % 4 and is kept if that is at least rate * 2^32 (rounded).  `state` is two int64 on the
 * device: state[0] the number of this call, which the call advances by one, state[1] the
 * library's, 0 before the first call.  Keeping it on the device lets a recorded call draw
 * afresh at every replay.  `used` (one int64 on the device, or null where no backward pass
 * follows) takes the number of this call.  What is dropped, infinities and NaN too, leaves
 * no trace.  y may be x or residual; another overlap is refused. */
int lmp_k_dropout(int dtype, size_t n, const void* x, const void* residual, double rate,
                  uint64_t seed, int64_t* state, int64_t* used, void* y);

/* dx = kept ? g / (1 - rate) : 0 by what the call numbered *used kept (the residual's
 * gradient is g).  dx may be g; another overlap is refused. */
int lmp_k_dropout_backward(int dtype, size_t n, const void* g, double rate, uint64_t seed,
                           const int64_t* used, void* dx);

/* ----------------------------------------------------------- gated linear */

typedef enum {
  LMP_GATE_SILU = 0,      /* a / (1 + e^-a) */
  LMP_GATE_GELU = 1,      /* a Phi(a), Phi the normal distribution's */
  LMP_GATE_GELU_TANH = 2, /* a / 2 (1 + tanh(sqrt(2 / pi) (a + 0.044715 a^3))) */
  LMP_GATE_RELU = 3,      /* max(a, 0); its slope at 0 is 0 */
  LMP_GATE_SIGMOID = 4,   /* 1 / (1 + e^-a) */
  LMP_GATE_COUNT = 5
} lmp_gate;

/* h = act(a) u for [a | u] = x w + bias: x [rows, in], w [in, 2 hidden] whose first
 * `hidden` columns are the gate's, bias 2 hidden values or null (0), h [rows, hidden].
 * pre [rows, 2 hidden] takes [a | u] for the backward pass (null where none follows).
 * in and hidden are positive.  Outputs do not overlap operands, here and below.
 *
 * Here and below a sum of k products errs by (4 k + 64) 2^-24 of their magnitudes' sum at
 * most, and what is not finite comes out as float32's products give it, also where a size's
 * products run on operands in two fp16 parts: sums that those do not hold well enough are
 * formed again in float32, a few at no cost, whole tiles of them four to eight times slower. */
int lmp_k_gated_linear_f32(int gate, size_t rows, size_t in, size_t hidden, const float* x,
                           size_t ldx, const float* w, size_t ldw, const float* bias, float* h,
                           size_t ldh, float* pre, size_t ldpre);

/* The gradients from the output gradient g [rows, hidden] and the pre that the forward call
 * wrote: with d = [g u act'(a) | g act(a)], dx = d w^T, dw = x^T d and db the column sums
 * of d.  Each of dx, dw and db may be null where it is not wanted (x is read for dw, w for
 * dx). */
int lmp_k_gated_linear_backward_f32(int gate, size_t rows, size_t in, size_t hidden,
                                    const float* g, size_t ldg, const float* x, size_t ldx,
                                    const float* w, size_t ldw, const float* pre, size_t ldpre,
                                    float* dx, size_t lddx, float* dw, size_t lddw, float* db);

/* -------------------------------------- cross entropy over a vocabulary */

/* loss[i] = log sum_v exp(z_iv) - z_i,t of z = x w + bias: x [rows, in], w [in, vocab],
 * bias vocab values or null (0), t = targets[i] (int64, on the device).  A row whose target
 * is negative is not counted: its loss is 0, whatever it holds.  A target of vocab or more
 * makes its row's loss NaN.  A logit of -inf has no share; a row of nothing else has the loss
 * NaN, and so has one with a logit of NaN or +inf.  in and vocab are positive.
 *
 * Workspace: the losses alone of large problems hold a maximum and a sum for 64 logits; other
 * sizes, and the gradients, hold logits.  Either comes in pieces of 512 MB (256 rows, if they
 * are more), 128 MB and less where memory is short, beside the operands' parts (as large as
 * x, w and, with the gradients, a piece's logits twice). */
int lmp_k_linear_cross_entropy_f32(size_t rows, size_t in, size_t vocab, const float* x,
                                   size_t ldx, const float* w, size_t ldw, const float* bias,
                                   const int64_t* targets, float* loss);

/* The losses and, of sum_i weights[i] loss[i] (weights null: 1 each), the gradients dx
 * [rows, in], dw [in, vocab] and db (vocab values), each null where it is not wanted (db
 * only with dw).  A row that is not counted has no part in them, whatever it and its weight
 * hold; its own dx is 0 (times w: NaN where w is infinite). */
int lmp_k_linear_cross_entropy_grad_f32(size_t rows, size_t in, size_t vocab, const float* x,
                                        size_t ldx, const float* w, size_t ldw,
                                        const float* bias, const int64_t* targets,
                                        const float* weights, float* loss, float* dx,
                                        size_t lddx, float* dw, size_t lddw, float* db);

#ifdef __cplusplus
}
#endif

#endif /* LMP_HIP_TRANSFORMER_H_ */
