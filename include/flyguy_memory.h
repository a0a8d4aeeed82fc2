/* The memory over decisions of the flyguy MI355X library (libflyguy_core.so): rotary positions, per-head norms with the
 * rotation in the same pass, and linear attention with a decay for each head, over whole stretches of moments and one
 * moment at a time.  An addition of this library: the reference remembers nothing from one decision to the next.
 *
 * Every call takes one argument structure, returns 0, or -1 with the reason in fc_last_error(); nothing is launched then.
 * Pointers are device memory of the current device unless marked (host).  Work goes to `stream` (a hipStream_t); no call
 * synchronises, allocates or keeps anything.  Values: FM_F32 float32, FM_BF16 bfloat16, FM_F16 binary16; sums, norms and
 * states are float32 whatever the values' type.
 */
#ifndef FLYGUY_MEMORY_H
#define FLYGUY_MEMORY_H

#ifdef __cplusplus
extern "C" {
#endif

#define FM_F32 0
#define FM_BF16 1
#define FM_F16 2

/* Heads of a stretch: value d of head h of moment t of stretch n at data + n seq + t moment + h head + d (strides in
 * values, not bytes). */
typedef struct fm_view {
    void* data;
    long long seq, moment, head;
} fm_view;

/* Queries (x[0]) and keys (x[1]; heads[1] 0: none), n_seq stretches of n_moments moments, dim <= 512 values per head.
 *   r = (mean(x^2) + eps)^-1/2;  z = x r weight[d]       (weight 0: z = x)
 *   the pairs (a, b) of the first `rotated` values, (i, i + rotated/2), or (2i, 2i+1) if interleaved, turned:
 *   y_a = z_a cos - z_b sin,  y_b = z_b cos + z_a sin,   (cos, sin) = table[position][i]
 * table: float32 [n_positions][rotated/2][2] (rotated 0: no rotation).  A moment's position is positions[n pos_seq + t
 * pos_moment] (int32, or int64 if wide) + first; positions 0: t + first.  A position outside the table gives NaN in the
 * rotated values.  At most 8e9 heads of moments.  Gradients (fm_turn_bwd): x the forward's inputs (read only where weight
 * is not 0), g the gradients of y, y the gradients of x, written; gweight: the weights' gradients, written; partial:
 * fm_turn_partial() floats.  y may be x itself (gradients: x or g), with the same strides; otherwise what is written must
 * lie outside what is read. */
typedef struct fm_turn_args {
    fm_view x[2], y[2], g[2];
    const float* weight[2];
    float* gweight[2];
    float* partial;
    const float* table;
    const void* positions;
    long long pos_seq, pos_moment, first, wide;
    long long heads[2], n_seq, n_moments, dim, rotated, interleaved, n_positions, dtype;
    double eps;
} fm_turn_args;
int fm_turn(const fm_turn_args* a, void* stream);
int fm_turn_bwd(const fm_turn_args* a, void* stream);
long long fm_turn_partial(const fm_turn_args* a);

/* Linear attention with a decay for each query head, l = exp(log_decay[h]) (log_decay 0 keeps everything, -inf nothing; above 0,
 * at most 1, states grow until they overflow); query head h reads key / value head h / (q_heads / k_heads):
 *   S_t = l S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t,   S_{-1} = state (0: zeros)
 * k_dim, v_dim <= 128, q_heads <= 65535, n_seq <= 16384, n_moments <= 2^31.  A value that is not finite reaches no output of an
 * earlier moment (no gradient of a later one), and no other stretch; the outputs and states that it does reach are NaN, or
 * infinite.
 * Stretches: n_seq of n_moments moments each, or (starts not 0) packed: n_moments in all, stretch n being moments starts[n] ..
 * starts[n+1] - 1 (int32, or int64 if wide; out of [0, n_moments]: brought into it), the views' seq unread.  Where starts fall,
 * stretches are cut short so that no two share a moment.  o: dense [moments][q_heads][v_dim], zeros at moments of no stretch.
 * state, state_out: float32 [n_seq][q_heads][k_dim][v_dim] (state_out 0: not wanted; it must not overlap state).  A stretch
 * without moments passes its state on as it is.
 * Gradients (fm_attention_bwd): go of o, gstate_out of state_out (0: zeros); gq, gk, gv dense like their tensors, gstate
 * float32; each 0 where not wanted.  workspace: fm_attention_workspace(a, backward) bytes. */
typedef struct fm_attention_args {
    fm_view q, k, v, go;
    const float* log_decay;
    const float* state;
    const void* starts;
    void* o;
    float* state_out;
    const float* gstate_out;
    void *gq, *gk, *gv;
    float* gstate;
    void* workspace;
    long long workspace_bytes;
    long long wide, n_seq, n_moments, q_heads, k_heads, k_dim, v_dim, dtype;
    double scale;
} fm_attention_args;
int fm_attention(const fm_attention_args* a, void* stream);
int fm_attention_bwd(const fm_attention_args* a, void* stream);
long long fm_attention_workspace(const fm_attention_args* a, int backward);

/* One moment of it for n <= 65535 rows: q, k, v (views without moments) and
 *   next[s] = l state[s] + k v^T,  o = scale q next[s]     (o: dense [n][q_heads][v_dim])
 * s = slots[row] (int32; 0: s = row), state and next float32 [n_states][q_heads][k_dim][v_dim] (next == state: in place;
 * else outside it).  A slot below 0 gives a row of zeros and touches no state; one past the states gives NaN and touches none.
 * No two rows may name the same slot. */
typedef struct fm_step_args {
    fm_view q, k, v;
    const float* log_decay;
    const float* state;
    float* next;
    const int* slots;
    void* o;
    long long n, n_states, q_heads, k_heads, k_dim, v_dim, dtype;
    double scale;
} fm_step_args;
int fm_step(const fm_step_args* a, void* stream);

/* The gated delta rule: a memory that moves what it holds under a key towards the key's new value.  Each query head has a state,
 * and each moment a decay a = exp(log_decay) (0 keeps everything, -inf forgets everything, above 0, at most 1, states grow) and a
 * rate beta of its own; query head h reads key / value head h / (q_heads / k_heads):
 *   e_t = v_t - (a_t S_{t-1})^T k_t,   S_t = a_t S_{t-1} + beta_t k_t e_t^T,   o_t = scale S_t^T q_t,   S_{-1} = state (0: zeros)
 * Meant for keys with beta |k|^2 <= 2 (beyond, a state may grow from moment to moment).  Sizes, stretches, packed stretches, o,
 * state and state_out as for fm_attention; also at most 8e9 heads of moments.  log_decay, beta: float32, strides in values.
 * A query that is not finite reaches its own output only.  A value of v that is not finite makes its column of outputs and of
 * the state NaN from its moment on; a key, decay (NaN or +inf) or rate that is not, all of the head's; no earlier moment, other
 * head or stretch (gradients: no other head or stretch).
 * saved: fm_delta_saved(a) bytes that the gradient reads (0: no gradient is wanted), workspace: fm_delta_workspace(a, backward)
 * bytes: by sizes alone where the tensors read (backward: q, k, go) have values, strides and starts of multiples of 16 bytes and
 * strides of moments from 0 to 2^22 - 1 values, or are dense; others are copied, and the room for that is counted by the views given.  Gradients (fm_delta_bwd): inputs and saved as the forward left them; go of o, gstate_out of state_out (0: zeros); gq, gk,
 * gv dense like their tensors, glog_decay, gbeta float32 [moments][q_heads], gstate float32; each 0 where not wanted.  glog_decay
 * is what is left of sums that cancel where little was remembered: off by the float32 roundings of their terms. */
typedef struct fm_delta_args {
    fm_view q, k, v, go;
    const float *log_decay, *beta;
    long long ld_seq, ld_moment, ld_head, be_seq, be_moment, be_head;
    const float* state;
    const void* starts;
    void* o;
    float* state_out;
    void* saved;
    long long saved_bytes;
    const float* gstate_out;
    void *gq, *gk, *gv;
    float *glog_decay, *gbeta, *gstate;
    void* workspace;
    long long workspace_bytes;
    long long wide, n_seq, n_moments, q_heads, k_heads, k_dim, v_dim, dtype;
    double scale;
} fm_delta_args;
int fm_delta(const fm_delta_args* a, void* stream);
int fm_delta_bwd(const fm_delta_args* a, void* stream);
long long fm_delta_workspace(const fm_delta_args* a, int backward);
long long fm_delta_saved(const fm_delta_args* a);

/* One moment of it for n <= 65535 rows, as fm_step: log_decay and beta of row i and head h at i row + h head.  What is not finite
 * reaches what it reaches there; an update that overflows float32 is NaN. */
typedef struct fm_delta_step_args {
    fm_view q, k, v;
    const float *log_decay, *beta;
    long long ld_row, ld_head, be_row, be_head;
    const float* state;
    float* next;
    const int* slots;
    void* o;
    long long n, n_states, q_heads, k_heads, k_dim, v_dim, dtype;
    double scale;
} fm_delta_step_args;
int fm_delta_step(const fm_delta_step_args* a, void* stream);

/* Layer norm of rows of `width` values (1 to 2^24), row i at x + i x_row (strides in values):
 *   m = mean(x), r = (mean((x - m)^2) + eps)^-1/2, xh = (x - m) r, y = xh weight + bias   (weight 0: 1; bias 0: 0)
 * (sums in float32: r is 0 where the squares pass its largest number).  stats: float32 [rows][2], (m, r) of each row, written if not 0.  Gradients (fm_norm_bwd): x, weight and stats the forward's,
 * g the gradient of y; gx, gweight, gbias the gradients, each 0 where not wanted; partial: fm_norm_partial() floats.  weight,
 * bias and their gradients are float32.  y may be x, gx may be x or g, with the same stride, where rows do not overlap; otherwise what is
 * written must lie outside what is read. */
typedef struct fm_norm_args {
    const void* x;
    void* y;
    const void* g;
    void* gx;
    long long x_row, y_row, g_row, gx_row;
    const float *weight, *bias;
    float *gweight, *gbias, *stats, *partial;
    long long rows, width, dtype;
    double eps;
} fm_norm_args;
int fm_norm(const fm_norm_args* a, void* stream);
int fm_norm_bwd(const fm_norm_args* a, void* stream);
long long fm_norm_partial(const fm_norm_args* a);

/* Dropout without a stored mask: number i = row width + column of rows x width (at most 1e12) becomes 0 where its draw is below
 * t = round(65536 share), else 65536 / (65536 - t) times itself; share 1: all zeros.  Draws: Philox4x32 of 10 rounds, key = counter[0]
 * (low word first), counter = (i / 8, counter[1]); draw i is half i % 8 of its four words, low halves first.  counter: device
 * memory, read when the kernel runs.  y: dense.  The same call on y's gradient gives x's.  y may be x where x is dense. */
typedef struct fm_drop_args {
    const void* x;
    void* y;
    const unsigned long long* counter;
    long long x_row, rows, width, dtype;
    double share;
} fm_drop_args;
int fm_drop(const fm_drop_args* a, void* stream);

#ifdef __cplusplus
}
#endif
#endif
