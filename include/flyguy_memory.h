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

#ifdef __cplusplus
}
#endif
#endif
