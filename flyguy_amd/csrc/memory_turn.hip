// Rotary positions and per-head norms of queries and keys (include/flyguy_memory.h: fm_turn, fm_turn_bwd).
#include <hip/hip_runtime.h>

#include "memory.h"

namespace fg {

constexpr int TURN_ROWS = 4;             // rows (waves) per workgroup
constexpr int TURN_MAX = 512;            // values of a head

// The turn of value e of a row: its partner's index, and the factors of y_e = z_e c + z_partner s.
struct Turn {
    int partner;
    float c, s;
};
__device__ __forceinline__ Turn turn_of(int e, const float* cs, int R, bool interleaved) {
    const int half = R >> 1;
    const bool second = interleaved ? (e & 1) : e >= half;
    const int i = interleaved ? e >> 1 : (second ? e - half : e);
    Turn t;
    t.partner = interleaved ? e ^ 1 : (second ? e - half : e + half);
    t.c = cs ? cs[2 * i] : NAN;
    t.s = cs ? (second ? cs[2 * i + 1] : -cs[2 * i + 1]) : NAN;
    return t;
}

// a moment's line of the table (0: its position lies outside)
__device__ __forceinline__ const float* table_line(const fm_turn_args& a, long long n, long long t) {
    const long long p = (a.positions ? index_at(a.positions, n * a.pos_seq + t * a.pos_moment, a.wide) : t) + a.first;
    return p >= 0 && p < a.n_positions ? a.table + p * a.rotated : nullptr;
}

// One wave per row (a head of a moment), lanes over its values; a partner's value is read again (a cache hit).
template <class T, int NE>
__global__ __launch_bounds__(64 * TURN_ROWS) void k_turn(fm_turn_args a) {
    const int H = (int)(a.heads[0] + a.heads[1]), lane = threadIdx.x & 63, D = (int)a.dim, R = (int)a.rotated;
    const long long row = (long long)blockIdx.x * TURN_ROWS + (threadIdx.x >> 6);
    if (row >= a.n_seq * a.n_moments * H) return;
    const long long m = row / H, n = m / a.n_moments, t = m % a.n_moments;
    int h = (int)(row % H);
    const int which = h >= a.heads[0];
    if (which) h -= (int)a.heads[0];
    const fm_view &xv = a.x[which], &yv = a.y[which];
    const T* x = (const T*)xv.data + n * xv.seq + t * xv.moment + h * xv.head;
    T* y = (T*)yv.data + n * yv.seq + t * yv.moment + h * yv.head;
    const float* w = a.weight[which];
    const float* cs = R ? table_line(a, n, t) : nullptr;
    float v[NE], r = 1.f, sum = 0.f;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        const int e = lane + 64 * i;
        v[i] = e < D ? widen(x[e]) : 0.f;
        sum += v[i] * v[i];
    }
    if (w) r = rsqrtf(wave_sum(sum, 64) / D + (float)a.eps);
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        const int e = lane + 64 * i;
        if (e >= D) continue;
        float z = v[i] * r * (w ? w[e] : 1.f);
        if (e < R) {
            const Turn u = turn_of(e, cs, R, a.interleaved);
            z = z * u.c + widen(x[u.partner]) * r * (w ? w[u.partner] : 1.f) * u.s;
        }
        y[e] = narrow<T>(z);
    }
}

// Its gradient: the turn undone (the sine's sign flipped), then, with xh = x r and u = g' w, gx = r (u - xh mean(u xh));
// the weights' gradients sum g' xh over rows: a wave keeps its rows' sums in registers (rows of queries and of keys in
// launches' halves of their own), a workgroup's waves are added in LDS in wave order, k_turn_gweight adds the workgroups.
template <class T, int NE>
__global__ __launch_bounds__(64 * TURN_ROWS) void k_turn_bwd(fm_turn_args a, int blocks) {
    __shared__ float sums[TURN_ROWS][64 * NE];
    const int which = blockIdx.y, H = (int)a.heads[which], lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int D = (int)a.dim, R = (int)a.rotated;
    const fm_view &xv = a.x[which], &yv = a.y[which], &gv = a.g[which];
    const float* w = a.weight[which];
    float gw[NE] = {};
    const long long rows = a.n_seq * a.n_moments * H;
    for (long long row = (long long)blockIdx.x * TURN_ROWS + wave; row < rows; row += (long long)blocks * TURN_ROWS) {
        const long long m = row / H, n = m / a.n_moments, t = m % a.n_moments;
        const int h = (int)(row % H);
        const T* g = (const T*)gv.data + n * gv.seq + t * gv.moment + h * gv.head;
        T* y = (T*)yv.data + n * yv.seq + t * yv.moment + h * yv.head;
        const float* cs = R ? table_line(a, n, t) : nullptr;
        float z[NE];
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const int e = lane + 64 * i;
            z[i] = e < D ? widen(g[e]) : 0.f;
            if (e < R) {
                const Turn u = turn_of(e, cs, R, a.interleaved);
                z[i] = z[i] * u.c - widen(g[u.partner]) * u.s;
            }
        }
        if (w) {
            const T* x = (const T*)xv.data + n * xv.seq + t * xv.moment + h * xv.head;
            float v[NE], sq = 0.f, dot = 0.f;
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const int e = lane + 64 * i;
                v[i] = e < D ? widen(x[e]) : 0.f;
                sq += v[i] * v[i];
            }
            const float r = rsqrtf(wave_sum(sq, 64) / D + (float)a.eps);
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const int e = lane + 64 * i;
                v[i] *= r;
                gw[i] += z[i] * v[i];
                z[i] *= e < D ? w[e] : 0.f;
                dot += z[i] * v[i];
            }
            dot = wave_sum(dot, 64) / D;
#pragma unroll
            for (int i = 0; i < NE; ++i) z[i] = r * (z[i] - v[i] * dot);
        }
#pragma unroll
        for (int i = 0; i < NE; ++i)
            if (lane + 64 * i < D) y[lane + 64 * i] = narrow<T>(z[i]);
    }
    if (!a.gweight[which]) return;
#pragma unroll
    for (int i = 0; i < NE; ++i) sums[wave][lane + 64 * i] = gw[i];
    __syncthreads();
    for (int e = threadIdx.x; e < D; e += 64 * TURN_ROWS) {
        float s = 0.f;
        for (int i = 0; i < TURN_ROWS; ++i) s += sums[i][e];
        a.partial[((size_t)which * blocks + blockIdx.x) * D + e] = s;
    }
}

// gweight[which][e] = the sum of the workgroups' partials, in order: one wave per value, the lanes' strided sums joined
__global__ __launch_bounds__(64) void k_turn_gweight(fm_turn_args a, int blocks) {
    const int which = blockIdx.y, e = blockIdx.x, D = (int)a.dim;
    if (!a.gweight[which]) return;
    float s = 0.f;
    for (int b = threadIdx.x; b < blocks; b += 64) s += a.partial[((size_t)which * blocks + b) * D + e];
    s = wave_sum(s, 64);
    if (threadIdx.x == 0) a.gweight[which][e] = s;
}

inline int turn_blocks(const fm_turn_args& a) {
    const long long rows = a.n_seq * a.n_moments * (a.heads[0] > a.heads[1] ? a.heads[0] : a.heads[1]);
    const long long b = (rows + TURN_ROWS - 1) / TURN_ROWS;
    return (int)(b < 1 ? 1 : b > 2048 ? 2048 : b);
}

const char* turn_args_wrong(const fm_turn_args& a, bool bwd) {
    if (a.dtype < FM_F32 || a.dtype > FM_F16) return "values of an unknown type";
    if (a.n_seq < 0 || a.n_moments < 0 || a.heads[0] < 0 || a.heads[1] < 0) return "a negative size";
    if (a.n_seq > 1LL << 40 || a.n_moments > 1LL << 40 || a.heads[0] > 1 << 20 || a.heads[1] > 1 << 20 ||
        (double)a.n_seq * (double)a.n_moments * (double)(a.heads[0] + a.heads[1]) > 8e9)
        return "more than 8e9 rows";
    if (a.dim < 1 || a.dim > TURN_MAX) return "heads of other than 1 to 512 values";
    if (a.rotated < 0 || a.rotated > a.dim || a.rotated % 2) return "rotated must be even and at most the head's values";
    if (a.rotated && (!a.table || a.n_positions < 0)) return "no table";
    for (int i = 0; i < 2; ++i) {
        if (!a.heads[i]) continue;
        const bool any = a.n_seq && a.n_moments;
        if (any && (!a.y[i].data || (bwd ? !a.g[i].data || (a.weight[i] && !a.x[i].data) : !a.x[i].data)))
            return "a null tensor";
        if (bwd && a.gweight[i] && (!a.weight[i] || !a.partial)) return "a weight's gradient without weight or partial";
    }
    return nullptr;
}

template <class T, int NE>
void launch_turn(const fm_turn_args& a, bool bwd, hipStream_t st) {
    if (bwd) {
        const int blocks = turn_blocks(a);
        k_turn_bwd<T, NE><<<dim3(blocks, a.heads[1] ? 2 : 1), 64 * TURN_ROWS, 0, st>>>(a, blocks);
        if (a.gweight[0] || a.gweight[1])
            k_turn_gweight<<<dim3((unsigned)a.dim, 2), 64, 0, st>>>(a, blocks);
        return;
    }
    const long long rows = a.n_seq * a.n_moments * (a.heads[0] + a.heads[1]);
    if (rows) k_turn<T, NE><<<(unsigned)((rows + TURN_ROWS - 1) / TURN_ROWS), 64 * TURN_ROWS, 0, st>>>(a);
}

template <class T>
void turn_of_type(const fm_turn_args& a, bool bwd, hipStream_t st) {
    if (a.dim <= 64) launch_turn<T, 1>(a, bwd, st);
    else if (a.dim <= 128) launch_turn<T, 2>(a, bwd, st);
    else if (a.dim <= 256) launch_turn<T, 4>(a, bwd, st);
    else launch_turn<T, 8>(a, bwd, st);
}

int turn(const fm_turn_args* a, bool bwd, void* stream) {
    clear_error();
    if (!a) return fail("fm_turn: no arguments");
    if (const char* e = turn_args_wrong(*a, bwd)) return fail((std::string(bwd ? "fm_turn_bwd: " : "fm_turn: ") + e).c_str());
    if (a->dtype == FM_F32) turn_of_type<float>(*a, bwd, (hipStream_t)stream);
    else if (a->dtype == FM_BF16) turn_of_type<bf16>(*a, bwd, (hipStream_t)stream);
    else turn_of_type<f16>(*a, bwd, (hipStream_t)stream);
    FG_CHECK(hipGetLastError(), -1);
    return 0;
}

}  // namespace fg

using namespace fg;

extern "C" {

int fm_turn(const fm_turn_args* a, void* stream) { return turn(a, false, stream); }
int fm_turn_bwd(const fm_turn_args* a, void* stream) { return turn(a, true, stream); }
long long fm_turn_partial(const fm_turn_args* a) { return 2LL * turn_blocks(*a) * a->dim; }

}  // extern "C"
