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

// Heads of whole 16-byte units (V values): a group of `lanes` lanes (a power of two) takes HB heads of a moment; lane j holds
// two units of a head.  Where pairs lie half apart and the turned part is whole units, units j and j + R / 2V of it, so that the
// lane's pairs are its own (HALVES; the rest goes two units a lane); side by side, units 2j and 2j + 1 (SIDE; SIDE_ANY: the
// turned part ends inside a unit, which costs the others 5% if they ask for it).  Half apart at any place (SPREAD), units 2j
// and 2j + 1 too, and partners pass through LDS inside the group: 27 us instead of the 62 of a wave per row at 8 x 981 moments
// of 16 float32 heads of 128 values, 106 of them turned.  The lane's angles, the weights and the moment's addresses serve all
// HB heads, and all their loads are under way at once.
enum Pairs { HALVES, SIDE, SIDE_ANY, SPREAD };
struct Lanes {
    int lanes, shift, q_chunks, chunks;  // lanes = 1 << shift; chunks of HB heads of queries, in all
};
template <class T, Pairs P>
struct Units {
    static constexpr int V = Vec<T>::N, ANGLES = P == SPREAD ? 2 * V : V;
    int a, b, R;                         // first values of the lane's units (b: dim or more: none); values turned
    float c[ANGLES], s[ANGLES];
    __device__ __forceinline__ Units(int j, int D, int turned) : R(turned) {
        const int ru = R / (2 * V);
        a = P == HALVES && j < ru ? j * V : 2 * j * V;
        b = P == HALVES && j < ru ? (j + ru) * V : a + V;
    }
    __device__ __forceinline__ void angles(const float* cs, int j, float sign) {
        if (a >= R) return;
        if constexpr (P == SPREAD) {                      // of value e of the lane's
#pragma unroll
            for (int i = 0; i < ANGLES; ++i) {
                const int e = a + i;
                const bool second = e >= R / 2;
                if (e < R) angle(cs, second ? e - R / 2 : e, i, second ? sign : -sign);
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (P == HALVES || (P == SIDE ? i < V / 2 || b < R : 2 * (j * V + i) < R)) angle(cs, j * V + i, i, sign);
        }
    }
    __device__ __forceinline__ void angle(const float* cs, int pair, int i, float sign) {
        const float2 f = cs ? reinterpret_cast<const float2*>(cs)[pair] : make_float2(NAN, NAN);
        c[i] = f.x;
        s[i] = sign * f.y;
    }
    // x, y: the values of units a, b (one that is not turned is not touched: it may be anything); row: the group's 2V floats a
    // lane of LDS (SPREAD)
    __device__ __forceinline__ void turn(float (&x)[V], float (&y)[V], float* row) const {
        if constexpr (P == SIDE) {
            if (a < R)
#pragma unroll
                for (int i = 0; i < V / 2; ++i) pair(x, i, 0);
            if (b < R)
#pragma unroll
                for (int i = 0; i < V / 2; ++i) pair(y, i, V / 2);
        } else if constexpr (P == SIDE_ANY) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                if (a + 2 * i < R) pair(x, i, 0);
                if (b + 2 * i < R) pair(y, i, V / 2);
            }
        } else if constexpr (P == HALVES) {
            if (a < R)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float p = x[i], q = y[i];
                    x[i] = p * c[i] - q * s[i];
                    y[i] = q * c[i] + p * s[i];
                }
        } else {
            // (one wave's LDS operations go in order: the compiler only has to leave them so)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                row[a + i] = x[i];
                row[b + i] = y[i];
            }
            asm volatile("" ::: "memory");
            partners(x, a, 0, row);
            partners(y, b, V, row);
            asm volatile("" ::: "memory");
        }
    }
    __device__ __forceinline__ void pair(float (&x)[V], int i, int at) const {
        const float p = x[2 * i], q = x[2 * i + 1];
        x[2 * i] = p * c[at + i] - q * s[at + i];
        x[2 * i + 1] = q * c[at + i] + p * s[at + i];
    }
    __device__ __forceinline__ void partners(float (&x)[V], int first, int at, const float* row) const {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = first + i;
            if (e < R) x[i] = x[i] * c[at + i] + row[e < R / 2 ? e + R / 2 : e - R / 2] * s[at + i];
        }
    }
    __device__ __forceinline__ static void read(const T* p, bool there, typename Vec<T>::type& v) {
        if (there) v = *reinterpret_cast<const typename Vec<T>::type*>(p);
        else
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = (T)0.f;
    }
    __device__ __forceinline__ static void write(T* p, bool there, const float (&x)[V]) {
        if (!there) return;
        typename Vec<T>::type v;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = narrow<T>(x[i]);
        *reinterpret_cast<typename Vec<T>::type*>(p) = v;
    }
    __device__ __forceinline__ static void read_weight(const float* w, int e, bool there, float (&f)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = there ? w[e + i] : 0.f;
    }
};

// sums of HB values over the lanes of a group, side by side
template <int HB>
__device__ __forceinline__ void group_sums(float (&v)[HB], int lanes) {
    for (int m = 1; m < lanes; m <<= 1)
#pragma unroll
        for (int i = 0; i < HB; ++i) v[i] += __shfl_xor(v[i], m);
}

template <class T, Pairs P, bool NORM, int HB>
__global__ __launch_bounds__(256) void k_turn_units(fm_turn_args a, Lanes l, float sign) {
    constexpr int V = Vec<T>::N;
    __shared__ float rows[P == SPREAD ? 256 * 2 * V : 1];
    const int D = (int)a.dim, R = (int)a.rotated, j = threadIdx.x & (l.lanes - 1);
    float* const row = rows + (P == SPREAD ? (threadIdx.x >> l.shift << l.shift) * 2 * V : 0);
    const long long item = block_number() * (256 >> l.shift) + (threadIdx.x >> l.shift);
    const long long m = item / l.chunks, n = m / a.n_moments, t = m - n * a.n_moments;
    if (n >= a.n_seq) return;                             // (a wave's lanes of other groups go on: sums stay in a group)
    int chunk = (int)(item - m * l.chunks);
    const int which = chunk >= l.q_chunks;
    if (which) chunk -= l.q_chunks;
    const fm_view xv = which ? a.x[1] : a.x[0], yv = which ? a.y[1] : a.y[0];
    const int h0 = chunk * HB, hn = min(HB, (int)(which ? a.heads[1] : a.heads[0]) - h0);
    const T* x = (const T*)xv.data + n * xv.seq + t * xv.moment + h0 * xv.head;
    T* y = (T*)yv.data + n * yv.seq + t * yv.moment + h0 * yv.head;
    Units<T, P> u(j, D, R);
    const bool ha = u.a < D, hb = u.b < D;
    typename Vec<T>::type va[HB], vb[HB];
#pragma unroll
    for (int i = 0; i < HB; ++i) {
        u.read(x + i * xv.head + u.a, ha && i < hn, va[i]);
        u.read(x + i * xv.head + u.b, hb && i < hn, vb[i]);
    }
    u.angles(R ? table_line(a, n, t) : nullptr, j, sign);
    const float* w = which ? a.weight[1] : a.weight[0];
    float wa[V], wb[V];
    if (NORM && w) {
        u.read_weight(w, u.a, ha, wa);
        u.read_weight(w, u.b, hb, wb);
    }
    float sum[HB] = {};
    if (NORM && w) {
#pragma unroll
        for (int i = 0; i < HB; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) sum[i] += widen(va[i][e]) * widen(va[i][e]) + widen(vb[i][e]) * widen(vb[i][e]);
        group_sums(sum, l.lanes);
    }
#pragma unroll
    for (int i = 0; i < HB; ++i) {
        float p[V], q[V];
        const float r = NORM && w ? rsqrtf(sum[i] / D + (float)a.eps) : 1.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            p[e] = widen(va[i][e]);
            q[e] = widen(vb[i][e]);
            if (NORM && w) {
                p[e] *= r * wa[e];
                q[e] *= r * wb[e];
            }
        }
        u.turn(p, q, row);
        u.write(y + i * yv.head + u.a, ha && i < hn, p);
        u.write(y + i * yv.head + u.b, hb && i < hn, q);
    }
}

// The gradient with a norm: the turn undone (the sine's sign flipped), then, with xh = x r and u = g' w, gx = r (u - xh
// mean(u xh)).  The weights' gradients sum g' xh over rows: a lane keeps its values' sums over its groups' rows, a
// workgroup's groups are added in LDS, k_turn_gweight adds the workgroups; always in the same order.
// partial [queries, keys][dim][blocks].  grid (blocks, queries and keys)
template <class T, Pairs P, int HB>
__global__ __launch_bounds__(256) void k_turn_units_bwd(fm_turn_args a, Lanes l) {
    constexpr int V = Vec<T>::N;
    __shared__ float shared[256 * 2 * V];                 // a group's row (SPREAD); then [groups][dim]: dim <= lanes x 2V
    const int D = (int)a.dim, R = (int)a.rotated, j = threadIdx.x & (l.lanes - 1), group = threadIdx.x >> l.shift;
    const int groups = 256 >> l.shift, which = blockIdx.y;
    const fm_view xv = a.x[which], yv = a.y[which], gv = a.g[which];
    const float* w = a.weight[which];
    const int H = (int)a.heads[which], chunks = which ? l.chunks - l.q_chunks : l.q_chunks;
    Units<T, P> u(j, D, R);
    const bool ha = u.a < D, hb = u.b < D;
    float wa[V], wb[V], sa[V] = {}, sb[V] = {};
    if (w) {
        u.read_weight(w, u.a, ha, wa);
        u.read_weight(w, u.b, hb, wb);
    }
    const long long items = a.n_seq * a.n_moments * chunks;
    for (long long item = (long long)blockIdx.x * groups + group; item < items; item += (long long)gridDim.x * groups) {
        const long long m = item / chunks, n = m / a.n_moments, t = m - n * a.n_moments;
        const int h0 = (int)(item - m * chunks) * HB, hn = min(HB, H - h0);
        const T* g = (const T*)gv.data + n * gv.seq + t * gv.moment + h0 * gv.head;
        const T* x = (const T*)xv.data + n * xv.seq + t * xv.moment + h0 * xv.head;
        T* y = (T*)yv.data + n * yv.seq + t * yv.moment + h0 * yv.head;
        typename Vec<T>::type ga[HB], gb[HB], va[HB], vb[HB];
#pragma unroll
        for (int i = 0; i < HB; ++i) {
            u.read(g + i * gv.head + u.a, ha && i < hn, ga[i]);
            u.read(g + i * gv.head + u.b, hb && i < hn, gb[i]);
            if (!w) continue;
            u.read(x + i * xv.head + u.a, ha && i < hn, va[i]);
            u.read(x + i * xv.head + u.b, hb && i < hn, vb[i]);
        }
        u.angles(R ? table_line(a, n, t) : nullptr, j, -1.f);
        // mean(u xh) = mean((g' w) x) r: both sums over x at once
        float p[HB][V], q[HB][V], sums[2 * HB] = {};
#pragma unroll
        for (int i = 0; i < HB; ++i) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                p[i][e] = widen(ga[i][e]);
                q[i][e] = widen(gb[i][e]);
            }
            u.turn(p[i], q[i], shared + (threadIdx.x >> l.shift << l.shift) * 2 * V);
            if (!w) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float x0 = widen(va[i][e]), x1 = widen(vb[i][e]);
                sums[i] += x0 * x0 + x1 * x1;
                sums[HB + i] += p[i][e] * wa[e] * x0 + q[i][e] * wb[e] * x1;
            }
        }
        if (w) group_sums(sums, l.lanes);
#pragma unroll
        for (int i = 0; i < HB; ++i) {
            if (w) {
                const float r = rsqrtf(sums[i] / D + (float)a.eps), dot = sums[HB + i] * r / D;
                const bool real = i < hn;                 // (a head past the last adds nothing, also where its r is not finite)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float x0 = widen(va[i][e]) * r, x1 = widen(vb[i][e]) * r;
                    if (real) {
                        sa[e] += p[i][e] * x0;
                        sb[e] += q[i][e] * x1;
                    }
                    p[i][e] = r * (p[i][e] * wa[e] - x0 * dot);
                    q[i][e] = r * (q[i][e] * wb[e] - x1 * dot);
                }
            }
            u.write(y + i * yv.head + u.a, ha && i < hn, p[i]);
            u.write(y + i * yv.head + u.b, hb && i < hn, q[i]);
        }
    }
    if (!a.gweight[which]) return;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < V; ++e) {
        if (ha) shared[group * D + u.a + e] = sa[e];
        if (hb) shared[group * D + u.b + e] = sb[e];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < D; e += 256) {
        float s = 0.f;
        for (int i = 0; i < groups; ++i) s += shared[i * D + e];
        a.partial[((size_t)which * D + e) * gridDim.x + blockIdx.x] = s;
    }
}

// what this wave loads is there (other lanes' stores may follow, to the same places)
__device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Any sizes and strides: one wave per row (a head of a moment), lanes over its values; a partner's value is read again (a
// cache hit).
template <class T, int NE>
__global__ __launch_bounds__(64 * TURN_ROWS) void k_turn(fm_turn_args a, float sign) {
    const int H = (int)(a.heads[0] + a.heads[1]), lane = threadIdx.x & 63, D = (int)a.dim, R = (int)a.rotated;
    const long long row = block_number() * TURN_ROWS + (threadIdx.x >> 6);
    if (row >= a.n_seq * a.n_moments * H) return;
    const long long m = row / H, n = m / a.n_moments, t = m % a.n_moments;
    int h = (int)(row % H);
    const int which = h >= a.heads[0];
    if (which) h -= (int)a.heads[0];
    const fm_view xv = which ? a.x[1] : a.x[0], yv = which ? a.y[1] : a.y[0];
    const T* x = (const T*)xv.data + n * xv.seq + t * xv.moment + h * xv.head;
    T* y = (T*)yv.data + n * yv.seq + t * yv.moment + h * yv.head;
    const float* w = which ? a.weight[1] : a.weight[0];
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
    for (int i = 0; i < NE; ++i) {                        // (all partners are read before anything is written: y may be x)
        const int e = lane + 64 * i;
        if (e >= D) continue;
        v[i] *= r * (w ? w[e] : 1.f);
        if (e < R) {
            const Turn u = turn_of(e, cs, R, a.interleaved);
            v[i] = v[i] * u.c + widen(x[u.partner]) * r * (w ? w[u.partner] : 1.f) * (sign * u.s);
        }
    }
    loads_done();
#pragma unroll
    for (int i = 0; i < NE; ++i)
        if (lane + 64 * i < D) y[lane + 64 * i] = narrow<T>(v[i]);
}

// Its gradient with a norm (see k_turn_units_bwd).
template <class T, int NE>
__global__ __launch_bounds__(64 * TURN_ROWS) void k_turn_bwd(fm_turn_args a) {
    __shared__ float sums[TURN_ROWS][64 * NE];
    const int which = blockIdx.y, H = (int)a.heads[which], lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int D = (int)a.dim, R = (int)a.rotated;
    const fm_view xv = a.x[which], yv = a.y[which], gv = a.g[which];
    const float* w = a.weight[which];
    float gw[NE] = {};
    const long long rows = a.n_seq * a.n_moments * H;
    for (long long row = (long long)blockIdx.x * TURN_ROWS + wave; row < rows; row += (long long)gridDim.x * TURN_ROWS) {
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
        loads_done();
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
        a.partial[((size_t)which * D + e) * gridDim.x + blockIdx.x] = s;
    }
}

// gweight[which][e] = the sum of the workgroups' partials: one wave per value, the lanes' strided sums joined
__global__ __launch_bounds__(64) void k_turn_gweight(fm_turn_args a, int blocks) {
    const int which = blockIdx.y, e = blockIdx.x;
    if (!a.gweight[which]) return;
    const float* p = a.partial + ((size_t)which * a.dim + e) * blocks;
    float s = 0.f;
    for (int b = threadIdx.x; b < blocks; b += 64) s += p[b];
    s = wave_sum(s, 64);
    if (threadIdx.x == 0) a.gweight[which][e] = s;
}

// workgroups of a gradient with a norm: 4 a CU
inline int turn_blocks(const fm_turn_args& a) {
    const long long rows = a.n_seq * a.n_moments * (a.heads[0] > a.heads[1] ? a.heads[0] : a.heads[1]);
    const long long b = (rows + TURN_ROWS - 1) / TURN_ROWS;
    return (int)(b < 1 ? 1 : b > 1024 ? 1024 : b);
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
void launch_any(const fm_turn_args& a, bool grad, float sign, hipStream_t st) {
    if (grad) {
        k_turn_bwd<T, NE><<<dim3(turn_blocks(a), a.heads[1] ? 2 : 1), 64 * TURN_ROWS, 0, st>>>(a);
        return;
    }
    const long long rows = a.n_seq * a.n_moments * (a.heads[0] + a.heads[1]);
    k_turn<T, NE><<<blocks_of((rows + TURN_ROWS - 1) / TURN_ROWS), 64 * TURN_ROWS, 0, st>>>(a, sign);
}

// 4 heads a group: queries and keys of 16 heads of 128 values in bfloat16, 8 x 2048 moments, forward and gradient with a norm:
// 209 / 178 / 173 / 172 us with 1 / 2 / 4 / 8; turned only, 2 x 16384 moments of 20 heads: 144 / 140 / 144 / 150.  The gradient
// with SPREAD pairs takes 2, which its registers hold: 280 us of the former (106 values turned), 330 with 1 or 4.
constexpr int TURN_HEADS = 4, TURN_HEADS_SPREAD = 2;
template <class T, int HB>
Lanes lanes_of(const fm_turn_args& a) {
    Lanes l;
    const int units = (int)a.dim / Vec<T>::N;
    for (l.shift = 0; 2 << l.shift < units; ++l.shift) {}
    l.lanes = 1 << l.shift;
    l.q_chunks = ((int)a.heads[0] + HB - 1) / HB;
    l.chunks = l.q_chunks + ((int)a.heads[1] + HB - 1) / HB;
    return l;
}
template <class T, Pairs P>
void launch_units(const fm_turn_args& a, bool grad, float sign, hipStream_t st) {
    constexpr int HB = TURN_HEADS, HG = P == SPREAD ? TURN_HEADS_SPREAD : TURN_HEADS;
    if (grad) {
        k_turn_units_bwd<T, P, HG><<<dim3(turn_blocks(a), a.heads[1] ? 2 : 1), 256, 0, st>>>(a, lanes_of<T, HG>(a));
        return;
    }
    const Lanes l = lanes_of<T, HB>(a);
    const int groups = 256 >> l.shift;
    const dim3 grid = blocks_of((a.n_seq * a.n_moments * l.chunks + groups - 1) / groups);
    if (a.weight[0] || a.weight[1]) k_turn_units<T, P, true, HB><<<grid, 256, 0, st>>>(a, l, sign);
    else k_turn_units<T, P, false, HB><<<grid, 256, 0, st>>>(a, l, sign);
}

// heads of whole 16-byte units, all aligned (k_turn_units), or anything (k_turn)
template <class T>
bool in_units(const fm_turn_args& a, bool grad) {
    if (a.dim % Vec<T>::N || ((uintptr_t)a.table & 7)) return false;
    for (int i = 0; i < 2; ++i)
        if (a.heads[i] && (!aligned16(a.x[i], sizeof(T)) || !aligned16(a.y[i], sizeof(T)) ||
                           (grad && !aligned16(a.g[i], sizeof(T)))))
            return false;
    return true;
}

template <class T>
void turn_of_type(const fm_turn_args& a, bool grad, float sign, hipStream_t st) {
    if (in_units<T>(a, grad)) {
        if (a.interleaved && a.rotated % Vec<T>::N == 0) launch_units<T, SIDE>(a, grad, sign, st);
        else if (a.interleaved) launch_units<T, SIDE_ANY>(a, grad, sign, st);
        else if (a.rotated % (2 * Vec<T>::N) == 0) launch_units<T, HALVES>(a, grad, sign, st);
        else launch_units<T, SPREAD>(a, grad, sign, st);
        return;
    }
    if (a.dim <= 64) launch_any<T, 1>(a, grad, sign, st);
    else if (a.dim <= 128) launch_any<T, 2>(a, grad, sign, st);
    else if (a.dim <= 256) launch_any<T, 4>(a, grad, sign, st);
    else launch_any<T, 8>(a, grad, sign, st);
}

int turn(const fm_turn_args* args, bool bwd, void* stream) {
    clear_error();
    if (!args) return fail("fm_turn: no arguments");
    if (const char* e = turn_args_wrong(*args, bwd)) return fail((std::string(bwd ? "fm_turn_bwd: " : "fm_turn: ") + e).c_str());
    fm_turn_args a = *args;
    hipStream_t st = (hipStream_t)stream;
    const bool grad = bwd && (a.weight[0] || a.weight[1]);
    if (bwd && !grad)                        // without a norm: g turned back
        for (int i = 0; i < 2; ++i) a.x[i] = a.g[i];
    if (!a.heads[1]) a.gweight[1] = nullptr;
    const bool any = a.n_seq * a.n_moments * (a.heads[0] + a.heads[1]) > 0;
    if (any || grad) {
        const float sign = bwd ? -1.f : 1.f;
        if (a.dtype == FM_F32) turn_of_type<float>(a, grad, sign, st);
        else if (a.dtype == FM_BF16) turn_of_type<bf16>(a, grad, sign, st);
        else turn_of_type<f16>(a, grad, sign, st);
        FG_CHECK(hipGetLastError(), -1);
    }
    if (grad && (a.gweight[0] || a.gweight[1])) {
        k_turn_gweight<<<dim3((unsigned)a.dim, 2), 64, 0, st>>>(a, turn_blocks(a));
        FG_CHECK(hipGetLastError(), -1);
    }
    return 0;
}

}  // namespace fg

using namespace fg;

extern "C" {

int fm_turn(const fm_turn_args* a, void* stream) { return turn(a, false, stream); }
int fm_turn_bwd(const fm_turn_args* a, void* stream) { return turn(a, true, stream); }
long long fm_turn_partial(const fm_turn_args* a) { return a ? 2LL * turn_blocks(*a) * a->dim : 0; }

}  // extern "C"
