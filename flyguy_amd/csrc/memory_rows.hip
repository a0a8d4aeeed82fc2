// Rows of numbers around the memory over decisions: layer norm with its gradients, and dropout from a counter-based generator
// (include/flyguy_memory.h: fm_norm, fm_norm_bwd, fm_drop).
#include <hip/hip_runtime.h>

#include <cmath>

#include "memory.h"

namespace fg {

// Layer norm.  m = mean(x), r = (mean((x - m)^2) + eps)^-1/2, xh = (x - m) r, y = xh w + b.  With u = g w:
// gx = r (u - mean(u) - xh mean(u xh)), gw = sum over rows of g xh, gb = sum over rows of g.
//
// A row is held by a group of lanes: a power of two up to a wave's 64, or (WIDE) the whole workgroup, NV units of V values a
// lane (16 bytes, 8 or single values, as rows are aligned), so that it is read once and its squares are summed about the
// mean.  A group walks several rows, with the weights (gradient: their gradients' sums) in registers all along.  Bound by the
// copy rate: 32,768 rows of 4,096 values of bfloat16 take 98 us forward (5.5 TB/s), 147 the gradient (5.5 TB/s), 4.5 the joining of the
// weights' sums.
struct Group {
    int lanes, shift;                    // lanes: 1 << shift (WIDE: 256)
};
template <int V>
struct FloatsOf {
    typedef float type __attribute__((ext_vector_type(V)));
};
template <class T, int V>
struct ValuesOf {
    typedef T type __attribute__((ext_vector_type(V)));
};

// the sums of N values over a group's lanes; WIDE: over the workgroup, by way of `shared` [4][N]
template <int N, bool WIDE>
__device__ __forceinline__ void sum_over(float (&v)[N], const Group& l, float* shared) {
    const int width = WIDE ? 64 : l.lanes;
    for (int m = 1; m < width; m <<= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], m);
    if constexpr (WIDE) {
        __syncthreads();                                  // (the last use of `shared` is over)
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) shared[(threadIdx.x >> 6) * N + i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = shared[i] + shared[N + i] + shared[2 * N + i] + shared[3 * N + i];
    }
}

template <class T, int V, int NV>
__device__ __forceinline__ void read_row(const T* x, int j, int lanes, int D, float (&v)[NV][V]) {
    typename ValuesOf<T, V>::type u[NV];                  // (lanes past the row read its first values: a branch each would wait)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = (i * lanes + j) * V;
        u[i] = *reinterpret_cast<const typename ValuesOf<T, V>::type*>(x + (at < D ? at : 0));
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) v[i][e] = (i * lanes + j) * V < D ? widen(u[i][e]) : 0.f;
}
template <class T, int V, int NV>
__device__ __forceinline__ void write_row(T* y, int j, int lanes, int D, const float (&v)[NV][V]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = (i * lanes + j) * V;
        typename ValuesOf<T, V>::type u;
#pragma unroll
        for (int e = 0; e < V; ++e) u[e] = narrow<T>(v[i][e]);
        if (at < D) *reinterpret_cast<typename ValuesOf<T, V>::type*>(y + at) = u;
    }
}
// a vector of D float32, `none` where it is not given
template <int V, int NV>
__device__ __forceinline__ void read_floats(const float* w, float none, int j, int lanes, int D, float (&v)[NV][V]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = (i * lanes + j) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) v[i][e] = w ? w[(at < D ? at : 0) + e] : none;
    }
}

// 1 over the deviation, from the sum of squares about a mean that is off by `off`: what rounding left of the mean is found with
// the squares and taken off too (a row of one value is exactly 0, where 1e-7 of it over the root of eps would be 3e-5)
__device__ __forceinline__ float deviation(float squares, float off, float n, float eps) {
    return rsqrtf(fmaxf(squares / n - off * off, 0.f) + eps);
}

template <class T, int V, int NV, bool WIDE>
__global__ __launch_bounds__(256) void k_norm(fm_norm_args a, Group l) {
    __shared__ float shared[WIDE ? 8 : 1];
    const int D = (int)a.width, lanes = WIDE ? 256 : l.lanes, j = threadIdx.x & (lanes - 1);
    const int groups = WIDE ? 1 : 256 >> l.shift, group = WIDE ? 0 : threadIdx.x >> l.shift;
    float w[NV][V], b[NV][V];
    read_floats<V, NV>(a.weight, 1.f, j, lanes, D, w);
    read_floats<V, NV>(a.bias, 0.f, j, lanes, D, b);
    for (long long row = (long long)blockIdx.x * groups + group; row < a.rows; row += (long long)gridDim.x * groups) {
        float v[NV][V], s[1] = {0.f}, q[2] = {0.f, 0.f};
        read_row<T, V, NV>((const T*)a.x + row * a.x_row, j, lanes, D, v);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) s[0] += v[i][e];
        sum_over<1, WIDE>(s, l, shared);
        const float mean = s[0] / (float)D;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const bool there = (i * lanes + j) * V < D;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[i][e] = there ? v[i][e] - mean : 0.f;
                q[0] += v[i][e] * v[i][e];
                q[1] += v[i][e];
            }
        }
        sum_over<2, WIDE>(q, l, shared);
        const float off = q[1] / (float)D, r = deviation(q[0], off, (float)D, (float)a.eps);
        if (j == 0 && a.stats) {
            a.stats[2 * row] = mean + off;
            a.stats[2 * row + 1] = r;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) v[i][e] = fmaf((v[i][e] - off) * r, w[i][e], b[i][e]);
        write_row<T, V, NV>((T*)a.y + row * a.y_row, j, lanes, D, v);
    }
}

// The weights' sums: a lane's over its group's rows, then the groups' in LDS, then (k_norm_sums) the workgroups', always in
// the same order.  partial [blocks][2][width]
template <class T, int V, int NV, bool WIDE>
__global__ __launch_bounds__(256) void k_norm_bwd(fm_norm_args a, Group l) {
    __shared__ float shared[WIDE ? 8 : 256 * NV * V];     // (a group's row: at most its lanes' values)
    const int D = (int)a.width, lanes = WIDE ? 256 : l.lanes, j = threadIdx.x & (lanes - 1);
    const int groups = WIDE ? 1 : 256 >> l.shift, group = WIDE ? 0 : threadIdx.x >> l.shift;
    float w[NV][V], sw[NV][V] = {}, sb[NV][V] = {};
    read_floats<V, NV>(a.weight, 1.f, j, lanes, D, w);
    const float part = 1.f / (float)D;
    for (long long row = (long long)blockIdx.x * groups + group; row < a.rows; row += (long long)gridDim.x * groups) {
        float v[NV][V], g[NV][V], s[2] = {0.f, 0.f};
        read_row<T, V, NV>((const T*)a.x + row * a.x_row, j, lanes, D, v);
        read_row<T, V, NV>((const T*)a.g + row * a.g_row, j, lanes, D, g);
        const float mean = a.stats[2 * row], r = a.stats[2 * row + 1];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const bool there = (i * lanes + j) * V < D;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[i][e] = there ? (v[i][e] - mean) * r : 0.f;
                sw[i][e] += g[i][e] * v[i][e];
                sb[i][e] += g[i][e];
                g[i][e] *= w[i][e];
                s[0] += g[i][e];
                s[1] += g[i][e] * v[i][e];
            }
        }
        if (!a.gx) continue;
        sum_over<2, WIDE>(s, l, shared);
        const float mu = s[0] * part, mx = s[1] * part;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) v[i][e] = r * (g[i][e] - mu - v[i][e] * mx);
        write_row<T, V, NV>((T*)a.gx + row * a.gx_row, j, lanes, D, v);
    }
    if (!a.gweight && !a.gbias) return;
    for (int which = 0; which < 2; ++which) {
        if (!(which ? a.gbias : a.gweight)) continue;
        float* to = a.partial + ((size_t)blockIdx.x * 2 + which) * D;
        if constexpr (!WIDE) __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int at = (i * lanes + j) * V;
            if (at >= D) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) (WIDE ? to : shared + group * D)[at + e] = which ? sb[i][e] : sw[i][e];
        }
        if constexpr (!WIDE) {
            __syncthreads();
            for (int e = threadIdx.x; e < D; e += 256) {
                float s = 0.f;
                for (int i = 0; i < groups; ++i) s += shared[i * D + e];
                to[e] = s;
            }
        }
    }
}

// Rows wider than a workgroup's registers: read again for the deviation, and again for the output.
template <class T>
__global__ __launch_bounds__(256) void k_norm_any(fm_norm_args a) {
    __shared__ float shared[8];
    const long long D = a.width;
    const Group l{256, 8};
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = (const T*)a.x + row * a.x_row;
        T* y = (T*)a.y + row * a.y_row;
        float s[1] = {0.f}, q[2] = {0.f, 0.f};
        for (long long e = threadIdx.x; e < D; e += 256) s[0] += widen(x[e]);
        sum_over<1, true>(s, l, shared);
        const float mean = s[0] / (float)D;
        for (long long e = threadIdx.x; e < D; e += 256) {
            const float v = widen(x[e]) - mean;
            q[0] += v * v;
            q[1] += v;
        }
        sum_over<2, true>(q, l, shared);
        const float off = q[1] / (float)D, r = deviation(q[0], off, (float)D, (float)a.eps);
        if (threadIdx.x == 0 && a.stats) {
            a.stats[2 * row] = mean + off;
            a.stats[2 * row + 1] = r;
        }
        for (long long e = threadIdx.x; e < D; e += 256)
            y[e] = narrow<T>(fmaf((widen(x[e]) - mean - off) * r, a.weight ? a.weight[e] : 1.f, a.bias ? a.bias[e] : 0.f));
    }
}
template <class T>
__global__ __launch_bounds__(256) void k_norm_any_bwd(fm_norm_args a) {
    __shared__ float shared[8];
    const long long D = a.width;
    const float part = 1.f / (float)D;
    const Group l{256, 8};
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = (const T*)a.x + row * a.x_row;
        const T* g = (const T*)a.g + row * a.g_row;
        T* gx = (T*)a.gx + row * a.gx_row;
        const float mean = a.stats[2 * row], r = a.stats[2 * row + 1];
        float s[2] = {0.f, 0.f};
        for (long long e = threadIdx.x; e < D; e += 256) {
            const float u = widen(g[e]) * (a.weight ? a.weight[e] : 1.f);
            s[0] += u;
            s[1] += u * ((widen(x[e]) - mean) * r);
        }
        sum_over<2, true>(s, l, shared);
        for (long long e = threadIdx.x; e < D; e += 256) {
            const float u = widen(g[e]) * (a.weight ? a.weight[e] : 1.f);
            gx[e] = narrow<T>(r * (u - s[0] * part - (widen(x[e]) - mean) * r * (s[1] * part)));
        }
    }
}
// their weights' sums, a column a thread over a slab of rows.  grid (blocks of columns, slabs)
template <class T>
__global__ __launch_bounds__(256) void k_norm_columns(fm_norm_args a) {
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x, D = a.width;
    if (e >= D) return;
    float sw = 0.f, sb = 0.f;
    for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float g = widen(((const T*)a.g)[row * a.g_row + e]);
        sw += g * ((widen(((const T*)a.x)[row * a.x_row + e]) - a.stats[2 * row]) * a.stats[2 * row + 1]);
        sb += g;
    }
    a.partial[(size_t)blockIdx.y * 2 * D + e] = sw;
    a.partial[((size_t)blockIdx.y * 2 + 1) * D + e] = sb;
}

// gweight, gbias: the sums of the workgroups' partials, 16 columns a workgroup, every 16th partial a lane
__global__ __launch_bounds__(256) void k_norm_sums(fm_norm_args a, int blocks) {
    __shared__ float shared[256];
    float* out = blockIdx.y ? a.gbias : a.gweight;
    if (!out) return;
    const long long D = a.width, e = (long long)blockIdx.x * 16 + (threadIdx.x & 15);
    float s = 0.f;
    if (e < D)
#pragma unroll 8
        for (int b = threadIdx.x >> 4; b < blocks; b += 16) s += a.partial[((size_t)b * 2 + blockIdx.y) * D + e];
    shared[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x < 16 && e < D) {
        s = 0.f;
        for (int i = 0; i < 16; ++i) s += shared[16 * i + threadIdx.x];
        out[e] = s;
    }
}

// widest rows of a wave, of a workgroup.  A wave's rows need no barrier, a workgroup's keep fewer values a lane.  8,192 rows, us
// forward and with gradients: of 768 values in bfloat16 9.5 and 28 by waves, 14.3 and 37 by workgroups; of 1,024 in float32 13.4
// and 39, 15.9 and 41; of 1,332 in float32 18.8 and 51 by waves, 17.0 and 48 by workgroups; of 2,048 in bfloat16 17.0 and 49, 16.5
// and 45.
constexpr int NORM_WAVE = 64 * 16, NORM_MOST = 256 * 32;

// a wave's rows: the fewest lanes, a power of two, that hold a row `held` values each
inline Group group_of(long long width, int held) {
    Group l{1, 0};
    while ((long long)l.lanes * held < width && l.lanes < 64) {
        l.lanes *= 2;
        ++l.shift;
    }
    return l;
}
inline int norm_rows_per_block(const fm_norm_args& a) {
    return a.width <= NORM_WAVE ? 256 >> group_of(a.width, 16).shift : 1;
}
// Workgroups of a gradient: 4 rows a group or more, at most 4 a CU, 2 where rows are 8 KB or more, whose values leave room for no
// more at a time; each leaves its sums to be joined.  Forward and gradient with at most 1,024 and 512: 32,768 rows of 4,096 values
// of bfloat16 287 and 275 us, 8,192 of 4,096 of float32 144 and 131, 32,768 of 2,048 of float32 274 and 258, of bfloat16 141 and 166.
inline int norm_blocks(const fm_norm_args& a) {
    const long long at_once = 4LL * norm_rows_per_block(a), b = (a.rows + at_once - 1) / at_once;
    const long long most = a.width * (a.dtype == FM_F32 ? 4 : 2) >= 8192 ? 512 : 1024;
    return (int)(b < 1 ? 1 : b > most ? most : b);
}

template <class T, int V, int HELD>
void launch_held(const fm_norm_args& a, bool bwd, hipStream_t st) {
    constexpr int NV = HELD / V;
    const bool wide = a.width > NORM_WAVE;
    const Group l = wide ? Group{256, 8} : group_of(a.width, HELD);
    const long long per = 256 >> l.shift, blocks = (a.rows + per - 1) / per;
    const unsigned grid = bwd ? (unsigned)norm_blocks(a) : (unsigned)(blocks < 2048 ? blocks : 2048);
    if (wide && bwd) k_norm_bwd<T, V, NV, true><<<grid, 256, 0, st>>>(a, l);
    else if (wide) k_norm<T, V, NV, true><<<grid, 256, 0, st>>>(a, l);
    else if constexpr (HELD <= 16) {
        if (bwd) k_norm_bwd<T, V, NV, false><<<grid, 256, 0, st>>>(a, l);
        else k_norm<T, V, NV, false><<<grid, 256, 0, st>>>(a, l);
    }
}

template <class T, int V>
void launch_norm(const fm_norm_args& a, bool bwd, hipStream_t st) {
    const long long each = a.width <= NORM_WAVE ? (a.width + 63) / 64 : (a.width + 255) / 256;
    if (each <= 8) launch_held<T, V, 8>(a, bwd, st);
    else if (each <= 16) launch_held<T, V, 16>(a, bwd, st);
    else launch_held<T, V, 32>(a, bwd, st);
}

template <class T>
void norm_of_type(const fm_norm_args& a, bool bwd, hipStream_t st) {
    const int size = sizeof(T);
    uintptr_t bits = (uintptr_t)a.x | (uintptr_t)(a.x_row * size) | (uintptr_t)(a.width * size);
    if (bwd) bits |= (uintptr_t)a.g | (uintptr_t)(a.g_row * size) | (uintptr_t)a.gx | (uintptr_t)(a.gx_row * size);
    else bits |= (uintptr_t)a.y | (uintptr_t)(a.y_row * size);
    // (8,192 rows of 1,332 values of bfloat16, forward and with gradients: 16.0 and 41 us in halves of a unit, 17.8 and 47 in single
    // values; of 6,004: 41 and 136, 55 and 206)
    const bool units = !(bits & 15), halves = !(bits & 7);
    if (a.width > NORM_MOST) {
        const unsigned blocks = (unsigned)(a.rows < 2048 ? a.rows : 2048);
        if (!bwd) k_norm_any<T><<<blocks, 256, 0, st>>>(a);
        else {
            // (the weights' sums first: gx may be written over x or g)
            if (a.gweight || a.gbias)
                k_norm_columns<T><<<dim3((unsigned)((a.width + 255) / 256), norm_blocks(a)), 256, 0, st>>>(a);
            if (a.gx) k_norm_any_bwd<T><<<blocks, 256, 0, st>>>(a);
        }
        return;
    }
    if (units) launch_norm<T, Vec<T>::N>(a, bwd, st);
    else if (halves) launch_norm<T, Vec<T>::N / 2>(a, bwd, st);
    else launch_norm<T, 1>(a, bwd, st);
}

const char* norm_wrong(const fm_norm_args& a, bool bwd, bool sizes_only = false) {
    if (a.dtype < FM_F32 || a.dtype > FM_F16) return "values of an unknown type";
    if (a.rows < 0 || a.rows > 1LL << 40) return "other than 0 to 2^40 rows";
    if (a.width < 1 || a.width > 1 << 24) return "rows of other than 1 to 2^24 values";
    if (!(a.eps >= 0)) return "eps below 0";
    if (!a.rows || sizes_only) return nullptr;
    if (!a.x || (bwd ? !a.g || !a.stats : !a.y)) return "a null tensor";
    if (bwd && (a.gweight || a.gbias) && !a.partial) return "no partial";
    return nullptr;
}

int norm(const fm_norm_args* args, bool bwd, void* stream) {
    const char* name = bwd ? "fm_norm_bwd: " : "fm_norm: ";
    clear_error();
    if (!args) return fail((std::string(name) + "no arguments").c_str());
    if (const char* e = norm_wrong(*args, bwd)) return fail((std::string(name) + e).c_str());
    const fm_norm_args& a = *args;
    hipStream_t st = (hipStream_t)stream;
    if (a.rows && (!bwd || a.gx || a.gweight || a.gbias)) {
        if (a.dtype == FM_F32) norm_of_type<float>(a, bwd, st);
        else if (a.dtype == FM_BF16) norm_of_type<bf16>(a, bwd, st);
        else norm_of_type<f16>(a, bwd, st);
        FG_CHECK(hipGetLastError(), -1);
    }
    if (bwd && (a.gweight || a.gbias)) {
        k_norm_sums<<<dim3((unsigned)((a.width + 15) / 16), 2), 256, 0, st>>>(a, a.rows ? norm_blocks(a) : 0);
        FG_CHECK(hipGetLastError(), -1);
    }
    return 0;
}

// ------------------------------------------------------------------------------------------------ dropout
// The generator: Philox4x32 of 10 rounds (Salmon, Moraes, Dror, Shaw: Parallel random numbers, as easy as 1, 2, 3; 2011), a
// bijection of a 128-bit counter (block, offset) by a 64-bit key (the seed); its 128 bits are 8 numbers' 16-bit draws.
__device__ __forceinline__ uint4 philox(unsigned long long block, unsigned long long offset, unsigned long long seed) {
    unsigned c0 = (unsigned)block, c1 = (unsigned)(block >> 32), c2 = (unsigned)offset, c3 = (unsigned)(offset >> 32);
    unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const unsigned long long p0 = (unsigned long long)c0 * 0xD2511F53u, p1 = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (unsigned)(p1 >> 32) ^ c1 ^ k0;
        c1 = (unsigned)p1;
        c2 = (unsigned)(p0 >> 32) ^ c3 ^ k1;
        c3 = (unsigned)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

// 8 numbers a lane.  FLAT: x and y dense and aligned, whole blocks at once; else number i at row i / width of any row stride.
// 32,768 x 2,048 numbers of bfloat16 take 44 us (6.1 TB/s: x partly in cache); a mask kept for the gradient would add a
// sixteenth or more to what both read and write, its 20 products of 32 bits for 8 numbers are hidden.
template <class T, bool FLAT>
__global__ __launch_bounds__(256) void k_drop(fm_drop_args a, unsigned least, float factor) {
    const unsigned long long seed = a.counter[0], offset = a.counter[1];
    const long long n = a.rows * a.width, blocks = (n + 7) >> 3;
    for (long long block = block_number() * 256 + threadIdx.x; block < blocks;
         block += (long long)gridDim.x * gridDim.y * 256) {
        const long long i0 = block * 8;
        typedef typename ValuesOf<T, 8>::type vec;
        vec v;
        if (FLAT && i0 + 8 <= n) v = *reinterpret_cast<const vec*>((const T*)a.x + i0);
        else {
            long long row = i0 / a.width, col = i0 - row * a.width;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = i0 + e < n ? ((const T*)a.x)[row * a.x_row + col] : (T)0.f;
                if (++col == a.width) {
                    col = 0;
                    ++row;
                }
            }
        }
        const uint4 w = philox((unsigned long long)block, offset, seed);
        const unsigned words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const unsigned d = e & 1 ? words[e >> 1] >> 16 : words[e >> 1] & 0xffffu;
            v[e] = d >= least ? narrow<T>(widen(v[e]) * factor) : (T)0.f;
        }
        T* y = (T*)a.y + i0;
        if (FLAT && i0 + 8 <= n) *reinterpret_cast<vec*>(y) = v;
        else
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (i0 + e < n) y[e] = v[e];
    }
}

template <class T>
void drop_of_type(const fm_drop_args& a, unsigned least, float factor, hipStream_t st) {
    const long long n = a.rows * a.width, blocks = ((n + 7) / 8 + 255) / 256;
    const bool flat = (a.x_row == a.width || a.rows == 1) && !(((uintptr_t)a.x | (uintptr_t)a.y) & 15);
    if (flat) k_drop<T, true><<<blocks_of(blocks), 256, 0, st>>>(a, least, factor);
    else k_drop<T, false><<<blocks_of(blocks), 256, 0, st>>>(a, least, factor);
}

}  // namespace fg

using namespace fg;

extern "C" {

int fm_norm(const fm_norm_args* a, void* stream) { return norm(a, false, stream); }
int fm_norm_bwd(const fm_norm_args* a, void* stream) { return norm(a, true, stream); }
long long fm_norm_partial(const fm_norm_args* a) { return a && !norm_wrong(*a, true, true) ? 2LL * norm_blocks(*a) * a->width : 0; }

int fm_drop(const fm_drop_args* a, void* stream) {
    clear_error();
    if (!a) return fail("fm_drop: no arguments");
    if (a->dtype < FM_F32 || a->dtype > FM_F16) return fail("fm_drop: values of an unknown type");
    if (a->rows < 0 || a->width < 0 || a->rows > 1LL << 40 || a->width > 1LL << 40 || (double)a->rows * (double)a->width > 1e12)
        return fail("fm_drop: other than 0 to 1e12 values");
    if (!(a->share >= 0 && a->share <= 1)) return fail("fm_drop: a share outside 0 to 1");
    if (!a->rows || !a->width) return 0;
    if (!a->x || !a->y || !a->counter) return fail("fm_drop: a null tensor");
    const unsigned least = (unsigned)lrint(a->share * 65536);
    const float factor = least < 65536 ? (float)(65536.0 / (65536 - least)) : 0.f;
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == FM_F32) drop_of_type<float>(*a, least, factor, st);
    else if (a->dtype == FM_BF16) drop_of_type<bf16>(*a, least, factor, st);
    else drop_of_type<f16>(*a, least, factor, st);
    FG_CHECK(hipGetLastError(), -1);
    return 0;
}

}  // extern "C"
