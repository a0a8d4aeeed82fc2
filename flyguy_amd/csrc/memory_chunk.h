// What the chunked kernels of the memory over decisions share: where packed stretches and their segments lie, numbers as sums
// of bfloat16 terms on the matrix cores, and chunks of moments in LDS.
#pragma once
#include "memory.h"

namespace fg {

// A: a launch's struct with starts, wide (its integers' width), n_seq, n_moments, and where stretches are cut, L, L0 (moments a
// segment, and of a stretch's first one) and nseg (segments of the longest stretch).

// bound i of packed stretches: their start i, brought into the moments (past the last one: past every moment)
template <class A>
__device__ __forceinline__ unsigned bound_of(const A& a, int i) {
    const long long b = index_at(a.starts, min(i, a.n_seq), a.wide);
    return i > a.n_seq ? ~0u : b < 0 ? 0u : b > a.n_moments ? (unsigned)a.n_moments : (unsigned)b;
}

// Packed moments belong to leaves of a search in rows of 8 bounds, in each row to the last one before the first bound past the
// moment: leaf n < n_seq is stretch n, leaf n_seq what lies past the last one.  As such a search never goes back while the
// moment goes on, leaves lie in order and share no moment whatever the starts are; where these do not fall, leaf n is
// [starts[n], starts[n+1]).  Its moments are those from the largest of the bounds that the search passes, to the least of those
// it stops at: the rows' 5 x 8 bounds in one load, and then the ends are bounds n and n + 1 unless a ballot finds others.
// All 64 lanes come here together.
constexpr int ROW_BITS = 3, ROWS = 5;    // 8^5 leaves
template <class A>
__device__ __forceinline__ void leaf_of(const A& a, int n, long long& first, long long& count) {
    n = __builtin_amdgcn_readfirstlane(n);
    const int lane = threadIdx.x & 63, at = lane & 7, shift = (lane >> ROW_BITS) * ROW_BITS, digit = n >> shift & 7;
    const unsigned bound = bound_of(a, ((n >> shift & ~7) + at) << shift);
    const int row = __builtin_ctz(~n) / ROW_BITS;         // (bound n + 1 stands in the first row that it does not overflow)
    unsigned low = __builtin_amdgcn_readlane((int)bound, n & 7);
    unsigned high = __builtin_amdgcn_readlane((int)bound, 8 * row + (n >> row * ROW_BITS & 7) + 1);
    high = min(high, (unsigned)a.n_moments);
    if (__ballot((at <= digit && bound > low) || (at == digit + 1 && bound < high))) {
        unsigned most = at <= digit ? bound : 0, least = at == digit + 1 ? bound : high;
        for (int m = 1; m < 64; m <<= 1) {
            most = max(most, (unsigned)__shfl_xor((int)most, m));
            least = min(least, (unsigned)__shfl_xor((int)least, m));
        }
        low = __builtin_amdgcn_readfirstlane((int)most);
        high = __builtin_amdgcn_readfirstlane((int)least);
    }
    first = low;
    count = high > low ? high - low : 0;
}
// the leaf that moment t lies in, and its moments; -1: t lies before the first
template <class A>
__device__ __forceinline__ int leaf_at(const A& a, unsigned t, long long& first, long long& count) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = a.n_seq;            // the last bound that is not past it, if none falls
    while (lo < hi) {
        const int step = (hi - lo + 63) >> 6, at = lo + (lane + 1) * step;
        lo += __popcll(__ballot(at <= hi && bound_of(a, at) <= t)) * step;
        hi = min(hi, lo + step - 1);
    }
    leaf_of(a, lo, first, count);
    if (t >= first && t < first + count) return lo;
    lo = 0;                              // some do, or t lies before the first: row by row
    for (int shift = (ROWS - 1) * ROW_BITS; shift >= 0; shift -= ROW_BITS) {
        const unsigned long long past = __ballot(lane > 7 || bound_of(a, lo + (lane << shift)) > t);
        const int before = __builtin_ctzll(past);
        if (!before) return -1;
        lo += (before - 1) << shift;
    }
    leaf_of(a, lo, first, count);
    return lo;
}

// the moments of stretch n: [first, first + count) of the views
template <class A>
__device__ __forceinline__ void stretch_of(const A& a, int n, long long& first, long long& count) {
    if (a.starts) {
        leaf_of(a, n, first, count);
        return;
    }
    first = 0;
    count = a.n_moments;
}

// the first moment of segment s of a stretch
template <class A>
__device__ __forceinline__ long long start_of(const A& a, long long s) { return s ? a.L0 + (s - 1) * a.L : 0; }

// Whole segments before moment `first` (at most n_moments <= 2^31, as L - 64 is).
template <class A>
__device__ __forceinline__ int segments_before(const A& a, long long first) { return (int)((unsigned)first / (unsigned)a.L); }

// The slot of a packed stretch's first segment: its segments and the next one's that has moments never share one, as floor(b /
// L) + 1 + floor((b + c) / L) - floor(b / L) >= ceil(c / L).  (A stretch without moments uses none.)
template <class A>
__device__ __forceinline__ int first_slot(const A& a, int n, long long first) {
    return !a.starts || a.nseg == 1 ? n * a.nseg : segments_before(a, first) + n;
}
// (stretch, segment, slot) of a workgroup; false: it has none.  Packed stretches: the first n_seq workgroups take their first
// segments, workgroup n_seq + e the segment s > 0 of the stretch with floor(b / L) + s - 1 = e, the one that moment (e + 1) L - 1
// lies in.  So most search nothing, and those without a segment come last (k_scan): 37 stretches of 1,531 moments in the middle,
// 4 heads of 64 x 128 values in bfloat16, take 98 us, 110 with a binary search by every workgroup and slots in the stretches'
// order.
template <class A>
__device__ __forceinline__ bool segment_of(const A& a, int block, int& n, int& seg, int& slot, long long& first,
                                           long long& count) {
    if (!a.starts || a.nseg == 1) {
        seg = block / a.n_seq;
        n = block - seg * a.n_seq;
        if (a.L0 != a.L) seg = a.nseg - 1 - seg;          // (the long segments first)
        stretch_of(a, n, first, count);
    } else {
        const int e = block - a.n_seq;
        if (e < 0) {
            n = block;
            seg = 0;
            stretch_of(a, n, first, count);
        } else {
            n = leaf_at(a, (unsigned)((e + 1) * a.L - 1), first, count);
            if (n < 0 || n == a.n_seq) return false;
            seg = e - segments_before(a, first) + 1;
        }
    }
    slot = first_slot(a, n, first) + seg;
    return seg == 0 || start_of(a, seg) < count;
}

typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// A number as a sum of bfloat16 terms, each the rest's nearest: 1, 2, 3 terms hold 8, 16, 24 bits.  A product of two sums
// keeps the pairs of terms (i, j) with i + j < the longer one's terms: what is dropped is below its last bit.
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
template <int P, int V>
struct Sum {
    typedef bf16 vec __attribute__((ext_vector_type(V)));
    typedef float wide __attribute__((ext_vector_type(V)));
    vec term[P];
    // values of any places (whole vectors: two values a conversion)
    __device__ __forceinline__ void of(wide r) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            term[p] = __builtin_convertvector(r, vec);
            if (p + 1 < P) r -= __builtin_convertvector(term[p], wide);
        }
    }
    // values that one sum takes: a term is taken off, exactly, by its pair's product with (-1, 0), without widening it; one that
    // is not finite spoils its neighbour, and the sum is not finite then anyway
    __device__ __forceinline__ void of_summed(wide r) {
        unsigned one = 0x0000bf80u, two = 0xbf800000u;    // (in registers: as constants of this instruction they come out
        asm("" : "+s"(one), "+s"(two));                   // as other numbers)
        const bf16x2 first = __builtin_bit_cast(bf16x2, one), second = __builtin_bit_cast(bf16x2, two);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            term[p] = __builtin_convertvector(r, vec);
            if (p + 1 == P) break;
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const bf16x2 t = pair(term[p], i);
                r[i] = __builtin_amdgcn_fdot2_f32_bf16(t, first, r[i], false);
                r[i + 1] = __builtin_amdgcn_fdot2_f32_bf16(t, second, r[i + 1], false);
            }
        }
    }
    __device__ __forceinline__ static bf16x2 pair(vec v, int i) {
        if constexpr (V == 4) return i ? __builtin_shufflevector(v, v, 2, 3) : __builtin_shufflevector(v, v, 0, 1);
        else return i == 0 ? __builtin_shufflevector(v, v, 0, 1) : i == 2 ? __builtin_shufflevector(v, v, 2, 3)
                  : i == 4 ? __builtin_shufflevector(v, v, 4, 5) : __builtin_shufflevector(v, v, 6, 7);
    }
};
typedef Sum<1, 8>::wide f32x8;
template <int PA, int PB>
__device__ __forceinline__ f32x4 mfma(const Sum<PA, 8>& a, const Sum<PB, 8>& b, f32x4 c) {
    constexpr int most = PA > PB ? PA : PB;
#pragma unroll
    for (int o = most - 1; o >= 0; --o)                   // (the small ones first)
#pragma unroll
        for (int i = 0; i < PA; ++i)
            if (o - i >= 0 && o - i < PB) c = mfma(a.term[i], b.term[o - i], c);
    return c;
}

// How a value type goes through the matrix cores: X terms hold a value exactly; W terms a weight or the state where they
// make an output (which has fewer bits; what cancels among the terms is off by 2^-16 of their magnitudes, and a third term costs 3
// to 11% of a pass of 128-value heads without changing its error against 64 bits); a chunk's moments (what fits LDS with X planes of x, y and v).
template <class T>
struct Form;
template <>
struct Form<bf16> {
    static constexpr int X = 1, W = 2, CHUNK = 64;
};
template <>
struct Form<f16> {
    static constexpr int X = 2, W = 2, CHUNK = 32;
};
template <>
struct Form<float> {
    static constexpr int X = 3, W = 3, CHUNK = 32;
};
constexpr int CHUNK_MAX = 64;
constexpr int S_TERMS = 3;               // terms of v times its decay: the state is a float32 result

// 16 bytes of a row from column c, value by value, zeros past the width
template <class T>
__device__ __forceinline__ uint4 load16(const T* row, int c, int width, bool there) {
    if (!there || c >= width) return make_uint4(0, 0, 0, 0);
    typename Vec<T>::type v;
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i) v[i] = c + i < width ? row[c + i] : (T)0.f;
    return __builtin_bit_cast(uint4, v);
}
// ... as terms into its planes in LDS, `plane` apart
template <class T>
__device__ __forceinline__ void store_terms(uint4 r, bf16* to, int plane) {
    if constexpr (Form<T>::X == 1) {
        *reinterpret_cast<uint4*>(to) = r;
    } else {
        constexpr int V = Vec<T>::N;
        const typename Vec<T>::type in = __builtin_bit_cast(typename Vec<T>::type, r);
        Sum<Form<T>::X, V> s;
        s.of(__builtin_convertvector(in, typename Sum<1, V>::wide));
#pragma unroll
        for (int p = 0; p < Form<T>::X; ++p) *reinterpret_cast<typename Sum<1, V>::vec*>(to + p * plane) = s.term[p];
    }
}

// 8 values side by side, of each plane
template <int P>
__device__ __forceinline__ Sum<P, 8> across(const bf16* p, int plane) {
    Sum<P, 8> s;
#pragma unroll
    for (int i = 0; i < P; ++i) s.term[i] = *reinterpret_cast<const bf16x8*>(p + i * plane);
    return s;
}
// Two 4 x 16 blocks of LDS, `apart` values apart, transposed: lane c of a block's 16 lanes gets its column c, 4 rows of each.
// p: this lane's share of the first block, 4 values of row c / 4.
__device__ __forceinline__ bf16x8 columns8(const bf16* p, int apart) {
    typedef __attribute__((address_space(3))) s16x4* at;
    const bf16x4 a = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at)p));
    const bf16x4 b = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at)(p + apart)));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <int P>
__device__ __forceinline__ Sum<P, 8> down(const bf16* p, int apart, int plane) {
    Sum<P, 8> s;
#pragma unroll
    for (int i = 0; i < P; ++i) s.term[i] = columns8(p + i * plane, apart);
    return s;
}

// Where a row's 8-value share q stands in LDS: rows of 8 or 16 shares, unpadded, the shares of row 4g + r (of 16) exchanged
// by q ^ (r, g), so that both the 16 rows of a share and the 4 shares of 4 rows that a transposing read takes are spread over
// the banks.  (Conflicts are counted all the same, 39% of the cycles in which LDS is busy; one source is the weights' pieces,
// written 8 bytes at a time 16 bytes apart.)  place(row, q + 4b) = place(row, q) ^ 32 b where q < 4.
template <int WIDTH>
__device__ __forceinline__ int place(int row, int q) {
    const int r = row & 3, g = row >> 2 & 3, swap = (g & 1) << 1 | g >> 1;
    return row * WIDTH + 8 * (q ^ (WIDTH == 128 ? r << 2 | swap : (r & 2) << 1 | swap));
}

// an opaque copy: what is computed from it stays where it is used, instead of in registers all along
template <class V>
__device__ __forceinline__ V here(V v) {
    asm volatile("" : "+v"(v));
    return v;
}

// a value that all lanes share, in a scalar register
__device__ __forceinline__ float shared_by_all(float v) {
    return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
}

__device__ __forceinline__ long long shared_by_all(long long v) {
    const unsigned lo = __builtin_amdgcn_readfirstlane((int)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
    return (long long)((unsigned long long)hi << 32 | lo);
}

// A chunk's rows in memory, `rows` of them `step` bytes apart from p, of `width` bytes: loads outside give zeros, stores
// outside are dropped, so that lanes without a row or column need no branch.  NOWHERE: such a lane's offset.
constexpr unsigned NOWHERE = 0xc0000000u;
constexpr long long STRIDE_MOST = 1 << 22;               // values from row to row: 64 rows end below 2^30 bytes
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const void* p, int rows, long long step, int width) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)((rows - 1) * step) + width, 0x00020000);
}
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

}  // namespace fg
