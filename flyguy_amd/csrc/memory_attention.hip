// Linear attention with a decay for each head (include/flyguy_memory.h: fm_attention, fm_attention_bwd, fm_step).
//
// One scan computes everything: with x, y, v of K, K, N values a moment, a state Z [K][N] and l = exp(log_decay),
//   Z_i = l Z_{i-1} + y_i v_i^T,   out_i = c x_i Z_i.
// The forward is the scan of (q, k, v); the gradient of q that of (go, v, k), with the start state transposed; the
// gradients of k and v those of (v, go, q) and (k, q, go) over the moments backwards, from the end state's gradient, which
// the last moment's term does not decay (c on what is added instead); the second one's end state, decayed once more, is the
// start state's gradient.  A gradient's three scans are one launch.
#include <hip/hip_runtime.h>

#include <cmath>
#include <type_traits>

#include "memory.h"

namespace fg {

constexpr int ATT_MAX = 128;             // values of a head

struct Scan {
    fm_view x, y, v;
    int xs, ys, vs;                      // query heads per head of x, y, v (1, or q_heads / k_heads)
    void* out;                           // dense [moments][heads][N], of the values' type or (wide) float32; 0: no output
    const float* init;                   // start state [n_seq][heads][K][N] (transposed: [N][K]); 0: zeros
    float* fin;                          // end state [n_seq][heads][K][N]; 0: not wanted
    float* seg;                          // [slots][heads][K][N]: segments' own states, then their start states
    int K, N, transposed, backwards, wide;
    float c;
};

struct Scans {
    Scan s[3];
    const float* log_decay;
    const void* starts;
    long long n_moments, L, L0;          // L: moments per segment, L0: of a stretch's first one (multiples of CHUNK_MAX)
    int wide, heads, n_seq, nseg, slots; // slots of segments: n_seq x nseg, or an upper bound for packed stretches
    int joined, scans;                   // the segments' start states are there (k_scan_join); the launch's scans
    int clearing;                        // places after the slots' for the outputs of moments that are in no stretch
};

// bound i of packed stretches: their start i, brought into the moments (past the last one: past every moment)
__device__ __forceinline__ unsigned bound_of(const Scans& a, int i) {
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
__device__ __forceinline__ void leaf_of(const Scans& a, int n, long long& first, long long& count) {
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
__device__ __forceinline__ int leaf_at(const Scans& a, unsigned t, long long& first, long long& count) {
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
__device__ __forceinline__ void stretch_of(const Scans& a, int n, long long& first, long long& count) {
    if (a.starts) {
        leaf_of(a, n, first, count);
        return;
    }
    first = 0;
    count = a.n_moments;
}

// (-inf: 0 times it would not be 0; NaN stays NaN)
__device__ __forceinline__ float log_decay_of(const Scans& a, int h) {
    const float d = a.log_decay[h];
    return d < -1e30f ? -1e30f : d;
}

// the first moment of segment s of a stretch
__device__ __forceinline__ long long start_of(const Scans& a, long long s) { return s ? a.L0 + (s - 1) * a.L : 0; }

// Whole segments before moment `first` (at most n_moments <= 2^31, as L - 64 is).
__device__ __forceinline__ int segments_before(const Scans& a, long long first) { return (int)((unsigned)first / (unsigned)a.L); }

// The slot of a packed stretch's first segment: its segments and the next one's that has moments never share one, as floor(b /
// L) + 1 + floor((b + c) / L) - floor(b / L) >= ceil(c / L).  (A stretch without moments uses none.)
__device__ __forceinline__ int first_slot(const Scans& a, int n, long long first) {
    return !a.starts || a.nseg == 1 ? n * a.nseg : segments_before(a, first) + n;
}
// (stretch, segment, slot) of a workgroup; false: it has none.  Packed stretches: the first n_seq workgroups take their first
// segments, workgroup n_seq + e the segment s > 0 of the stretch with floor(b / L) + s - 1 = e, the one that moment (e + 1) L - 1
// lies in.  So most search nothing, and those without a segment come last (k_scan): 37 stretches of 1,531 moments in the middle,
// 4 heads of 64 x 128 values in bfloat16, take 98 us, 110 with a binary search by every workgroup and slots in the stretches'
// order.
__device__ __forceinline__ bool segment_of(const Scans& a, int block, int& n, int& seg, int& slot, long long& first,
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

// A state's value at (k, c) of the start state of stretch n, decayed once where the scan goes forwards (Z = l S).
__device__ __forceinline__ float start_value(const Scan& s, size_t at, int k, int c, const Keep& keep) {
    if (!s.init || k >= s.K || c >= s.N) return 0.f;
    const float z = s.init[at + (s.transposed ? (size_t)c * s.K + k : (size_t)k * s.N + c)];
    return s.backwards ? z : keep(z);
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

// The scan in chunks, on the matrix cores (v_mfma_f32_16x16x32_bf16).  With i, j the moments inside a chunk of n and Z the
// state before it, decayed once (Z = l S),
//   out_i = c sum_{j <= i} l^(i-j) (x_i . y_j) v_j + c' l^i x_i Z,   Z' = l^n Z + sum_j c'' l^(n-j) y_j v_j^T
// (forwards c' = c, c'' = 1; backwards c' = 1, c'' = c, so that the end state's gradient comes in and the start state's goes
// out unscaled).  A stretch's last chunk, where it is short, has its moments in the last rows and zeros before them, so that
// its decays to the chunk's end are a whole chunk's.
// A workgroup of 4 waves walks one segment of one head; wave w owns the state's columns 16 NT w .., in accumulators all
// along: a 16 x 16 accumulator block holds, in lane (column c, group g), rows 4g .. 4g + 3, which is also how a product's
// operand wants it with the rows as the summed index.  So the state passes from product to product in registers, and the
// order of the summed index (any, if both operands have it) is chosen so: state blocks 2b, 2b + 1 are the rows 32 b + 8g +
// (0 .. 3), (4 .. 7), and a lane's 8 values of x or y are then side by side.  y^T and v^T come out of LDS by transposing
// reads.  Outputs are formed transposed, so that a lane stores a row's values side by side.  The weights (x . y) l^(i-j) of
// the chunk's 16 x 16 blocks on and below the diagonal are dealt to the waves and shared through LDS; the state's additions,
// which do not need them, run before the barrier that waits for them (780 -> 759 us a learning step of 8 x 4096 moments of 16
// heads of 128 values, bfloat16).
// A value of v that is not finite reaches only the outputs from its moment on (there: NaN), though 0 weights meet it in the
// products: such a chunk's products run with zeros in its place.
// What bounds it: a chunk's phases between its three barriers, which do not overlap, with the two workgroups a CU that
// registers and LDS (60 KB) of 128 x 128 states both allow.  32,768 moments of 8 such heads in bfloat16, 57 segments, take 96
// us: 1.6 waves a SIMD, whose vector instructions (sums of terms, decays) take 38% of the time and matrix instructions 26%;
// LDS is read 22% of it.  512 heads of 4,096 moments in one segment each: 620 us, 3.5 TB/s of a copy's 5.2; 477 without loads
// and stores, 480 without the products.
constexpr int WAVES = 4;
template <class T, int KT, int NT, bool OUT>
struct Tile {
    static constexpr int CH = Form<T>::CHUNK, KW = 32 * KT, NW = 16 * NT * WAVES;
    static constexpr int XP = CH * KW, VP = CH * NW, PIECES = CH == 64 ? 6 : 2;
    static constexpr int LDS = Form<T>::X * 2 * (XP * (OUT ? 2 : 1) + VP) + (OUT ? PIECES * Form<T>::W * 1024 : 0);
    // waves a SIMD that LDS lets in, at most 4 (128 registers); two blocks of columns a wave: 3 or 2
    static constexpr int FIT = 160 * 1024 / LDS * WAVES / 4, MOST = NT == 1 ? 4 : KT == 2 ? 3 : 2;
    static constexpr int PER_SIMD = FIT < 1 ? 1 : FIT > MOST ? MOST : FIT;
};
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

// The outputs of the moments before the first stretch and after the last one: zeros, by all 256 threads of each of the workgroups
// that come after the slots'.  (A pack of 4,096 moments in a place for 262,144, 8 heads of 128 values, bfloat16: 6,014 us cleared
// byte by byte in the stretches' own workgroups, 438 by these.)
__device__ __forceinline__ void clear_outside(const Scans& a, const Scan& s, int size, long long share) {
    const long long shares = (long long)a.clearing * a.heads, row = (long long)a.heads * s.N * size;
    if (!s.out || share >= shares) return;
    long long past, rest;
    leaf_of(a, a.n_seq, past, rest);
    auto clear = [&](uintptr_t from, uintptr_t to) {      // (the ends up to a multiple of 16 bytes one by one)
        const uintptr_t up = (from + 15) & ~(uintptr_t)15, down = to & ~(uintptr_t)15, lo = up < to ? up : to,
                        hi = down > lo ? down : lo;
        if (share == 0 && threadIdx.x < lo - from) ((char*)from)[threadIdx.x] = 0;
        if (share == 0 && threadIdx.x < to - hi) ((char*)hi)[threadIdx.x] = 0;
        for (uintptr_t p = lo + 16 * (share * 256 + threadIdx.x); p < hi; p += 16 * 256 * shares)
            *(uint4*)p = make_uint4(0, 0, 0, 0);
    };
    clear((uintptr_t)s.out, (uintptr_t)s.out + bound_of(a, 0) * row);
    clear((uintptr_t)s.out + past * row, (uintptr_t)s.out + (past + rest) * row);
}

template <class T, int KT, int NT, bool VEC, bool OUT>
__global__ __launch_bounds__(64 * WAVES, (Tile<T, KT, NT, OUT>::PER_SIMD)) void k_scan(Scans a) {
    using S = Tile<T, KT, NT, OUT>;
    constexpr int X = Form<T>::X, W = Form<T>::W, CH = S::CH, JB = CH / 16, VN = Vec<T>::N;
    constexpr int KW = S::KW, NW = S::NW, XP = S::XP, VP = S::VP, PIECES = S::PIECES;
    constexpr int XC = KW / VN, VC = NW / VN;                                // 16-byte shares of a row
    constexpr int XR = 64 * WAVES / XC, VR = 64 * WAVES / VC;                // rows between a thread's shares
    constexpr int XV = CH / XR, VV = CH / VR;                                // a thread's shares
    static_assert(XV * XR == CH && VV * VR == CH, "");
    __shared__ __align__(16) bf16 sx[OUT ? X * XP : 8], sy[X * XP], sv[X * VP];
    __shared__ __align__(16) bf16x8 sp[OUT ? PIECES : 1][W][64];
    // (heads first, then scans: a packed launch's workgroups without a segment come last, or some CUs would get only such; and
    // a gradient's scans read the same moments at about the same time)
    const unsigned block = (unsigned)block_number(), group = block / a.heads, place_in = group / a.scans;
    const int h = (int)(block - group * a.heads);
    const Scan& s = a.s[group - place_in * a.scans];
    if (place_in >= (unsigned)a.slots) {
        if (OUT && a.clearing)
            clear_outside(a, s, s.wide ? 4 : (int)sizeof(T), (long long)(place_in - a.slots) * a.heads + h);
        return;
    }
    int n, seg, slot;
    long long first, count;
    if (!segment_of(a, (int)place_in, n, seg, slot, first, count)) return;
    n = __builtin_amdgcn_readfirstlane(n);
    seg = __builtin_amdgcn_readfirstlane(seg);
    slot = __builtin_amdgcn_readfirstlane(slot);
    first = shared_by_all(first);
    count = shared_by_all(count);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int w0 = 16 * NT * wave;                        // this wave's columns from here
    const long long from = start_of(a, seg), most = seg ? a.L : a.L0, left = count - from < most ? count - from : most;
    const bool last = from + left == count;
    if (!OUT && last) return;                             // (the last segment's own state is needed by none)
    const float ld = shared_by_all(log_decay_of(a, h));
    const size_t at = ((size_t)n * a.heads + h) * s.K * s.N;
    const float e2 = shared_by_all(ld * 1.44269504f);
    auto power = [&](int i) { return __builtin_amdgcn_exp2f(e2 * (float)i); };

    f32x4 z[2 * KT][NT];                                  // the state
    auto row_of = [&](int b, int r) { return 32 * (b >> 1) + 8 * g + 4 * (b & 1) + r; };
    // the column of lane c in block t; a lane's outputs are then side by side
    auto col_of = [&](int t, int m) { return w0 + (NT == 2 ? 8 * (m >> 2) + 4 * t + (m & 3) : m); };
    {
        // the start state: the segment's where k_scan_join has left it, else the stretch's, decayed once where the scan goes
        // forwards (not at all if there are no moments: it goes through as it is), joined with the segments' own before this one
        const size_t step = (size_t)a.heads * s.K * s.N, mine = ((size_t)slot * a.heads + h) * s.K * s.N;
        const bool ready = a.nseg > 1 && a.joined && count, flip = !ready && s.transposed;
        const float* z0 = !OUT ? nullptr : ready ? s.seg + mine : s.init ? s.init + at : nullptr;
        const int zk = flip ? 1 : s.N, zc = flip ? s.K : 1, before = OUT && a.nseg > 1 && !a.joined ? seg : 0;
        const Keep once(!ready && !s.backwards && count ? ld : 0.f), over(ld * (float)a.L), over0(ld * (float)a.L0);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int b = 0; b < 2 * KT; ++b) z[b][t] = f32x4{0.f, 0.f, 0.f, 0.f};
            const int col = min(col_of(t, c), s.N - 1);   // (what a lane without a row or column reads is dropped below)
            if (z0)
#pragma unroll
                for (int b = 0; b < 2 * KT; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r) z[b][t][r] = once(z0[min(row_of(b, r), s.K - 1) * zk + col * zc]);
            for (int i = 0; i < before; ++i) {
                const float* own = s.seg + mine - (size_t)(before - i) * step + col;
#pragma unroll
                for (int b = 0; b < 2 * KT; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r) z[b][t][r] = (i ? over : over0)(z[b][t][r]) + own[min(row_of(b, r), s.K - 1) * s.N];
            }
#pragma unroll
            for (int b = 0; b < 2 * KT; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) z[b][t][r] = row_of(b, r) < s.K && col_of(t, c) < s.N ? z[b][t][r] : 0.f;
        }
    }

    // this thread's shares of a chunk's rows
    const int xrow = tid / XC, xcol = tid % XC * VN, vrow = tid / VC, vcol = tid % VC * VN;
    auto rows_from = [&](long long i0) { return (int)(left - i0 < CH ? left - i0 : CH); };
    // the chunk from the segment's moment i0: its moment lowest in memory, and a row's place from there
    auto lowest = [&](long long i0, int rows) {
        return (a.starts ? first : 0) + (s.backwards ? count - from - i0 - rows : from + i0);
    };
    auto in_memory = [&](int row, int pad) { return s.backwards ? CH - 1 - row : row - pad; };
    auto base = [&](const fm_view& v, int share, long long low) {
        return (const T*)v.data + (a.starts ? 0 : n * v.seq) + (h / share) * v.head + low * v.moment;
    };
    const int sx_ = (int)s.x.moment * (int)sizeof(T), sy_ = (int)s.y.moment * (int)sizeof(T), sv_ = (int)s.v.moment * (int)sizeof(T);
    const int row_sign = s.backwards ? -1 : 1;
    uint4 rx[XV], ry[XV], rv[VV];
    auto fetch = [&](long long i0) {                      // the chunk from the segment's moment i0
        const int rows = rows_from(i0), pad = CH - rows;
        const long long low = lowest(i0, rows);
        const T *px = OUT ? base(s.x, s.xs, low) : nullptr, *py = base(s.y, s.ys, low), *pv = base(s.v, s.vs, low);
        if constexpr (VEC) {
            const auto bx = rows_at(px, rows, sx_, s.K * (int)sizeof(T)), by = rows_at(py, rows, sy_, s.K * (int)sizeof(T));
            const auto bv = rows_at(pv, rows, sv_, s.N * (int)sizeof(T));
            // (the lanes' places anew each time, from the thread's number: kept, they cost registers that the products need)
            const int t = here(tid), xr = t / XC, xc = t % XC * VN, vr = t / VC, vc = t % VC * VN;
            const unsigned ax = xc < s.K ? in_memory(xr, 0) * sx_ + xc * (int)sizeof(T) : NOWHERE;
            const unsigned ay = xc < s.K ? in_memory(xr, 0) * sy_ + xc * (int)sizeof(T) : NOWHERE;
            const unsigned av = vc < s.N ? in_memory(vr, 0) * sv_ + vc * (int)sizeof(T) : NOWHERE;
            auto load = [&](__amdgpu_buffer_rsrc_t r, unsigned at, int row, int step) {
                if (pad) at = row < pad ? NOWHERE : at - (s.backwards ? 0 : pad * step);
                return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0));
            };
#pragma unroll
            for (int i = 0; i < XV; ++i) {
                if (OUT) rx[i] = load(bx, ax + i * XR * row_sign * sx_, xr + i * XR, sx_);
                ry[i] = load(by, ay + i * XR * row_sign * sy_, xr + i * XR, sy_);
            }
#pragma unroll
            for (int i = 0; i < VV; ++i) rv[i] = load(bv, av + i * VR * row_sign * sv_, vr + i * VR, sv_);
        } else {
#pragma unroll
            for (int i = 0; i < XV; ++i) {
                const int row = xrow + i * XR;
                const bool there = row >= pad;
                if (OUT) rx[i] = load16(px + in_memory(row, pad) * s.x.moment, xcol, s.K, there);
                ry[i] = load16(py + in_memory(row, pad) * s.y.moment, xcol, s.K, there);
            }
#pragma unroll
            for (int i = 0; i < VV; ++i)
                rv[i] = load16(pv + in_memory(vrow + i * VR, pad) * s.v.moment, vcol, s.N, vrow + i * VR >= pad);
        }
    };
    if (left > 0) fetch(0);

    const float cv = s.backwards ? s.c : 1.f;
    float rest[4];                                        // the decay from a 16-row block's row to its end, times c''
#pragma unroll
    for (int r = 0; r < 4; ++r) rest[r] = cv * power(16 - 4 * g - r);
    const float cz = s.backwards ? 1.f : s.c;
    const float p16 = shared_by_all(power(16)), p32 = shared_by_all(power(32)), p48 = shared_by_all(power(48));
    auto blocks = [&](int i) { return i == 0 ? 1.f : i == 1 ? p16 : i == 2 ? p32 : p48; };
    Keep keep(ld * CH);                                   // over a whole chunk
    keep.one = shared_by_all(keep.one);
    keep.f = shared_by_all(keep.f);
    char* const out = OUT ? (char*)s.out : nullptr;
    const int size = s.wide ? 4 : (int)sizeof(T);
    const long long out_first = a.starts ? 0 : n * a.n_moments;
    const int so_ = a.heads * s.N * size, oc = w0 + 4 * NT * g;
    const int xto = place<KW>(xrow, xcol >> 3) + (xcol & 7), vto = place<NW>(vrow, vcol >> 3) + (vcol & 7);
    const int xat = place<KW>(c, g), yat = place<KW>(4 * g + (c >> 2), c & 3);
    const bf16* const vdown = sv + (NT == 2 ? place<NW>(4 * g + (c >> 2), 4 * wave + (c & 3))
                                            : place<NW>(4 * g + (c >> 2), 2 * wave + (c >> 1 & 1)) + 4 * (c & 1));
    if (OUT)                                              // the pieces' blocks above the diagonal: zeros for good
        for (int i = tid; i < W * 64; i += 64 * WAVES) {
            reinterpret_cast<bf16x4*>(&sp[0][0][i])[1] = bf16x4{};
            if (PIECES == 6) reinterpret_cast<bf16x4*>(&sp[4][0][i])[1] = bf16x4{};
        }

    for (long long i0 = 0; i0 < left; i0 += CH) {
        const int rows = rows_from(i0), pad = CH - rows;
        __syncthreads();                                  // (the chunk before is read)
#pragma unroll
        for (int i = 0; i < XV; ++i) {
            // (a row 16 on has its shares in the same order)
            const int to = XR % 16 ? place<KW>(xrow + i * XR, xcol >> 3) + (xcol & 7) : xto + i * XR * KW;
            if (OUT) store_terms<T>(rx[i], sx + to, XP);
            store_terms<T>(ry[i], sy + to, XP);
        }
#pragma unroll
        for (int i = 0; i < VV; ++i) {
            const int to = VR % 16 ? place<NW>(vrow + i * VR, vcol >> 3) + (vcol & 7) : vto + i * VR * NW;
            store_terms<T>(rv[i], sv + to, VP);
        }
        __syncthreads();

        f32x4 o[JB][NT];
        if (OUT && out) {
            // the weights' 16 x 16 blocks, rows j, columns i >= j; two of rows 32 jj .. make a piece: (jj, i) = (0, 0) (0, 1)
            // (0, 2) (0, 3) (1, 2) (1, 3)
            for (int block = wave; block < JB * (JB + 1) / 2; block += WAVES) {
                const int i = block < 1 ? 0 : block < 3 ? 1 : block < 6 ? 2 : 3, j = block - i * (i + 1) / 2;
                const int d0 = here(16 * (i - j) + c - 4 * g);
                f32x4 p;
#pragma unroll
                for (int b = 0; b < KT; ++b) {
                    const int at = here(xat) ^ 32 * b;
                    p = mfma(across<X>(sy + 16 * j * KW + at, XP), across<X>(sx + 16 * i * KW + at, XP),
                             b ? p : f32x4{0.f, 0.f, 0.f, 0.f});
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float f = s.c * power(max(d0 - r, 0));
                    p[r] = d0 >= r ? f * p[r] : 0.f;      // (whatever x . y is there)
                }
                Sum<W, 4> w;
                w.of_summed(p);
#pragma unroll
                for (int t = 0; t < W; ++t) reinterpret_cast<bf16x4*>(&sp[j < 2 ? i : i + 2][t][lane])[j & 1] = w.term[t];
            }
#pragma unroll
            for (int b = 0; b < KT; ++b) {
                Sum<W, 8> zf[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    zf[t].of_summed(__builtin_shufflevector(z[2 * b][t], z[2 * b + 1][t], 0, 1, 2, 3, 4, 5, 6, 7));
                const int at = here(xat) ^ 32 * b;
#pragma unroll
                for (int i = 0; i < JB; ++i) {
                    const Sum<X, 8> xf = across<X>(sx + 16 * i * KW + at, XP);
#pragma unroll
                    for (int t = 0; t < NT; ++t) o[i][t] = mfma(zf[t], xf, b ? o[i][t] : f32x4{0.f, 0.f, 0.f, 0.f});
                }
            }
            float f[JB];
            if (pad) {
                const int c1 = here(c) - pad;
#pragma unroll
                for (int i = 0; i < JB; ++i) f[i] = cz * power(max(16 * i + c1, 0));
            } else {
                const float f0 = cz * power(here(c));
#pragma unroll
                for (int i = 0; i < JB; ++i) f[i] = f0 * blocks(i);
            }
#pragma unroll
            for (int i = 0; i < JB; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[i][t][r] *= f[i];
        }
        // (the next chunk on its way from here: earlier, its registers push the products' operands out)
        if (i0 + CH < left) fetch(i0 + CH);
        // the state after the chunk; of the stretch's last one forwards, S rather than l S
        const bool ends = last && i0 + CH >= left;
        if (!ends || s.fin) {
            if (ends) {
                const int early = s.backwards ? 0 : 1;
                const Keep k(ld * (float)(CH - pad - early));
                keep.one = shared_by_all(k.one);
                keep.f = shared_by_all(k.f);
#pragma unroll
                for (int r = 0; r < 4; ++r) rest[r] = cv * power(16 - 4 * g - r - early);
            }
            if (keep.one != 0.f && keep.f != 0.f) {           // (one instruction a value, either way)
#pragma unroll
                for (int b = 0; b < 2 * KT; ++b)
#pragma unroll
                    for (int r = 0; r < 4 * NT; ++r) z[b][r >> 2][r & 3] = fmaf(keep.f, z[b][r >> 2][r & 3], z[b][r >> 2][r & 3]);
            } else {
#pragma unroll
                for (int b = 0; b < 2 * KT; ++b)
#pragma unroll
                    for (int r = 0; r < 4 * NT; ++r) z[b][r >> 2][r & 3] *= keep.one + keep.f;       // (one of them is 0)
            }
#pragma unroll
            for (int jj = 0; jj < JB / 2; ++jj) {
                Sum<S_TERMS, 8> w[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const Sum<X, 8> vf = down<X>(vdown + 32 * jj * NW + 4 * t, 16 * NW, VP);
                    f32x8 v = __builtin_convertvector(vf.term[X - 1], f32x8);
#pragma unroll
                    for (int p = X - 2; p >= 0; --p) v += __builtin_convertvector(vf.term[p], f32x8);
#pragma unroll
                    for (int r = 0; r < 8; ++r) v[r] *= rest[r & 3] * blocks(JB - 1 - 2 * jj - (r >> 2));
                    w[t].of_summed(v);
                }
#pragma unroll
                for (int b = 0; b < 2 * KT; ++b) {
                    const bf16* p = sy + 32 * jj * KW + (here(yat) ^ 32 * (b >> 1)) + 4 * (b & 1);
                    const Sum<X, 8> yt = down<X>(p, 16 * KW, XP);
#pragma unroll
                    for (int t = 0; t < NT; ++t) z[b][t] = mfma(yt, w[t], z[b][t]);
                }
            }
        }
        if (OUT && out) {
            __syncthreads();                              // (the weights' pieces are there, long since: the state came between)
            float odd = 0.f;                              // (0 times what is not finite is NaN)
            unsigned none = 0;
            asm("" : "+s"(none));
#pragma unroll
            for (int jj = 0; jj < JB / 2; ++jj) {
                Sum<X, 8> vf[NT];
                float bad = 0.f;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    vf[t] = down<X>(vdown + 32 * jj * NW + 4 * t, 16 * NW, VP);
#pragma unroll
                    for (int r = 0; r < 8; r += 2)
                        bad = __builtin_amdgcn_fdot2_f32_bf16(Sum<1, 8>::pair(vf[t].term[0], r), __builtin_bit_cast(bf16x2, none), bad, false);
                }
                odd += bad;
                if (__ballot(!(bad == 0.f)))
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int r = 0; r < 8; ++r)
                            if (!(fabsf((float)vf[t].term[0][r]) < INFINITY))
#pragma unroll
                                for (int p = 0; p < X; ++p) vf[t].term[p][r] = (bf16)0.f;
#pragma unroll
                for (int i = 2 * jj; i < JB; ++i) {
                    Sum<W, 8> w;
#pragma unroll
                    for (int t = 0; t < W; ++t) w.term[t] = sp[jj ? i + 2 : i][t][lane];
#pragma unroll
                    for (int t = 0; t < NT; ++t) o[i][t] = mfma(vf[t], w, o[i][t]);
                }
            }
            if (__ballot(!(odd == 0.f))) {
                const int g4 = here(4 * g), c1 = here(c);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    int since = CH;                       // the first row of the lane's column that is not finite
#pragma unroll
                    for (int jj = 0; jj < JB / 2; ++jj) {
                        const bf16x8 v = columns8(vdown + 32 * jj * NW + 4 * t, 16 * NW);
#pragma unroll
                        for (int r = 0; r < 8; ++r)
                            if (!(fabsf((float)v[r]) < INFINITY))
                                since = min(since, 32 * jj + 16 * (r >> 2) + g4 + (r & 3));
                    }
                    since = min(since, __shfl_xor(since, 16));
                    since = min(since, __shfl_xor(since, 32));
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int f = __shfl(since, g4 + r);
#pragma unroll
                        for (int i = 0; i < JB; ++i)
                            if (16 * i + c1 >= f) o[i][t][r] = NAN;
                    }
                }
            }
            char* const po = out + ((out_first + lowest(i0, rows)) * a.heads + h) * s.N * size;
            if constexpr (VEC) {
                const auto bo = rows_at(po, rows, so_, s.N * size);
                const int c1 = here(c), oc1 = here(oc);
                // (a row before the first, or past the last, is outside)
                const unsigned at = oc1 < s.N ? in_memory(c1, pad) * so_ + oc1 * size : NOWHERE;
#pragma unroll
                for (int i = 0; i < JB; ++i) {
                    const unsigned to = at + 16 * i * row_sign * so_;
                    if (sizeof(T) == 4 || s.wide) {
#pragma unroll
                        for (int t = 0; t < NT; ++t)      // (columns past the row's end would be the next one's)
                            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o[i][t]), bo,
                                                                   oc1 + 4 * t < s.N ? to + 16 * t : NOWHERE, 0, 0);
                    } else if constexpr (sizeof(T) == 2) {
                        typedef T vec __attribute__((ext_vector_type(4)));
                        vec v[NT];
#pragma unroll
                        for (int t = 0; t < NT; ++t) v[t] = __builtin_convertvector(o[i][t], vec);
                        if constexpr (NT == 2) {
                            const auto both = __builtin_shufflevector(v[0], v[NT - 1], 0, 1, 2, 3, 4, 5, 6, 7);
                            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, both), bo, to, 0, 0);
                        } else {
                            __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, v[0]), bo, to, 0, 0);
                        }
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < JB; ++i) {
                    if (16 * i + c < pad) continue;
                    char* to = po + (long long)in_memory(16 * i + c, pad) * so_ + oc * size;
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            if (oc + 4 * t + r >= s.N) continue;
                            if (s.wide) reinterpret_cast<float*>(to)[4 * t + r] = o[i][t][r];
                            else reinterpret_cast<T*>(to)[4 * t + r] = narrow<T>(o[i][t][r]);
                        }
                }
            }
        }
    }

    float* to = !OUT ? s.seg + ((size_t)slot * a.heads + h) * s.K * s.N : last && s.fin ? s.fin + at : nullptr;
    if (to) {
        const int k0 = here(8 * g);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int c0 = here(col_of(t, c));
            if (c0 < s.N)
#pragma unroll
                for (int b = 0; b < 2 * KT; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int k = k0 + 32 * (b >> 1) + 4 * (b & 1) + r;
                        if (k < s.K) to[k * s.N + c0] = z[b][t][r];
                    }
        }
    }
}

// Segments' start states from their own: Z_0 = the stretch's, Z_{s+1} = l^L Z_s + own_s, in place; 4 values a lane (K x N a
// multiple of 4) or one.  A value's chain is as long as its segments are many, so 16 of them are under way at once.
// grid (blocks of values x heads, stretches, scans)
template <int V>
__global__ __launch_bounds__(256) void k_scan_join(Scans a) {
    typedef float vec __attribute__((ext_vector_type(V)));
    const Scan& s = a.s[blockIdx.z];
    const int h = blockIdx.x % a.heads, n = blockIdx.y, i = (blockIdx.x / a.heads * 256 + threadIdx.x) * V;
    long long first, count;
    stretch_of(a, n, first, count);
    if (i >= s.K * s.N || !count) return;                 // (without moments there are no segments)
    const float ld = log_decay_of(a, h);
    const Keep once(ld), keep(ld * (float)a.L), keep0(ld * (float)a.L0);
    vec z;
#pragma unroll
    for (int j = 0; j < V; ++j)
        z[j] = start_value(s, ((size_t)n * a.heads + h) * s.K * s.N, (i + j) / s.N, (i + j) % s.N, once);
    const size_t step = (size_t)a.heads * s.K * s.N;
    float* p = s.seg + ((size_t)first_slot(a, n, first) * a.heads + h) * s.K * s.N + i;
    constexpr int AHEAD = 16;                             // segments' states under way at once
    auto walk = [&](auto plain) {                         // (the other kind's tests, for all: 16.6 us instead of 15.0)
        for (long long first_of = 0; !first_of || start_of(a, first_of) < count; first_of += AHEAD, p += AHEAD * step) {
            vec own[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
                if (start_of(a, first_of + j + 1) < count) own[j] = *reinterpret_cast<const vec*>(p + j * step);
                else own[j] = (vec)0.f;
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                if (j && start_of(a, first_of + j) >= count) return;
                *reinterpret_cast<vec*>(p + j * step) = z;
                const Keep& over = first_of + j ? keep : keep0;
#pragma unroll
                for (int e = 0; e < V; ++e) z[e] = (plain.value ? over.times(z[e]) : over(z[e])) + own[j][e];
            }
        }
    };
    if (keep.plain() && keep0.plain()) walk(std::true_type{});
    else walk(std::false_type{});
}

// gradients of shared heads: out[m][j][d] = the sum over a key head's `share` query heads of part[m][share j + i][d]; the
// first `first` workgroups those of k, the rest those of v
template <class T>
__global__ __launch_bounds__(256) void k_share(const float* part_k, T* out_k, int K, long long nk, long long first,
                                               const float* part_v, T* out_v, int V, long long nv, int share) {
    const long long block = block_number();
    const bool of_v = block >= first;
    const float* part = of_v ? part_v : part_k;
    T* out = of_v ? out_v : out_k;
    const int D = of_v ? V : K;
    const long long i = (block - (of_v ? first : 0)) * 256 + threadIdx.x, row = i / D;
    if (i >= (of_v ? nv : nk)) return;
    const int d = (int)(i - row * D);
    float s = 0.f;
    for (int j = 0; j < share; ++j) s += part[(row * share + j) * D + d];
    out[i] = narrow<T>(s);
}

// moments of no stretch at all
template <class T>
__global__ __launch_bounds__(256) void k_zeros(T* out, long long n) {
    const long long i = block_number() * 256 + threadIdx.x;
    if (i < n) out[i] = (T)0.f;
}

// One moment: a workgroup takes CB columns of a row's state of one head, CB / 4 lanes a row of it, every (1024 / CB)th row a
// lane, all a lane's loads under way at once; the lanes' shares of q S are joined over rows by shuffles, then in LDS.
// VEC: 16-byte loads and stores of the states (v_dim a multiple of 4, states aligned).
// grid (blocks of columns, heads, rows)
template <class T, int CB, bool VEC>
__global__ __launch_bounds__(256) void k_step(fm_step_args a) {
    constexpr int LR = CB / 4, RG = 256 / LR, ROWS = ATT_MAX / RG;
    __shared__ float part[4][CB];
    const int tid = threadIdx.x, cg = tid % LR, rg = tid / LR, h = blockIdx.y, K = (int)a.k_dim, N = (int)a.v_dim;
    const int c0 = blockIdx.x * CB + 4 * cg;
    const long long n = blockIdx.z, slot = a.slots ? a.slots[n] : n;
    T* o = (T*)a.o + (n * a.q_heads + h) * N + blockIdx.x * CB;
    const int cols = min(CB, N - (int)blockIdx.x * CB);
    if (slot < 0 || slot >= a.n_states) {
        if (tid < cols) o[tid] = narrow<T>(slot < 0 ? 0.f : NAN);
        return;
    }
    const int hk = h / (int)(a.q_heads / a.k_heads);
    const T* q = (const T*)a.q.data + n * a.q.seq + h * a.q.head;
    const T* k = (const T*)a.k.data + n * a.k.seq + hk * a.k.head;
    const T* v = (const T*)a.v.data + n * a.v.seq + hk * a.v.head;
    const size_t at = ((size_t)slot * a.q_heads + h) * K * N;
    float4 s[ROWS];
    float kr[ROWS], qr[ROWS], vv[4];
    auto load = [&](const float* p) {
        if (VEC) return c0 < N ? *reinterpret_cast<const float4*>(p + c0) : make_float4(0.f, 0.f, 0.f, 0.f);
        return make_float4(c0 < N ? p[c0] : 0.f, c0 + 1 < N ? p[c0 + 1] : 0.f, c0 + 2 < N ? p[c0 + 2] : 0.f,
                           c0 + 3 < N ? p[c0 + 3] : 0.f);
    };
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = rg + i * RG;
        s[i] = r < K ? load(a.state + at + (size_t)r * N) : make_float4(0.f, 0.f, 0.f, 0.f);
        kr[i] = r < K ? widen(k[r]) : 0.f;
        qr[i] = r < K ? widen(q[r]) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) vv[j] = c0 + j < N ? widen(v[c0 + j]) : 0.f;
    const Keep keep(a.log_decay[h]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = rg + i * RG;
        if (r >= K) break;
        s[i] = make_float4(fmaf(kr[i], vv[0], keep(s[i].x)), fmaf(kr[i], vv[1], keep(s[i].y)),
                           fmaf(kr[i], vv[2], keep(s[i].z)), fmaf(kr[i], vv[3], keep(s[i].w)));
        float* p = a.next + at + (size_t)r * N + c0;
        if (VEC) {
            if (c0 < N) *reinterpret_cast<float4*>(p) = s[i];
        } else {
            if (c0 < N) p[0] = s[i].x;
            if (c0 + 1 < N) p[1] = s[i].y;
            if (c0 + 2 < N) p[2] = s[i].z;
            if (c0 + 3 < N) p[3] = s[i].w;
        }
        fma4(qr[i], s[i], acc);
    }
#pragma unroll
    for (int m = LR; m < 64; m <<= 1) {
        acc.x += __shfl_xor(acc.x, m);
        acc.y += __shfl_xor(acc.y, m);
        acc.z += __shfl_xor(acc.z, m);
        acc.w += __shfl_xor(acc.w, m);
    }
    if ((tid & 63) < LR) *reinterpret_cast<float4*>(&part[tid >> 6][4 * cg]) = acc;
    __syncthreads();
    if (tid < cols) o[tid] = narrow<T>((float)a.scale * (part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid]));
}

// ------------------------------------------------------------------------------------------------ host
const char* heads_wrong(long long dtype, long long qh, long long kh, long long kd, long long vd) {
    if (dtype < FM_F32 || dtype > FM_F16) return "values of an unknown type";
    if (qh < 1 || kh < 1 || qh % kh || qh > 65535) return "query heads must be a multiple of key heads, at most 65535";
    if (kd < 1 || kd > ATT_MAX || vd < 1 || vd > ATT_MAX) return "heads of other than 1 to 128 values";
    return nullptr;
}

// two arrays of n floats share memory
bool overlap(const float* a, const float* b, long long n) {
    return a && b && (uintptr_t)a < (uintptr_t)b + 4 * n && (uintptr_t)b < (uintptr_t)a + 4 * n;
}

const char* attention_wrong(const fm_attention_args& a, bool bwd, bool sizes_only = false) {
    if (const char* e = heads_wrong(a.dtype, a.q_heads, a.k_heads, a.k_dim, a.v_dim)) return e;
    if (a.n_seq < 0 || a.n_seq > 16384) return "other than 0 to 16384 stretches";
    if (a.n_moments < 0 || a.n_moments > 1LL << 31) return "other than 0 to 2^31 moments";
    if (sizes_only) return nullptr;
    if (!a.log_decay) return "no decays";
    const bool any = a.n_seq && a.n_moments;
    if (any && (!a.q.data || !a.k.data || !a.v.data)) return "a null tensor";
    if (!bwd && a.n_moments && (a.n_seq || a.starts) && !a.o) return "a null tensor";
    if (!bwd && overlap(a.state, a.state_out, a.n_seq * a.q_heads * a.k_dim * a.v_dim)) return "state_out must not be state";
    if (bwd && any && !a.go.data) return "a null tensor";
    return nullptr;
}

// float32 partial gradients of shared key / value heads
long long shared_floats(const fm_attention_args& a, bool of_v) {
    const long long moments = a.n_moments * (a.starts ? 1 : a.n_seq);
    return a.q_heads > a.k_heads ? moments * a.q_heads * (of_v ? a.v_dim : a.k_dim) : 0;
}

// The kernel's forms by the products' sizes: K up to 64 or 128 rows of state; N up to 64 columns, a block of 16 a wave, or up
// to 128, two blocks a wave (a wave's reads of x and y then serve two: at N = 128, one block and 8 waves measured the same
// within 1%, and 4 waves in two workgroups 6% more).
template <class T, int KT, int NT>
constexpr int groups_per_cu() { return Tile<T, KT, NT, true>::PER_SIMD; }
template <class T>
int groups_per_cu(int K, int N) {
    return K <= 64 ? (N <= 64 ? groups_per_cu<T, 2, 1>() : groups_per_cu<T, 2, 2>())
                   : (N <= 64 ? groups_per_cu<T, 4, 1>() : groups_per_cu<T, 4, 2>());
}

// How a launch's scans are cut into segments: as the following estimate (us) has it cheapest.  A CU with w workgroups takes
// 1.7 + b w (3 + K N / 1024) for a chunk of each, K and N as the kernel's form has them, b = 0.207 for bfloat16 (64 moments a
// chunk), 0.147 for binary16, 0.257 for float32 (32); the longest workgroup ends alone.  More than one segment a stretch cost
// a pass for their own states (0.55 of the constant, 0.2 of the rest; a stretch's last segment needs none), its launch, and
// the joining's traffic.  Packed stretches, whose lengths only the device knows, are taken to be of any length up to twice the
// middle one.  (264 packs, all alike, of any length up to twice the middle, with one six times as long, or of exponential
// lengths, a quarter each: against twice, 1.5 times takes 2% more, 2.5 and 3 times 2% less, but up to 47% more where all are
// alike, 6 times the same.)  Fitted to 550 measured times (13% rms): 15 sets of stretches of one or of mixed lengths, forward
// and gradient, 5 to 12 cuts of each.  The cut so chosen takes 5% (rms) more than the best of them where the host knows the
// lengths, 6% where packed ones are mixed, 20% where packed ones are all the same, 15% where one of them is four times the
// others.
struct Cut {
    int nseg, slots, K, N, joined;
    long long L, L0;
};
// From this many values of a chain's segments up they are joined by a kernel of its own; fewer, each segment of the main pass
// joins those before it as it begins (a launch less).  150 sets of stretches, alike and packed, states of 16 x 16 to 128 x
// 128, forward and gradient: from 32,768 values up takes 0.5% more in the mean, from 98,304 2.5%, from 196,608 8%, always the
// kernel 0.5% (small states prefer it, up to 1.45 times as fast; short packs the other way, 2.4 times), never the kernel 24%.
constexpr int JOIN_FROM = 49152;
Cut cut_of(const fm_attention_args& p, int scans) {
    Cut c;
    const int widest = (int)(p.k_dim > p.v_dim ? p.k_dim : p.v_dim);
    c.K = scans == 1 ? (int)p.k_dim : widest;             // (a gradient's scans have them both ways round)
    c.N = scans == 1 ? (int)p.v_dim : widest;
    c.nseg = 1;
    c.joined = 0;
    c.slots = (int)p.n_seq;
    c.L = (p.n_moments + CHUNK_MAX - 1) / CHUNK_MAX * CHUNK_MAX;
    if (!c.L) c.L = CHUNK_MAX;
    c.L0 = c.L;
    if (!p.n_seq || !p.n_moments) return c;
    const int cap = p.dtype == FM_F32 ? groups_per_cu<float>(c.K, c.N) : p.dtype == FM_BF16 ? groups_per_cu<bf16>(c.K, c.N)
                                                                                            : groups_per_cu<f16>(c.K, c.N);
    const int chunk = p.dtype == FM_BF16 ? Form<bf16>::CHUNK : Form<float>::CHUNK;
    const double one = (p.dtype == FM_BF16 ? 0.207 : p.dtype == FM_F16 ? 0.147 : 0.257) *
                       (3 + (c.K <= 64 ? 1 : 2) * (c.N <= 64 ? 1 : 2) * 4.0);
    const bool packed = p.starts && p.n_seq > 1;
    const double middle = (double)p.n_moments / (packed ? p.n_seq : 1), longest = packed ? 2 * middle : middle;
    const double chains = (double)p.n_seq * p.q_heads * scans;
    // each, most: moments of a group in the middle, of the longest
    auto pass = [&](double groups, double each, double most, double a, double b) {
        double left = groups / 256, t = 0;
        if (left <= 0) return 0.0;
        for (; left > 0; left -= cap) {
            if (left > 64 * cap) {                        // (many rounds: each full)
                t += (a + b * cap) * left / cap;
                break;
            }
            t += a + b * (left < cap ? ceil(left) : cap);
        }
        return t * (each / chunk + 0.3) + (a + b) * (most - each) / chunk;
    };
    double best = 0.95 * pass(chains, middle, longest, 1.7, one);     // (whole where it is about the same)
    for (int nseg = 2; nseg <= 1024; nseg += nseg < 4 ? 1 : nseg / 2) {
        const long long L = ((long long)ceil(longest / nseg) + CHUNK_MAX - 1) / CHUNK_MAX * CHUNK_MAX;
        if (L >= longest) continue;
        const double each = packed ? middle / L + 0.5 : ceil(middle / L), states = chains * each * c.K * c.N * 4;
        const int joined = ceil(longest / L) * c.K * c.N >= JOIN_FROM;
        const double t = pass(chains * each, packed ? middle / each : (double)L, (double)L, 1.7, one) +
                         pass(chains * (each - 1), (double)L, (double)L, 0.55 * 1.7, 0.2 * one) +
                         (joined ? 28 + states * 2 / 5.7e6 : 14 + states * (each - 1) / 2 / 5.7e6);
        if (t < best) {
            best = t;
            c.L = L;
            c.nseg = nseg;
            c.joined = joined;
        }
        if (L == CHUNK_MAX) break;
    }
    // a packed launch that is best left whole cuts stretches past 8 times the middle all the same: that costs the others up to
    // 7 us, and spares one long stretch among many from being walked alone
    if (packed && c.nseg == 1 && p.n_seq > 8) {
        c.L = ((long long)ceil(8 * middle) + CHUNK_MAX - 1) / CHUNK_MAX * CHUNK_MAX;
        c.joined = 0;
    }
    c.nseg = (int)((p.n_moments + c.L - 1) / c.L);
    c.L0 = c.L;
    // More chains than half the workgroups that fit, but not all of them: a first segment so short that those left over, one
    // after another, walk the first segments while the chains' workgroups walk the rest.  (84 such sets, 55 to 92% of what fits, 700
    // to 6,000 moments of each type: gradients take 2.4% less in the mean, 15% less at best, 12 x 2048 moments of 8 heads of 128
    // float32 values 600 -> 508 us, and 6% more at worst, 12 x 700 in binary16 156 -> 166.)
    const double fit = 256.0 * cap;
    if (!p.starts && chains < fit && 2 * chains > fit) {      // (packed stretches find their segments by L alone)
        const double turns = ceil(chains / (fit - chains));
        const long long L0 = (long long)(middle / (1 + turns)) / CHUNK_MAX * CHUNK_MAX;
        const double rest = middle - L0, states = chains * c.K * c.N * 8;
        const double t = (1.7 + one * cap) * (fmax(rest, turns * L0) / chunk + 0.3 * (1 + turns)) +
                         pass(chains, (double)L0, (double)L0, 0.55 * 1.7, 0.2 * one) + 14 + states / 2 / 5.7e6;
        if (L0 && t < best) {
            c.L0 = L0;
            c.L = (p.n_moments - L0 + CHUNK_MAX - 1) / CHUNK_MAX * CHUNK_MAX;
            c.nseg = 2;
            c.joined = 0;
        }
    }
    if (c.nseg > 1) c.slots = p.starts ? (int)(p.n_moments / c.L + p.n_seq) : (int)p.n_seq * c.nseg;
    return c;
}
// floats of segments' states of one scan
long long segment_floats(const fm_attention_args& p, const Cut& c) {
    return c.nseg == 1 ? 0 : (long long)c.slots * p.q_heads * p.k_dim * p.v_dim;
}

constexpr int CLEARING = 256;            // workgroups of a packed launch that clear: one a CU
template <class T, int KT, int NT, bool VEC>
void launch_form(Scans& a, int count, hipStream_t st) {
    int most = 1;
    for (int i = 0; i < count; ++i) most = a.s[i].K * a.s[i].N > most ? a.s[i].K * a.s[i].N : most;
    const dim3 grid = blocks_of((long long)a.slots * a.heads * count);
    a.scans = count;
    a.clearing = a.starts ? (CLEARING + a.heads * count - 1) / (a.heads * count) : 0;
    if (a.nseg > 1) {
        k_scan<T, KT, NT, VEC, false><<<grid, 64 * WAVES, 0, st>>>(a);
        auto blocks = [&](int v) { return dim3((most / v + 255) / 256 * a.heads, a.n_seq, count); };
        if (a.joined && most % 4 == 0) k_scan_join<4><<<blocks(4), 256, 0, st>>>(a);
        else if (a.joined) k_scan_join<1><<<blocks(1), 256, 0, st>>>(a);
    }
    k_scan<T, KT, NT, VEC, true><<<blocks_of((long long)(a.slots + a.clearing) * a.heads * count), 64 * WAVES, 0, st>>>(a);
}
template <class T, bool VEC>
void launch_sized(Scans& a, int count, const Cut& c, hipStream_t st) {
    if (c.K <= 64) c.N <= 64 ? launch_form<T, 2, 1, VEC>(a, count, st) : launch_form<T, 2, 2, VEC>(a, count, st);
    else c.N <= 64 ? launch_form<T, 4, 1, VEC>(a, count, st) : launch_form<T, 4, 2, VEC>(a, count, st);
}

template <class T>
void launch_scans(Scans& a, int count, const Cut& cut, bool vec, hipStream_t st) {
    if (!a.n_seq || !count) return;
    a.L = cut.L;
    a.L0 = cut.L0;
    a.nseg = cut.nseg;
    a.slots = cut.slots;
    a.joined = cut.joined;
    vec ? launch_sized<T, true>(a, count, cut, st) : launch_sized<T, false>(a, count, cut, st);
}

Scans scans_of(const fm_attention_args& p) {
    Scans a{};
    a.log_decay = p.log_decay;
    a.starts = p.starts;
    a.n_moments = p.n_moments;
    a.wide = (int)p.wide;
    a.heads = (int)p.q_heads;
    a.n_seq = (int)p.n_seq;
    return a;
}

// 16-byte loads, whole stores: heads of a multiple of 16 bytes, everything aligned, a chunk's rows within 2^30 bytes
bool wide_rows(const fm_attention_args& p, bool bwd) {
    const int size = p.dtype == FM_F32 ? 4 : 2;
    if (p.k_dim * size % 16 || p.v_dim * size % 16) return false;
    if (!aligned16(p.q, size) || !aligned16(p.k, size) || !aligned16(p.v, size)) return false;
    auto near = [](long long s) { return s >= 0 && s < STRIDE_MOST; };
    if (!near(p.q.moment) || !near(p.k.moment) || !near(p.v.moment) || !near(p.q_heads * ATT_MAX)) return false;
    if (!bwd) return !((uintptr_t)p.o & 15);
    return near(p.go.moment) && aligned16(p.go, size) &&
           !(((uintptr_t)p.gq | (uintptr_t)p.gk | (uintptr_t)p.gv | (uintptr_t)p.workspace) & 15);
}

template <class T>
void zeros(void* out, long long n, hipStream_t st) {
    if (out && n) k_zeros<T><<<blocks_of((n + 255) / 256), 256, 0, st>>>((T*)out, n);
}

template <class T>
void attention_fwd(const fm_attention_args& p, hipStream_t st) {
    const int share = (int)(p.q_heads / p.k_heads);
    if (p.starts && !p.n_seq) {
        zeros<T>(p.o, p.n_moments * p.q_heads * p.v_dim, st);
        return;
    }
    Scans a = scans_of(p);
    const Cut cut = cut_of(p, 1);
    float* seg = segment_floats(p, cut) ? (float*)p.workspace : nullptr;
    a.s[0] = Scan{p.q, p.k, p.v, 1, share, share, p.o, p.state, p.state_out, seg, (int)p.k_dim, (int)p.v_dim, 0, 0, 0,
                  (float)p.scale};
    launch_scans<T>(a, 1, cut, wide_rows(p, false), st);
}

template <class T>
void attention_bwd(const fm_attention_args& p, hipStream_t st) {
    const int share = (int)(p.q_heads / p.k_heads), K = (int)p.k_dim, V = (int)p.v_dim;
    const float c = (float)p.scale;
    if (p.starts && !p.n_seq) {
        zeros<T>(p.gq, p.n_moments * p.q_heads * K, st);
        zeros<T>(p.gk, p.n_moments * p.k_heads * K, st);
        zeros<T>(p.gv, p.n_moments * p.k_heads * V, st);
        return;
    }
    const Cut cut = cut_of(p, 3);
    const long long floats = segment_floats(p, cut);
    float* seg[3];
    for (int i = 0; i < 3; ++i) seg[i] = floats ? (float*)p.workspace + i * floats : nullptr;
    // shared key / value heads: each query head's part in float32, then their sum
    float* part_k = (float*)p.workspace + 3 * floats;
    float* part_v = part_k + shared_floats(p, false);
    const int part = share > 1;
    Scans a = scans_of(p);
    int n = 0;
    if (p.gq) a.s[n++] = Scan{p.go, p.v, p.k, 1, share, share, p.gq, p.state, nullptr, seg[0], V, K, 1, 0, 0, c};
    if (p.gk) a.s[n++] = Scan{p.v, p.go, p.q, share, 1, 1, part ? part_k : p.gk, p.gstate_out, nullptr, seg[1], V, K, 1, 1, part, c};
    if (p.gv || p.gstate)
        a.s[n++] = Scan{p.k, p.q, p.go, share, 1, 1, part && p.gv ? part_v : p.gv, p.gstate_out, p.gstate, seg[2], K, V, 0, 1, part, c};
    launch_scans<T>(a, n, cut, wide_rows(p, true), st);
    if (!part) return;
    const long long rows = p.n_moments * (p.starts ? 1 : p.n_seq) * p.k_heads;
    const long long nk = p.gk ? rows * K : 0, nv = p.gv ? rows * V : 0;
    const long long bk = (nk + 255) / 256, bv = (nv + 255) / 256;
    if (bk + bv) k_share<T><<<blocks_of(bk + bv), 256, 0, st>>>(part_k, (T*)p.gk, K, nk, bk, part_v, (T*)p.gv, V, nv, share);
}

// 32 columns a workgroup: 416 rows of 8 states of 128 x 128, 90 us with 32 or 64 columns, 101 with 128; one row of 8 states of
// 64 x 64 finds 16 workgroups.
template <class T>
void step_of_type(const fm_step_args& a, hipStream_t st) {
    constexpr int CB = 32;
    const dim3 grid((unsigned)((a.v_dim + CB - 1) / CB), (unsigned)a.q_heads, (unsigned)a.n);
    if (a.v_dim % 4 || (((uintptr_t)a.state | (uintptr_t)a.next) & 15)) k_step<T, CB, false><<<grid, 256, 0, st>>>(a);
    else k_step<T, CB, true><<<grid, 256, 0, st>>>(a);
}

}  // namespace fg

using namespace fg;

extern "C" {

long long fm_attention_workspace(const fm_attention_args* a, int backward) {
    if (!a || attention_wrong(*a, false, true)) return 0;
    const Cut cut = cut_of(*a, backward ? 3 : 1);
    return 4 * (segment_floats(*a, cut) * (backward ? 3 : 1) + (backward ? shared_floats(*a, false) + shared_floats(*a, true) : 0));
}

int fm_attention(const fm_attention_args* a, void* stream) {
    clear_error();
    if (!a) return fail("fm_attention: no arguments");
    if (const char* e = attention_wrong(*a, false)) return fail((std::string("fm_attention: ") + e).c_str());
    const long long need = fm_attention_workspace(a, 0);
    if (need && (!a->workspace || a->workspace_bytes < need)) return fail("fm_attention: the workspace is too small");
    if (a->dtype == FM_F32) attention_fwd<float>(*a, (hipStream_t)stream);
    else if (a->dtype == FM_BF16) attention_fwd<bf16>(*a, (hipStream_t)stream);
    else attention_fwd<f16>(*a, (hipStream_t)stream);
    FG_CHECK(hipGetLastError(), -1);
    return 0;
}

int fm_attention_bwd(const fm_attention_args* a, void* stream) {
    clear_error();
    if (!a) return fail("fm_attention_bwd: no arguments");
    if (const char* e = attention_wrong(*a, true)) return fail((std::string("fm_attention_bwd: ") + e).c_str());
    const long long need = fm_attention_workspace(a, 1);
    if (need && (!a->workspace || a->workspace_bytes < need)) return fail("fm_attention_bwd: the workspace is too small");
    if (a->dtype == FM_F32) attention_bwd<float>(*a, (hipStream_t)stream);
    else if (a->dtype == FM_BF16) attention_bwd<bf16>(*a, (hipStream_t)stream);
    else attention_bwd<f16>(*a, (hipStream_t)stream);
    FG_CHECK(hipGetLastError(), -1);
    return 0;
}

int fm_step(const fm_step_args* a, void* stream) {
    clear_error();
    if (!a) return fail("fm_step: no arguments");
    if (const char* e = heads_wrong(a->dtype, a->q_heads, a->k_heads, a->k_dim, a->v_dim))
        return fail((std::string("fm_step: ") + e).c_str());
    if (a->n < 0 || a->n > 65535 || a->n_states < 0) return fail("fm_step: other than 0 to 65535 rows");
    if (!a->n) return 0;
    if (!a->q.data || !a->k.data || !a->v.data || !a->log_decay || !a->state || !a->next || !a->o)
        return fail("fm_step: a null tensor");
    if (!a->slots && a->n_states < a->n) return fail("fm_step: fewer states than rows");
    if (a->next != a->state && overlap(a->state, a->next, a->n_states * a->q_heads * a->k_dim * a->v_dim))
        return fail("fm_step: next must be state or lie outside it");
    if (a->dtype == FM_F32) step_of_type<float>(*a, (hipStream_t)stream);
    else if (a->dtype == FM_BF16) step_of_type<bf16>(*a, (hipStream_t)stream);
    else step_of_type<f16>(*a, (hipStream_t)stream);
    FG_CHECK(hipGetLastError(), -1);
    return 0;
}

}  // extern "C"
