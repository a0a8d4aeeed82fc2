// The gated delta rule (include/flyguy_memory.h: fm_delta, fm_delta_bwd, fm_delta_step): a linear memory that moves what it holds
// under a key towards the key's new value.  With a_t = exp(log_decay_t) and a state S [K][V] of each head,
//   e_t = v_t - (a_t S_{t-1})^T k_t,   S_t = a_t S_{t-1} + beta_t k_t e_t^T,   o_t = c S_t^T q_t.
//
// In chunks of C moments, with G_i the sum of a chunk's log decays up to moment i, D_ij = exp(G_i - G_j) for j <= i, E = exp(G),
// F = exp(G_end - G) and S the state before the chunk, the errors solve a triangular system:
//   (I + N) e = v - E K S,  N = strict lower(K K^T D) beta;   with T = (I + N)^-1:
//   e = T (v - E K S),   o = c E Q S + P e,  P = c lower(Q K^T D) beta,   S' = E_end S + K^T (F beta e).
// Backwards, with X the gradient of S' and g that of o:
//   y = T^T (P^T g + beta F K X) (the gradient of v),   X' = E_end X + Q^T (c E g) - K^T (E y),
// and with H = c lower(g e^T) D, Z = -strict lower(y e^T) D:
//   gq = c E g S^T + H beta K,   r = -E y S^T + Z beta K,   w = F e X^T + Z^T K + H^T Q,   gk = r + beta w,   gbeta = k . w,
//   gG = q . gq + k . r - beta gbeta, and at the chunk's end E_end <S, X> + sum_i F_i beta_i k_i . (X e_i) besides; a log decay's
//   gradient is the sum of gG from its moment to the chunk's end.
// (beta_j, exp(-G_j) and a writing k_j stand only together, as do exp(G_i) and a reading q_i or k_i: so one dot product of a
// row with its gradient is the factor's gradient.)
//
// T and P need no state: k_delta_prep makes them for all chunks at once.  k_delta_scan then walks each head's chunks with the
// state in registers, and k_delta_back walks them backwards; k_delta_grads makes the gradients of all chunks at once from the
// states and errors that the two walks leave.
#include <hip/hip_runtime.h>

#include <cmath>

#include "memory_chunk.h"

namespace fg {

constexpr int DELTA_MAX = 128;           // values of a head
constexpr int T_TERMS = 3;               // terms of T, of what it multiplies and of the state: the state is a float32 result

// How stretches are cut (memory_chunk.h): into chunks, and into segments of whole chunks.
struct Cuts {
    const void* starts;
    long long n_moments, L, L0;
    int wide, n_seq, nseg, slots;
};
struct Delta {
    fm_view q, k, v, go;
    const float *log_decay, *beta;
    long long ld_seq, ld_moment, ld_head, be_seq, be_moment, be_head;
    Cuts chunks, segs;
    int heads, share, K, V;
    float c;
    int vec;                             // whole stores: heads of a multiple of 16 bytes, outputs aligned
    // workspace, by chunk slot and head
    char* prep;                          // T and P as the products' operands, then the chunk's factors
    char* turned;                        // the same of their transposes, kept for the gradient (0: not wanted)
    float *states, *errors;              // S before each chunk [KW][VW], e [CH][VW] (0: not kept)
    float *grads, *ys;                   // X after each chunk, y, the same way
    // by segment slot and head: a segment's own end state, then its joined one (backwards: X before it) [KW][VW]; what it makes of the
    // state before it, M with S' = M S + own, and M^T [KW][KW]
    float *own, *trans, *trans_t;
    // whole tensors
    const float* init;
    float* fin;
    void* o;
    const float* gfin;
    float* ginit;
    void *gq, *gk, *gv;                  // gk, gv: of the values' type, or (shared heads) float32 parts of each query head
    float *glog_decay, *gbeta;
};

// Terms (memory_chunk.h: Form): X hold an input exactly; W what makes an output in the values' type alone, 3 all that a float32 result
// depends on (the state, and a decay's and rate's gradients: with 2 of them these were off by 3.6e-6 and 6.4e-6 of their
// size, by 4e-7 in float32's own products).
template <class T, bool BWD = false>
struct DeltaForm {
    static constexpr int X = Form<T>::X, W = BWD ? T_TERMS : Form<T>::W, CH = Form<T>::CHUNK, JB = CH / 16, PIECES = JB == 4 ? 6 : 2;
    // operands in units of 64 lanes x 16 bytes: P's terms, then T's, up to whole loads of a workgroup
    static constexpr int P_UNITS = PIECES * W, T_UNITS = PIECES * T_TERMS, UNITS = (P_UNITS + T_UNITS + 3) / 4 * 4;
    // factors: E_end as 1 + x or x (Keep), the first moment that is not finite (as int), 0; then E, F beta, F, beta and G (high
    // and low part) of each moment
    static constexpr int FACTORS = 4 + 6 * CH;
    static constexpr int PREP = UNITS * 1024 + FACTORS * 4;
};
enum { F_E = 4 };
template <class F>
__device__ __forceinline__ const float* factors_of(const char* prep) {
    return reinterpret_cast<const float*>(prep + F::UNITS * 1024);
}

// piece of rows' block i and the pair jj of summed blocks 2jj, 2jj + 1 of a lower triangular matrix (JB 4: (0,0) (0,1) (0,2)
// (0,3) (1,2) (1,3) as (jj, i)); of its transpose, pair ii and block j: (0,0) (0,1) (1,0) .. (1,3)
__device__ __forceinline__ constexpr int piece_of(int jj, int i) { return jj ? i + 2 : i; }
__device__ __forceinline__ constexpr int tpiece_of(int ii, int j) { return ii ? j + 2 : j; }
// block n of the lower triangle, row by row
__device__ __forceinline__ void block_of(int n, int& i, int& j) {
    i = n < 1 ? 0 : n < 3 ? 1 : n < 6 ? 2 : 3;
    j = n - i * (i + 1) / 2;
}

// ------------------------------------------------------------------------------------------------ a chunk's rows
// rows of a chunk in memory: 16 bytes of row `row` from value `col`; zeros past the rows and columns (whole units: k_delta_pack)
template <class T>
struct Chunk {
    int rows, width, step;
    __amdgpu_buffer_rsrc_t rsrc;
    __device__ __forceinline__ Chunk(const T* data, int rows, long long step, int width)
        : rows(rows), width(width), step((int)step * (int)sizeof(T)),
          rsrc(rows_at(data, rows, step * (int)sizeof(T), (width + Vec<T>::N - 1) / Vec<T>::N * 16)) {}
    __device__ __forceinline__ uint4 operator()(int row, int col) const {
        const unsigned at = row < rows && col < width ? row * step + col * (int)sizeof(T) : NOWHERE;
        return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0));
    }
};
template <class T>
__device__ __forceinline__ Chunk<T> chunk_of(const Delta& a, const fm_view& v, int n, int head, long long moment, int rows, int width) {
    return Chunk<T>((const T*)v.data + (a.chunks.starts ? 0 : n * v.seq) + head * v.head + moment * v.moment, rows, v.moment, width);
}
// a value that is not finite among 16 bytes
template <class T>
__device__ __forceinline__ bool odd16(uint4 r) {
    const typename Vec<T>::type v = __builtin_bit_cast(typename Vec<T>::type, r);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i) s = fmaf(widen(v[i]), 0.f, s);
    return !(s == 0.f);
}
template <int P>
__device__ __forceinline__ f32x8 widened(const Sum<P, 8>& s) {
    f32x8 v = __builtin_convertvector(s.term[P - 1], f32x8);
#pragma unroll
    for (int p = P - 2; p >= 0; --p) v += __builtin_convertvector(s.term[p], f32x8);
    return v;
}
template <int P>
__device__ __forceinline__ f32x4 widened(const bf16* p, int plane) {
    f32x4 v = __builtin_convertvector(*reinterpret_cast<const bf16x4*>(p + (P - 1) * plane), f32x4);
#pragma unroll
    for (int i = P - 2; i >= 0; --i) v += __builtin_convertvector(*reinterpret_cast<const bf16x4*>(p + i * plane), f32x4);
    return v;
}
__device__ __forceinline__ f32x8 joined(f32x4 a, f32x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
// a sum's first terms
template <int W, int P>
__device__ __forceinline__ Sum<W, 8> first_terms(const Sum<P, 8>& s) {
    Sum<W, 8> r;
#pragma unroll
    for (int i = 0; i < W; ++i) r.term[i] = s.term[i];
    return r;
}
// Products of several accumulators with a shared operand, a pair of terms of all of them at a time: an accumulator's next product
// waits for its last one, so that these stand apart.  ROWS: the shared one is the second.
template <bool ROWS, int N, int PA, int PB>
__device__ __forceinline__ void mfmas(f32x4* c, const Sum<PA, 8>* a, const Sum<PB, 8>& b) {
    constexpr int most = PA > PB ? PA : PB;
#pragma unroll
    for (int o = most - 1; o >= 0; --o)
#pragma unroll
        for (int i = 0; i < PA; ++i)
            if (o - i >= 0 && o - i < PB)
#pragma unroll
                for (int n = 0; n < N; ++n)
                    c[n] = ROWS ? mfma(a[n].term[i], b.term[o - i], c[n]) : mfma(b.term[o - i], a[n].term[i], c[n]);
}
// a product of two inputs: all pairs of terms where these are two (binary16: the last is 2^-18 of the product), else mfma's
template <int P>
__device__ __forceinline__ f32x4 mfma_whole(const Sum<P, 8>& a, const Sum<P, 8>& b, f32x4 c) {
    if constexpr (P == 2) c = mfma(a.term[1], b.term[1], c);
    return mfma(a, b, c);
}
__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
// a state times one + f (Keep): one instruction a value, either way
template <int B>
__device__ __forceinline__ void decayed(f32x4 (&z)[B], float one, float f) {
    if (one != 0.f && f != 0.f) {
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) z[b][r] = fmaf(f, z[b][r], z[b][r]);
    } else {
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) z[b][r] *= one + f;       // (one of them is 0)
    }
}
// What stands before it is issued before what follows, vector instructions aside.  A SIMD has one wave here: each part of a chunk
// reads the next part's operands from LDS before its own products, or their wait would be in the open (the compiler reads an
// operand right before its product).
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0x6); }
// (before a loop that uses what was loaded: its first iteration's wait would be every iteration's, for its stores)
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }
constexpr float GONE = -110.f;           // a log decay whose factor is 0 in float32
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }

// Tensors whose heads are not whole, aligned 16-byte units, or whose moments lie far apart, are copied so that they are, with
// zeros at a head's end: all other kernels load units.  grid (workgroups, tensors)
struct Packs {
    fm_view from[3];
    void* to[3];
    int heads[3], width[3];
    long long moments, n_moments;        // all; of a stretch
};
template <class T>
__global__ __launch_bounds__(256) void k_delta_pack(Packs p) {
    constexpr int VN = Vec<T>::N;
    const int t = blockIdx.y, H = p.heads[t], D = p.width[t], units = (D + VN - 1) / VN;
    const fm_view& v = p.from[t];
    const long long all = p.moments * H * units;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += 256LL * gridDim.x) {
        const long long row = i / units, m = row / H, n = m / p.n_moments;
        const int col = (int)(i - row * units) * VN, h = (int)(row - m * H);
        const T* from = (const T*)v.data + n * v.seq + (m - n * p.n_moments) * v.moment + h * v.head;
        reinterpret_cast<uint4*>(p.to[t])[i] = load16(from, col, D, true);
    }
}

// ------------------------------------------------------------------------------------------------ T, P and the factors
// A workgroup a chunk and head.  K K^T and Q K^T on the matrix cores; N in float32 in LDS; T by blocks of 16: those on the diagonal by
// forward substitution, a lane a column, then T_ij = -T_ii sum_k N_ik T_kj down each column of blocks, in float32 products
// whose second operand stays in registers.  G is summed in 64 bits and kept in two floats: a difference of two of them is
// exact to its own last bits however much has been forgotten before.  BOTH: the operands of the transposes too, for the gradient.
// A moment whose key, decay or rate is not finite spoils all from there on (k_delta_scan): here its chunk ends before it.
// 8 x 4,096 moments, 16 heads of 128 in bfloat16 take 180 us with both (100 one way): vector instructions take 63% of the cycles
// at 4 workgroups a CU, and 0.57 GB are written.  32,768 moments, 8 heads: 61 us.
template <class T, int KT, bool BOTH>
__global__ __launch_bounds__(256) void k_delta_prep(Delta a) {
    using F = DeltaForm<T>;
    using B = DeltaForm<T, true>;
    constexpr int X = F::X, CH = F::CH, JB = F::JB, KW = 32 * KT, XP = CH * KW, VN = Vec<T>::N, XC = KW / VN;
    constexpr int NP = CH + 4;                            // a row of N and T, padded
    // q and k; then, when their products are made, N and T (4 workgroups a CU)
    constexpr int ROWS_BYTES = 2 * X * XP * 2, NT_BYTES = 2 * CH * NP * 4;
    __shared__ __align__(16) char room[ROWS_BYTES > NT_BYTES ? ROWS_BYTES : NT_BYTES];
    bf16 *const sq = reinterpret_cast<bf16*>(room), *const sk = sq + X * XP;
    float *const sn = reinterpret_cast<float*>(room), *const st = sn + CH * NP;
    __shared__ __align__(16) float hi[CH], lo[CH], sb[CH];
    __shared__ int bad;
    const unsigned block = (unsigned)block_number();
    const int place_in = (int)(block / a.heads), h = (int)(block - (unsigned)place_in * a.heads);
    if (place_in >= a.chunks.slots) return;
    int n, seg, slot;
    long long first, count;
    if (!segment_of(a.chunks, place_in, n, seg, slot, first, count)) return;
    const long long from = (long long)seg * CH, left = count - from;
    const int rows = (int)(left < CH ? left : CH);
    if (rows <= 0) return;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, c = lane & 15;
    const long long moment = first + from;
    char* const prep = a.prep + ((size_t)slot * a.heads + h) * F::PREP;
    char* const turned_prep = BOTH ? a.turned + ((size_t)slot * a.heads + h) * B::PREP : nullptr;
    float ld = 0.f, be = 0.f;
    {
        const Chunk<T> q = chunk_of<T>(a, a.q, n, h, moment, rows, a.K), k = chunk_of<T>(a, a.k, n, h / a.share, moment, rows, a.K);
        constexpr int N = CH * XC / 256;
        static_assert(N * 256 == CH * XC, "");
        u32x4 rq[N], rk[N];                               // (all on their way at once)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            rq[i] = __builtin_bit_cast(u32x4, q((i * 256 + tid) / XC, (i * 256 + tid) % XC * VN));
            rk[i] = __builtin_bit_cast(u32x4, k((i * 256 + tid) / XC, (i * 256 + tid) % XC * VN));
        }
        if (tid < rows) {
            ld = a.log_decay[(a.chunks.starts ? 0 : n * a.ld_seq) + (moment + tid) * a.ld_moment + h * a.ld_head];
            be = a.beta[(a.chunks.starts ? 0 : n * a.be_seq) + (moment + tid) * a.be_moment + h * a.be_head];
        }
        if (tid == 0) bad = rows;
        __syncthreads();
        if (tid < rows && (!(ld < INFINITY) || !(fabsf(be) < INFINITY))) atomicMin(&bad, tid);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = (i * 256 + tid) / XC, col = (i * 256 + tid) % XC * VN, to = place<KW>(row, col >> 3) + (col & 7);
            store_terms<T>(__builtin_bit_cast(uint4, rq[i]), sq + to, XP);
            store_terms<T>(__builtin_bit_cast(uint4, rk[i]), sk + to, XP);
            if (odd16<T>(__builtin_bit_cast(uint4, rk[i]))) atomicMin(&bad, row);
        }
    }
    __syncthreads();
    const int stop = bad;                                 // rows from here on: nothing
    if (stop < rows)
        for (int i = tid; i < CH * XC; i += 256)
            if (i / XC >= stop) store_terms<T>(make_uint4(0, 0, 0, 0), sk + place<KW>(i / XC, i % XC * VN >> 3) + (i % XC * VN & 7), XP);
    if (wave == 0) {
        double s = lane < stop ? (double)fmaxf(ld, GONE) : 0.0;
        for (int m = 1; m < 64; m <<= 1) {
            const double t = __shfl_up(s, m);
            if (lane >= m) s += t;
        }
        const double end = __shfl(s, CH - 1);             // (rows past the last add nothing)
        const float b = lane < stop ? be : 0.f, high = (float)s;
        if (lane < CH) {
            hi[lane] = high;
            lo[lane] = (float)(s - (double)high);
            sb[lane] = b;
        }
        const float e = lane < rows ? exp_of((float)s) : 0.f;              // (a row past the last adds nothing to a gradient)
        const float left_over = exp_of((float)(end - s));
        const Keep keep((float)end);
        auto write = [&](float* f) {
            if (lane < CH) {
                f[F_E + lane] = e;
                f[F_E + CH + lane] = left_over * b;
                f[F_E + 2 * CH + lane] = left_over;
                f[F_E + 3 * CH + lane] = b;
                f[F_E + 4 * CH + lane] = high;
                f[F_E + 5 * CH + lane] = (float)(s - (double)high);
            }
            if (lane == 0) {
                f[0] = keep.one;
                f[1] = keep.f;
                f[2] = __int_as_float(stop < rows ? stop : CH);
                f[3] = 0.f;
            }
        };
        write(const_cast<float*>(factors_of<F>(prep)));
        if (BOTH) write(const_cast<float*>(factors_of<B>(turned_prep)));
    }
    __syncthreads();

    bf16x8 *const units = reinterpret_cast<bf16x8*>(prep), *const turned_units = reinterpret_cast<bf16x8*>(turned_prep);
    // a block of P as half an operand, and the half above the diagonal beside it
    auto store_halves = [&](auto form, bf16x8* to, int unit, int half, bool alone, f32x4 p) {
        constexpr int W = decltype(form)::W;
        Sum<W, 4> s;
        s.of_summed(p);
#pragma unroll
        for (int t = 0; t < W; ++t) {
            bf16x4* const at = reinterpret_cast<bf16x4*>(&to[(unit * W + t) * 64 + lane]);
            at[half] = s.term[t];
            if (alone) at[1 - half] = bf16x4{};
        }
    };
    constexpr int BLOCKS = JB * (JB + 1) / 2, TASKS = (BOTH ? 3 : 2) * BLOCKS, MINE = (TASKS + 3) / 4, NS = (BLOCKS + 3) / 4;
    f32x4 p[MINE];                                        // this wave's blocks: of N (task < BLOCKS), P, and P by rows
#pragma unroll
    for (int m = 0; m < MINE; ++m) p[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < KT; ++b) {
        const int at = place<KW>(c, g) ^ 32 * b;
#pragma unroll
        for (int m = 0; m < MINE; ++m) {                  // (past the last: some block once more)
            const int task = min(4 * m + wave, TASKS - 1), kind = task / BLOCKS;
            int i, j;
            block_of(task - kind * BLOCKS, i, j);
            // P forwards: rows j, columns i; else rows i, columns j
            const bf16* const ra = kind == 1 ? sk + 16 * j * KW : (kind ? sq : sk) + 16 * i * KW;
            const bf16* const rb = kind == 1 ? sq + 16 * i * KW : sk + 16 * j * KW;
            p[m] = mfma_whole(across<X>(ra + at, XP), across<X>(rb + at, XP), p[m]);
        }
    }
#pragma unroll
    for (int m = 0; m < MINE; ++m) {
        const int task = 4 * m + wave, kind = task / BLOCKS;
        if (task >= TASKS) break;
        int i, j;
        block_of(task - kind * BLOCKS, i, j);
        const int ri = 16 * i + (kind == 1 ? c : 4 * g), cj = 16 * j + (kind == 1 ? 4 * g : c);     // a lane's first
        const f32x4 h4 = *reinterpret_cast<const f32x4*>(&hi[kind == 1 ? cj : ri]), l4 = *reinterpret_cast<const f32x4*>(&lo[kind == 1 ? cj : ri]);
        const f32x4 b4 = *reinterpret_cast<const f32x4*>(&sb[kind == 1 ? cj : ri]);
        const float h1 = hi[kind == 1 ? ri : cj], l1 = lo[kind == 1 ? ri : cj], b1 = sb[cj];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = kind == 1 ? ri : ri + r, col = kind == 1 ? cj + r : cj;
            const float apart = kind == 1 ? (h1 - h4[r]) + (l1 - l4[r]) : (h4[r] - h1) + (l4[r] - l1);
            const float d = exp_of(fminf(apart, 88.f)) * (kind == 1 ? b4[r] : b1);
            p[m][r] = kind ? (row >= col ? a.c * d * p[m][r] : 0.f) : (row > col ? d * p[m][r] : 0.f);
        }
        if (kind == 1) store_halves(F{}, units, piece_of(j >> 1, i), j & 1, !(j & 1) && i == j, p[m]);
        else if (BOTH && kind == 2) store_halves(B{}, turned_units, tpiece_of(i >> 1, j), i & 1, (i & 1) && i == j, p[m]);
    }
    __syncthreads();                                      // (q and k are read)
#pragma unroll
    for (int m = 0; m < NS; ++m) {
        int i, j;
        block_of(4 * m + wave, i, j);
        if (4 * m + wave < BLOCKS)
#pragma unroll
            for (int r = 0; r < 4; ++r) sn[(16 * i + 4 * g + r) * NP + 16 * j + c] = p[m][r];
    }
    __syncthreads();
    if (tid < CH) {                                       // the diagonal blocks: column c of block tid / 16
        const int b0 = tid & ~15, col = tid & 15;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s[4] = {i == col ? 1.f : 0.f, 0.f, 0.f, 0.f};           // (four sums: a chain of dependent products a quarter as long)
#pragma unroll
            for (int j = 0; j < i; j += 4) {
                const f32x4 row = *reinterpret_cast<const f32x4*>(&sn[(b0 + i) * NP + b0 + j]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (j + e < i) s[e] = fmaf(-row[e], x[j + e], s[e]);
            }
            x[i] = (s[0] + s[1]) + (s[2] + s[3]);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) st[(b0 + i) * NP + b0 + col] = x[i];
    }
    __syncthreads();
    if (wave < JB - 1) {                                  // column `wave` of the blocks below the diagonal
        const int j = wave;
        f32x4 t[JB];
#pragma unroll
        for (int r = 0; r < 4; ++r) t[0][r] = st[(16 * j + 4 * g + r) * NP + 16 * j + c];
#pragma unroll
        for (int d = 1; d < JB; ++d) {                    // block (j + d, j)
            const int i = j + d;
            if (i >= JB) break;
            f32x4 s = {0.f, 0.f, 0.f, 0.f}, o = s;
#pragma unroll
            for (int k = 0; k < JB - 1; ++k) {
                if (k >= d) break;
                const f32x4 na = *reinterpret_cast<const f32x4*>(&sn[(16 * i + c) * NP + 16 * (j + k) + 4 * g]);
#pragma unroll
                for (int r = 0; r < 4; ++r) s = mfma4(na[r], t[k][r], s);
            }
            const f32x4 ta = *reinterpret_cast<const f32x4*>(&st[(16 * i + c) * NP + 16 * i + 4 * g]);
#pragma unroll
            for (int r = 0; r < 4; ++r) o = mfma4(-ta[r], s[r], o);
            t[d] = o;
#pragma unroll
            for (int r = 0; r < 4; ++r) st[(16 * i + 4 * g + r) * NP + 16 * j + c] = o[r];
        }
    }
    __syncthreads();
    for (int task = wave; task < (BOTH ? 2 : 1) * F::PIECES; task += 4) {
        f32x4 half[2];
        if (task >= F::PIECES) {                          // rows j, summed over i
            const int m = task - F::PIECES, ii = m >= 2, j = ii ? m - 2 : m;
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    half[e][r] = 2 * ii + e >= j ? st[(16 * (2 * ii + e) + 4 * g + r) * NP + 16 * j + c] : 0.f;
        } else {                                          // rows i, summed over j
            const int jj = task >= 4, i = jj ? task - 2 : task;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int j = 2 * jj + e;
                half[e] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (j <= i) half[e] = *reinterpret_cast<const f32x4*>(&st[(16 * i + c) * NP + 16 * j + 4 * g]);
            }
        }
        Sum<T_TERMS, 8> s;
        s.of_summed(joined(half[0], half[1]));
        bf16x8* const to = task < F::PIECES ? units + (F::P_UNITS + task * T_TERMS) * 64 : turned_units + (B::P_UNITS + (task - F::PIECES) * T_TERMS) * 64;
#pragma unroll
        for (int t = 0; t < T_TERMS; ++t) to[t * 64 + lane] = s.term[t];
    }
}

// A chunk's inputs in LDS: rows of q, k and of 64 columns of a third tensor (as terms, swizzled: place), the operands that
// k_delta_prep left and its first factors.
// Inputs of one term go there straight from memory (a wave 1 KB at a time), a chunk ahead into the other of two rooms; others
// pass through registers, where they become terms, a chunk ahead too.
template <class T, class F, int KT>
struct Stage {
    static constexpr int X = F::X, CH = F::CH, KW = 32 * KT, NW = 64, XP = CH * KW, VP = CH * NW, VN = Vec<T>::N;
    static constexpr bool STRAIGHT = X == 1;
    static constexpr int K_AT = 2 * X * XP, W_AT = 2 * K_AT, U_AT = W_AT + 2 * X * VP, F_AT = U_AT + F::UNITS * 1024;   // bytes
    static constexpr int BYTES = F_AT + (STRAIGHT ? 1024 : (16 + 8 * CH)), ROOMS = STRAIGHT ? 2 : 1;
    static constexpr int XC = KW / VN, VC = NW / VN, XR = 256 / XC, VR = 256 / VC, XV = CH / XR, VV = CH / VR, UV = F::UNITS / 4;
    static_assert(XV * XR == CH && VV * VR == CH && F::FACTORS * 4 >= (STRAIGHT ? 1024 : 16 + 8 * CH), "");
    uint4 rq[STRAIGHT ? 1 : XV], rk[STRAIGHT ? 1 : XV], rw[STRAIGHT ? 1 : VV];
    u32x4 ru[STRAIGHT ? 1 : UV], rf;
    static constexpr int QV = CH * KW / 2048, WV = CH * NW / 2048;        // units of 1 KB a wave
    unsigned oq[QV], ok[QV], ow[WV];                      // a lane's places in them
    unsigned long long mq[QV], mw[WV];                    // the lanes that have one
    int placed = -1;                                      // ... for chunks of so many rows
    char* room;
    int tid, wave, lane;
    const Delta& a;
    const fm_view& w;
    int n, h, hw, c0, slot0;
    long long first, count;
    bool with_q, with_w;                 // whether q and P, and the third tensor, are wanted

    __device__ __forceinline__ Stage(char* room, const Delta& a, const fm_view& w, int n, int h, int hw, int c0, int slot0,
                                     long long first, long long count, bool with_q = true, bool with_w = true)
        : room(room), tid(threadIdx.x), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), lane(threadIdx.x & 63), a(a), w(w),
          n(n), h(h), hw(hw), c0(c0), slot0(slot0), first(first), count(count), with_q(with_q), with_w(with_w) {
        if constexpr (STRAIGHT) {                         // columns past a head's end: zeros for good
            for (int i = tid; i < ROOMS * BYTES / 16; i += 256) reinterpret_cast<uint4*>(room)[i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
        }
    }
    __device__ __forceinline__ const bf16* q(int which) const { return reinterpret_cast<const bf16*>(room + which * BYTES); }
    __device__ __forceinline__ bf16* k(int which) const { return reinterpret_cast<bf16*>(room + which * BYTES + K_AT); }
    __device__ __forceinline__ const bf16* third(int which) const { return reinterpret_cast<const bf16*>(room + which * BYTES + W_AT); }
    __device__ __forceinline__ const bf16x8* units(int which) const { return reinterpret_cast<const bf16x8*>(room + which * BYTES + U_AT); }
    __device__ __forceinline__ const float* factors(int which) const { return reinterpret_cast<const float*>(room + which * BYTES + F_AT); }

    __device__ __forceinline__ const char* prepared(long long i0) const {
        return a.prep + ((size_t)(slot0 + i0 / CH) * a.heads + h) * F::PREP;
    }
    // 1 KB: a lane's 16 bytes from `offset` bytes past `base` to 16 bytes times the lane's number behind `to`, of the lanes in `mask`.
    // (m0, the place in LDS, is the compiler's to set before each instruction of its own that reads it: it keeps nothing there.  A base
    // that a vector instruction leaves in scalar registers less than five wait states before would be read too early: `base` and
    // `prepared` are sums of scalar instructions, and tests/test_delta_loads.py looks at all that stands before these loads.)
    __device__ __forceinline__ static void straight(const void* base, unsigned offset, unsigned long long mask, const char* to) {
        const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)to);
        unsigned long long active;
        asm volatile("s_mov_b32 m0, %1\n\ts_and_saveexec_b64 %0, %4\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b64 exec, %0" : "=&s"(active)
                     : "s"(at), "v"(offset), "s"(base), "s"(mask) : "memory", "scc");
    }
    // a lane's place in unit 4 i + wave of rows of WIDTH values, and the lanes whose columns are the head's
    template <int WIDTH>
    __device__ __forceinline__ unsigned place_of(int i, int rows, long long step, int col0, int width, unsigned long long& mask) const {
        const int at = (4 * i + wave) * 512 + lane * 8, row = at / WIDTH;
        const int col = col0 + (place<WIDTH>(row, at % WIDTH >> 3) - row * WIDTH);
        mask = __ballot(col < width);
        return (unsigned)(min(row, rows - 1) * (int)step + (col < width ? col : 0)) * (unsigned)sizeof(T);
    }
    __device__ __forceinline__ void places_of(int rows) {
#pragma unroll
        for (int i = 0; i < QV; ++i) {
            oq[i] = place_of<KW>(i, rows, a.q.moment, 0, a.K, mq[i]);
            ok[i] = place_of<KW>(i, rows, a.k.moment, 0, a.K, mq[i]);
        }
#pragma unroll
        for (int i = 0; i < WV; ++i) ow[i] = place_of<NW>(i, rows, w.moment, c0, a.V, mw[i]);
    }
    __device__ __forceinline__ const T* base(const fm_view& v, int head, long long i0) const {
        return (const T*)v.data + (a.chunks.starts ? 0 : n * v.seq) + head * v.head + (first + i0) * v.moment;
    }
    // A quarter of it: issued all at once, the loads' wave waits for their queue (2,000 cycles a chunk).
    __device__ __forceinline__ void fetch_part(long long i0, int which, int part) {
        // (rows past the chunk's last are the last once more: k_delta_prep's factors leave them out)
        const int rows = (int)(count - i0 < CH ? count - i0 : CH);
        if (part == 0 && rows != placed) places_of(placed = rows);
        char* const to = room + which * BYTES + wave * 1024;
        const char* const prep = prepared(i0);
        if (part == 0 && with_q) {
            const T* const from = base(a.q, h, i0);
#pragma unroll
            for (int i = 0; i < QV; ++i) straight(from, oq[i], mq[i], to + i * 4096);
        }
        if (part == 1) {
            const T* const from = base(a.k, h / a.share, i0);
#pragma unroll
            for (int i = 0; i < QV; ++i) straight(from, ok[i], mq[i], to + K_AT + i * 4096);
        }
        if (part == 2) {
            const T* const from = base(w, hw, i0);
#pragma unroll
            for (int i = 0; i < WV; ++i)
                if (with_w) straight(from, ow[i], mw[i], to + W_AT + i * 4096);
            straight(prep + F::UNITS * 1024, lane * 16, ~0ull, room + which * BYTES + F_AT);      // (all waves the same)
        }
#pragma unroll
        for (int i = 0; i < UV; ++i) {
            if (part != 2 + (i >= UV / 2)) continue;
            if (with_q || 4 * i + wave >= F::P_UNITS) straight(prep + (4 * i + wave) * 1024, lane * 16, ~0ull, to + U_AT + i * 4096);
        }
    }
    // the chunk from moment i0 on its way into room `which`
    __device__ __forceinline__ void fetch(long long i0, int which) {
        if constexpr (STRAIGHT) {
#pragma unroll
            for (int part = 0; part < 4; ++part) fetch_part(i0, which, part);
        } else {
            const int rows = (int)(count - i0 < CH ? count - i0 : CH);
            const char* const prep = prepared(i0);
            const Chunk<T> cq = chunk_of<T>(a, a.q, n, h, first + i0, rows, a.K), ck = chunk_of<T>(a, a.k, n, h / a.share, first + i0, rows, a.K);
            const Chunk<T> cw = chunk_of<T>(a, w, n, hw, first + i0, rows, a.V);
#pragma unroll
            for (int i = 0; i < XV; ++i) {
                if (with_q) rq[i] = cq(tid / XC + i * XR, tid % XC * VN);
                rk[i] = ck(tid / XC + i * XR, tid % XC * VN);
            }
#pragma unroll
            for (int i = 0; i < VV; ++i) rw[i] = with_w ? cw(tid / VC + i * VR, c0 + tid % VC * VN) : make_uint4(0, 0, 0, 0);
            const u32x4* const u = reinterpret_cast<const u32x4*>(prep);
#pragma unroll
            for (int i = 0; i < UV; ++i) ru[i] = u[i * 256 + tid];        // (P too, where it is not wanted)
            rf = reinterpret_cast<const u32x4*>(prep + F::UNITS * 1024)[min(tid, CH / 2)];
        }
    }
    // what this wave has on its way is there (before its stores: they are not waited for)
    __device__ __forceinline__ void landed() const {
        if constexpr (STRAIGHT) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    // what has landed is there for all waves, and what was there before is read by all
    __device__ __forceinline__ void arrive() {
        if constexpr (STRAIGHT) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        } else {
            __syncthreads();
            bf16 *const sq = const_cast<bf16*>(q(0)), *const sk = k(0), *const sw = const_cast<bf16*>(third(0));
            const int xrow = tid / XC, xcol = tid % XC * VN, vrow = tid / VC, vcol = tid % VC * VN;
#pragma unroll
            for (int i = 0; i < XV; ++i) {
                const int to = place<KW>(xrow + i * XR, xcol >> 3) + (xcol & 7);
                if (with_q) store_terms<T>(rq[i], sq + to, XP);
                store_terms<T>(rk[i], sk + to, XP);
            }
#pragma unroll
            for (int i = 0; i < VV; ++i)
                store_terms<T>(rw[i], sw + place<NW>(vrow + i * VR, vcol >> 3) + (vcol & 7), VP);
#pragma unroll
            for (int i = 0; i < UV; ++i) reinterpret_cast<u32x4*>(room + U_AT)[i * 256 + tid] = ru[i];
            if (tid < 1 + CH / 2) reinterpret_cast<u32x4*>(room + F_AT)[tid] = rf;
            __syncthreads();
        }
    }
};

// ------------------------------------------------------------------------------------------------ the walk forwards
// A workgroup of 4 waves walks one head's chunks for 64 columns of its state, a wave 16: columns never meet, so waves share only
// what they read.  A chunk's rows and operands go through LDS, the next chunk's on their way in registers meanwhile.  An
// accumulator block of 16 x 16 (lane (c, g): column c, rows 4g .. 4g + 3) is the operand of the product that sums over its
// rows, so S, v - E K S and e pass between products in registers; outputs are formed transposed, so that a lane stores a row's
// values side by side.
// A value of v that is not finite makes its column NaN from its moment on; a key, decay or rate that is not, all columns:
// such moments are left out of the products (0 times them would not be 0) and marked in what is stored.
// What bounds it: a chunk depends on the one before it, and its four products on each other, at one wave a SIMD: 8 x 4,096 moments,
// 16 heads of 128 in bfloat16, one workgroup a CU, take 400 us (KEEP; 6.2 a chunk), matrix instructions 25% of the cycles.  Two
// workgroups a CU have no room in LDS for two chunks each (116,736 bytes a workgroup at heads of 64, 149,504 at 128, also for a
// segment's own states, which read neither q nor P), and without the second room the loads are in the open.  8 waves over 128
// columns could share one chunk (8 KB a room more), in half the registers each: the walks take 239 to 474 of 512 in bfloat16; not
// tried.  Those of float32 heads over 64 take 322 to 512 (16 x 512 moments, 8 heads of 128, KEEP: 109 us, 6.8 a chunk).  Chunks of 64 moments for binary16 and
// float32 too, whose terms take two and three times the registers: walks the same, k_delta_prep 20 -> 29 us, k_delta_grads 48 -> 80
// (16 x 512 moments, 8 heads of 64, float32).
enum Walk { PLAY, KEEP, OWN };            // outputs; outputs, states and errors kept; a segment's own end state alone
template <class T, int KT, Walk WALK>
__global__ __launch_bounds__(256, 1) void k_delta_scan(Delta a) {
    using F = DeltaForm<T>;
    constexpr int X = F::X, W = F::W, CH = F::CH, JB = F::JB, KW = 32 * KT, XP = CH * KW, NW = 64, VP = CH * NW;
    using In = Stage<T, F, KT>;
    __shared__ __align__(16) char room[In::ROOMS * In::BYTES];
    const int blocks_v = (a.V + NW - 1) / NW, blocks = WALK == OWN ? blocks_v + KT / 2 : blocks_v;
    // (a segment's blocks of columns 8 workgroups apart: on one XCD, whose L2 then holds what they all read)
    const unsigned block = (unsigned)block_number(), unit = block / (8 * blocks) * 8 + (block & 7), place_in = unit / a.heads;
    const int vb = (int)(block / 8 % blocks), h = (int)(unit - place_in * a.heads);
    if (place_in >= (unsigned)a.segs.slots) return;
    int n, seg, slot;
    long long first, count;
    if (!segment_of(a.segs, (int)place_in, n, seg, slot, first, count)) return;
    n = __builtin_amdgcn_readfirstlane(n);
    seg = __builtin_amdgcn_readfirstlane(seg);
    slot = __builtin_amdgcn_readfirstlane(slot);
    const int slot0 = first_slot(a.chunks, n, shared_by_all(first)) + (int)(seg * (a.segs.L / CH));
    const long long from = start_of(a.segs, seg), left = shared_by_all(count - from < a.segs.L ? count - from : a.segs.L);
    const bool last = shared_by_all(count) == from + left;
    first = shared_by_all(first) + from;
    // a segment's own state: none is needed of the last one; the first one's is the true one, which needs no M
    const bool moves = WALK == OWN && vb >= blocks_v;     // columns of M
    if (WALK == OWN && (last || (moves && seg == 0))) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int v0 = NW * vb, col = v0 + 16 * wave + c, VW = NW * blocks_v;
    const size_t at_state = ((size_t)n * a.heads + h) * a.K * a.V;
    auto row_of = [&](int b, int r) { return 32 * (b >> 1) + 8 * g + 4 * (b & 1) + r; };
    const size_t seg_state = (size_t)a.heads * KW * VW, at_seg = (size_t)slot * seg_state + (size_t)h * KW * VW;
    f32x4 z[2 * KT];
#pragma unroll
    for (int b = 0; b < 2 * KT; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int k = row_of(b, r);
            if (moves) z[b][r] = k == col - NW * blocks_v ? 1.f : 0.f;
            else if (seg) z[b][r] = WALK == OWN ? 0.f : a.own[at_seg - seg_state + (size_t)k * VW + col];
            else z[b][r] = a.init && k < a.K && col < a.V ? a.init[at_state + (size_t)k * a.V + col] : 0.f;
        }
    In in(room, a, a.v, n, h, h / a.share, v0, slot0, first, left, WALK != OWN, !moves);
    int which = 0;
    if (left > 0) in.fetch(0, 0);
    loads_done();
    const int xat = place<KW>(c, g), yat = place<KW>(4 * g + (c >> 2), c & 3);
    const int vat = place<NW>(4 * g + (c >> 2), 2 * wave + (c >> 1 & 1)) + 4 * (c & 1);
    for (long long i0 = 0; i0 < left; i0 += CH, which ^= In::ROOMS - 1) {
        const int rows = (int)(left - i0 < CH ? left - i0 : CH);
        const long long next = i0 + CH;
        in.arrive();
        const long long coming = next < left ? next : i0;    // (after the last chunk it once more, for nothing: no branch)
        const bf16 *const sq = in.q(which), *const vdown = in.third(which) + vat;
        bf16* const sk = in.k(which);
        const bf16x8 *const sp = in.units(which) + lane, *const stt = sp + F::P_UNITS * 64;
        const float* const sf = in.factors(which);
        const int bad = __builtin_amdgcn_readfirstlane(__float_as_int(sf[2]));
        if (bad < CH) {                                   // keys from there on: nothing
            for (int i = tid; i < X * CH * KW / 8; i += 256)
                if (i % (CH * KW / 8) / (KW / 8) >= bad) reinterpret_cast<uint4*>(sk)[i] = make_uint4(0, 0, 0, 0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        }
        const size_t mine = (size_t)(slot0 + i0 / CH) * a.heads + h;
        if (WALK == KEEP) {
            float* const to = a.states + mine * KW * VW + col;
#pragma unroll
            for (int b = 0; b < 2 * KT; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) to[row_of(b, r) * VW] = z[b][r];
        }
        f32x4 e[JB], o[JB];
#pragma unroll
        for (int i = 0; i < JB; ++i) e[i] = o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        Sum<X, 8> kf[2][JB], qf[2][JB], vf[JB / 2];
        Sum<T_TERMS, 8> tf[F::PIECES];
        auto read_rows = [&](int b) {
#pragma unroll
            for (int i = 0; i < JB; ++i) {
                kf[b & 1][i] = across<X>(sk + 16 * i * KW + (xat ^ 32 * b), XP);
                if (WALK != OWN) qf[b & 1][i] = across<X>(sq + 16 * i * KW + (xat ^ 32 * b), XP);
            }
        };
        read_rows(0);
#pragma unroll
        for (int b = 0; b < KT; ++b) {
            if (b + 1 < KT) read_rows(b + 1);
            else {
#pragma unroll
                for (int jj = 0; jj < JB / 2; ++jj) vf[jj] = down<X>(vdown + 32 * jj * NW, 16 * NW, VP);
#pragma unroll
                for (int m = 0; m < JB; ++m)
#pragma unroll
                    for (int t = 0; t < T_TERMS; ++t) tf[m].term[t] = stt[(m * T_TERMS + t) * 64];
            }
            if (In::STRAIGHT) {
#pragma unroll
                for (int part = 4 / KT * b; part < 4 / KT * (b + 1); ++part) in.fetch_part(coming, which ^ 1, part);
            }
            in_order();
            Sum<T_TERMS, 8> zf;
            zf.of_summed(joined(z[2 * b], z[2 * b + 1]));
            mfmas<true, JB>(e, kf[b & 1], zf);
            if (WALK != OWN) mfmas<false, JB>(o, qf[b & 1], first_terms<W>(zf));
            in_order();
        }
        if (!In::STRAIGHT && next < left) in.fetch(next, 0);
        Sum<X, 8> kt[JB / 2][2 * KT];
        auto read_columns = [&](int jj) {
#pragma unroll
            for (int b = 0; b < 2 * KT; ++b) kt[jj][b] = down<X>(sk + 32 * jj * KW + (yat ^ 32 * (b >> 1)) + 4 * (b & 1), 16 * KW, XP);
        };
        int since = CH;                                   // the column's first moment that is not finite
        {
            f32x4 d[JB];
#pragma unroll
            for (int jj = 0; jj < JB / 2; ++jj) {
                f32x8 v = widened(vf[jj]);
                float s = 0.f;
#pragma unroll
                for (int r = 0; r < 8; ++r) s = fmaf(v[r], 0.f, s);
                if (__ballot(!(s == 0.f)))
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (!(fabsf(v[r]) < INFINITY)) {
                            since = min(since, 32 * jj + 16 * (r >> 2) + 4 * g + (r & 3));
                            v[r] = 0.f;
                        }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int i = 2 * jj + half;
                    const f32x4 f = *reinterpret_cast<const f32x4*>(&sf[F_E + 16 * i + 4 * g]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) d[i][r] = fmaf(-f[r], e[i][r], v[4 * half + r]);
                }
            }
#pragma unroll
            for (int i = 0; i < JB; ++i) e[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int m = JB; m < F::PIECES; ++m)
#pragma unroll
                for (int t = 0; t < T_TERMS; ++t) tf[m].term[t] = stt[(m * T_TERMS + t) * 64];
            read_columns(0);
            in_order();
#pragma unroll
            for (int jj = 0; jj < JB / 2; ++jj) {
                Sum<T_TERMS, 8> df;
                df.of_summed(joined(d[2 * jj], d[2 * jj + 1]));
                if (jj) mfmas<true, JB - 2>(e + 2, tf + JB, df);
                else mfmas<true, JB>(e, tf, df);
            }
            in_order();
        }
        if (__ballot(since < CH)) {
            since = min(since, __shfl_xor(since, 16));
            since = min(since, __shfl_xor(since, 32));
        }
        since = min(since, bad);
        const bool spoiled = __ballot(since < CH) != 0;
        // the state after the chunk
        Sum<W, 8> pf[F::PIECES];
        f32x4 fb[JB];
        float fo[JB];
#pragma unroll
        for (int i = 0; i < JB; ++i) {
            fb[i] = *reinterpret_cast<const f32x4*>(&sf[F_E + CH + 16 * i + 4 * g]);
            fo[i] = a.c * sf[F_E + 16 * i + c];
        }
        decayed<2 * KT>(z, sf[0], sf[1]);
#pragma unroll
        for (int jj = 0; jj < JB / 2; ++jj) {
            if (jj + 1 < JB / 2) read_columns(jj + 1);
            if (WALK != OWN && jj == JB / 2 - 1) {
#pragma unroll
                for (int m = 0; m < F::PIECES; ++m)
#pragma unroll
                    for (int t = 0; t < W; ++t) pf[m].term[t] = sp[(m * W + t) * 64];
            }
            in_order();
            Sum<T_TERMS, 8> uf;
            uf.of_summed(joined(e[2 * jj] * fb[2 * jj], e[2 * jj + 1] * fb[2 * jj + 1]));
            mfmas<true, 2 * KT>(z, kt[jj], uf);
            in_order();
        }
        if (spoiled && since < CH)
#pragma unroll
            for (int b = 0; b < 2 * KT; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) z[b][r] = NAN;
        if constexpr (WALK != OWN) {
        // outputs
#pragma unroll
        for (int i = 0; i < JB; ++i) o[i] *= fo[i];
#pragma unroll
        for (int jj = 0; jj < JB / 2; ++jj) {
            Sum<W, 8> ef;
            ef.of_summed(joined(e[2 * jj], e[2 * jj + 1]));
            if (jj) mfmas<false, JB - 2>(o + 2, pf + JB, ef);
            else mfmas<false, JB>(o, pf, ef);
        }
        if (spoiled)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int f = __shfl(since, 4 * g + r);
#pragma unroll
                for (int i = 0; i < JB; ++i)
                    if (16 * i + c >= f) o[i][r] = NAN;
            }
        }
        in.landed();
        if (WALK == KEEP) {
            float* const to = a.errors + mine * CH * VW + col;
#pragma unroll
            for (int i = 0; i < JB; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * i + 4 * g + r;
                    to[row * VW] = row < since ? e[i][r] : row < rows ? NAN : 0.f;
                }
        }
        if constexpr (WALK != OWN) {
            const int oc = v0 + 16 * wave + 4 * g, step = a.heads * a.V * (int)sizeof(T);
            T* const po = (T*)a.o + (((a.chunks.starts ? 0 : n * a.chunks.n_moments) + first + i0) * a.heads + h) * a.V;
            typedef T vec4 __attribute__((ext_vector_type(4)));
            if (a.vec) {                                  // (what lies outside is dropped)
                const auto to = rows_at(po, rows, step, a.V * (int)sizeof(T));
                const unsigned at = oc < a.V ? c * step + oc * (int)sizeof(T) : NOWHERE;
#pragma unroll
                for (int i = 0; i < JB; ++i) {
                    const vec4 v = __builtin_convertvector(o[i], vec4);
                    const unsigned there = 16 * i + c < rows ? at + 16 * i * step : NOWHERE;
                    if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), to, there, 0, 0);
                    else __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, v), to, there, 0, 0);
                }
            } else {
#pragma unroll
                for (int i = 0; i < JB; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (16 * i + c < rows && oc + r < a.V) po[(long long)(16 * i + c) * a.heads * a.V + oc + r] = narrow<T>(o[i][r]);
            }
        }
    }
    if (WALK == OWN) {
#pragma unroll
        for (int b = 0; b < 2 * KT; ++b) {
            const int at = col - NW * blocks_v;
            if (moves && a.trans_t)
                *reinterpret_cast<f32x4*>(a.trans_t + (((size_t)slot * a.heads + h) * KW + at) * KW + row_of(b, 0)) = z[b];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (moves) a.trans[(((size_t)slot * a.heads + h) * KW + row_of(b, r)) * KW + at] = z[b][r];
                else a.own[at_seg + (size_t)row_of(b, r) * VW + col] = z[b][r];
            }
        }
        return;
    }
    if (last && a.fin && col < a.V)
#pragma unroll
        for (int b = 0; b < 2 * KT; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int k = row_of(b, r);
                if (k < a.K) a.fin[at_state + (size_t)k * a.V + col] = z[b][r];
            }
}

// ------------------------------------------------------------------------------------------------ the walk backwards
// The same of X, the gradient of the state after a chunk: y = T^T (P^T g + F beta K X), X' = E_end X + Q^T (c E g) - K^T (E y).
// (KEEP of float32 heads over 64 takes all 512 registers and spills 20: 145 us where the walk forwards takes 109.)
template <class T, int KT, Walk WALK>
__global__ __launch_bounds__(256, 1) void k_delta_back(Delta a) {
    using F = DeltaForm<T, true>;
    constexpr int X = F::X, W = F::W, CH = F::CH, JB = F::JB, KW = 32 * KT, XP = CH * KW, NW = 64, VP = CH * NW;
    using In = Stage<T, F, KT>;
    __shared__ __align__(16) char room[In::ROOMS * In::BYTES];
    const int blocks_v = (a.V + NW - 1) / NW, blocks = blocks_v;
    // (a segment's blocks of columns 8 workgroups apart: on one XCD, whose L2 then holds what they all read)
    const unsigned block = (unsigned)block_number(), unit = block / (8 * blocks) * 8 + (block & 7), place_in = unit / a.heads;
    const int vb = (int)(block / 8 % blocks), h = (int)(unit - place_in * a.heads);
    if (place_in >= (unsigned)a.segs.slots) return;
    int n, seg, slot;
    long long first, count;
    if (!segment_of(a.segs, (int)place_in, n, seg, slot, first, count)) return;
    n = __builtin_amdgcn_readfirstlane(n);
    seg = __builtin_amdgcn_readfirstlane(seg);
    slot = __builtin_amdgcn_readfirstlane(slot);
    const int slot0 = first_slot(a.chunks, n, shared_by_all(first)) + (int)(seg * (a.segs.L / CH));
    const long long from = start_of(a.segs, seg), left = shared_by_all(count - from < a.segs.L ? count - from : a.segs.L);
    const bool last = shared_by_all(count) == from + left;
    first = shared_by_all(first) + from;
    if (WALK == OWN && seg == 0) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int v0 = NW * vb, col = v0 + 16 * wave + c, VW = NW * blocks_v;
    const size_t at_state = ((size_t)n * a.heads + h) * a.K * a.V;
    auto row_of = [&](int b, int r) { return 32 * (b >> 1) + 8 * g + 4 * (b & 1) + r; };
    const size_t seg_state = (size_t)a.heads * KW * VW, at_seg = (size_t)slot * seg_state + (size_t)h * KW * VW;
    f32x4 z[2 * KT];
#pragma unroll
    for (int b = 0; b < 2 * KT; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int k = row_of(b, r);
            if (!last) z[b][r] = WALK == OWN ? 0.f : a.own[at_seg + seg_state + (size_t)k * VW + col];
            else z[b][r] = a.gfin && k < a.K && col < a.V ? a.gfin[at_state + (size_t)k * a.V + col] : 0.f;
        }
    In in(room, a, a.go, n, h, h, v0, slot0, first, left);
    int which = 0;
    const long long end = left > 0 ? (left - 1) / CH * CH : -1;
    if (end >= 0) in.fetch(end, 0);
    loads_done();
    const int xat = place<KW>(c, g), yat = place<KW>(4 * g + (c >> 2), c & 3);
    const int gat = place<NW>(4 * g + (c >> 2), 2 * wave + (c >> 1 & 1)) + 4 * (c & 1);
    for (long long i0 = end; i0 >= 0; i0 -= CH, which ^= In::ROOMS - 1) {
        in.arrive();
        const long long coming = i0 ? i0 - CH : i0;       // (after the last chunk it once more, for nothing: no branch)
        const bf16 *const sq = in.q(which), *const sk = in.k(which), *const gdown = in.third(which) + gat;
        const bf16x8 *const sp = in.units(which) + lane, *const stt = sp + F::P_UNITS * 64;
        const float* const sf = in.factors(which);
        const size_t mine = (size_t)(slot0 + i0 / CH) * a.heads + h;
        if (WALK != OWN) {
            float* const to = a.grads + mine * KW * VW + col;
#pragma unroll
            for (int b = 0; b < 2 * KT; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) to[row_of(b, r) * VW] = z[b][r];
        }
        f32x4 d[JB], y[JB];
#pragma unroll
        for (int i = 0; i < JB; ++i) d[i] = y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        Sum<X, 8> kf[2][JB], gf[JB / 2];
        Sum<W, 8> pf[F::PIECES];
        Sum<T_TERMS, 8> tf[F::PIECES];
        f32x4 fb[JB], fe[JB];
        auto read_rows = [&](int b) {
#pragma unroll
            for (int i = 0; i < JB; ++i) kf[b & 1][i] = across<X>(sk + 16 * i * KW + (xat ^ 32 * b), XP);
        };
        read_rows(0);
#pragma unroll
        for (int b = 0; b < KT; ++b) {
            if (b + 1 < KT) read_rows(b + 1);
            else {
#pragma unroll
                for (int ii = 0; ii < JB / 2; ++ii) gf[ii] = down<X>(gdown + 32 * ii * NW, 16 * NW, VP);
#pragma unroll
                for (int m = 0; m < F::PIECES; ++m)
#pragma unroll
                    for (int t = 0; t < W; ++t) pf[m].term[t] = sp[(m * W + t) * 64];
#pragma unroll
                for (int i = 0; i < JB; ++i) {
                    fe[i] = *reinterpret_cast<const f32x4*>(&sf[F_E + 16 * i + 4 * g]);
                    fb[i] = *reinterpret_cast<const f32x4*>(&sf[F_E + CH + 16 * i + 4 * g]);
                }
            }
            if (In::STRAIGHT) {
#pragma unroll
                for (int part = 4 / KT * b; part < 4 / KT * (b + 1); ++part) in.fetch_part(coming, which ^ 1, part);
            }
            in_order();
            Sum<T_TERMS, 8> zf;
            zf.of_summed(joined(z[2 * b], z[2 * b + 1]));
            mfmas<true, JB>(d, kf[b & 1], zf);
            in_order();
        }
        if (!In::STRAIGHT && i0) in.fetch(i0 - CH, 0);
#pragma unroll
        for (int m = 0; m < F::PIECES; ++m)
#pragma unroll
            for (int t = 0; t < T_TERMS; ++t) tf[m].term[t] = stt[(m * T_TERMS + t) * 64];
        in_order();
#pragma unroll
        for (int i = 0; i < JB; ++i) d[i] *= fb[i];
#pragma unroll
        for (int ii = 0; ii < JB / 2; ++ii) {
            if (ii) mfmas<true, JB>(d, pf + 2, gf[ii]);
            else mfmas<true, 2>(d, pf, gf[ii]);
        }
        in_order();
        Sum<X, 8> qt[2 * KT], kt[2 * KT];                 // (of the first 32 moments; then of the others)
        auto read_columns = [&](int jj) {
#pragma unroll
            for (int b = 0; b < 2 * KT; ++b) {
                const int at = 32 * jj * KW + (yat ^ 32 * (b >> 1)) + 4 * (b & 1);
                qt[b] = down<X>(sq + at, 16 * KW, XP);
                kt[b] = down<X>(sk + at, 16 * KW, XP);
            }
        };
        read_columns(0);
        in_order();
#pragma unroll
        for (int ii = 0; ii < JB / 2; ++ii) {
            Sum<T_TERMS, 8> df;
            df.of_summed(joined(d[2 * ii], d[2 * ii + 1]));
            if (ii) mfmas<true, JB>(y, tf + 2, df);
            else mfmas<true, 2>(y, tf, df);
        }
        in_order();
        if (WALK != OWN) {
            float* const to = a.ys + mine * CH * VW + col;
#pragma unroll
            for (int i = 0; i < JB; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) to[(16 * i + 4 * g + r) * VW] = y[i][r];
        }
        decayed<2 * KT>(z, sf[0], sf[1]);
#pragma unroll
        for (int jj = 0; jj < JB / 2; ++jj) {
            const f32x8 f = joined(fe[2 * jj], fe[2 * jj + 1]);
            Sum<T_TERMS, 8> gt, yt;
            gt.of_summed(widened(gf[jj]) * (f * a.c));
            yt.of_summed(-joined(y[2 * jj], y[2 * jj + 1]) * f);
            mfmas<true, 2 * KT>(z, qt, gt);
            mfmas<true, 2 * KT>(z, kt, yt);
            in_order();
            if (jj + 1 < JB / 2) read_columns(jj + 1);
        }
        in.landed();
    }
    if (WALK == OWN) {
#pragma unroll
        for (int b = 0; b < 2 * KT; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) a.own[at_seg + (size_t)row_of(b, r) * VW + col] = z[b][r];
        return;
    }
    if (seg == 0 && a.ginit && col < a.V)
#pragma unroll
        for (int b = 0; b < 2 * KT; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int k = row_of(b, r);
                if (k < a.K) a.ginit[at_state + (size_t)k * a.V + col] = z[b][r];
            }
}

// Segments' end states from their own: S_0 = own_0, S_s = M_s S_{s-1} + own_s, in place; backwards X_s = M_s^T X_{s+1} + own_s
// from the last segment's.  This is the one part that no other chain fills the machine beside: a workgroup takes 16 columns, a
// wave 32 rows of M, whose terms stay its own; S passes between waves through LDS, in two rooms for one barrier a segment.  A segment
// of 128 x 128 takes 2.6 us (64 columns a workgroup, M's terms in LDS: 5.5, with 96 KB read from LDS by each wave), most of it
// for M's terms; a second M on its way changes nothing.  The last segment's end state (backwards: the first one's X) is left to
// the walk.  grid (blocks of 16 columns x heads, a head's on one XCD where their number is a multiple of 8; stretches)
template <int KT, bool BACK>
__global__ __launch_bounds__(64 * KT) void k_delta_join(Delta a) {
    constexpr int KW = 32 * KT;
    __shared__ __align__(16) bf16x8 sz[2][KT][T_TERMS][64];
    const int VW = 64 * ((a.V + 63) / 64), h = blockIdx.x % a.heads, n = blockIdx.y;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int col = 16 * (blockIdx.x / a.heads) + c;
    long long first, count;
    stretch_of(a.segs, n, first, count);
    const int segments = (int)((count + a.segs.L - 1) / a.segs.L), slot = first_slot(a.segs, n, first);
    if (segments < 3) return;                             // (one end state, and it is the true one)
    const ptrdiff_t step = (ptrdiff_t)a.heads * KW * VW * (BACK ? -1 : 1), mstep = (ptrdiff_t)a.heads * KW * KW * (BACK ? -1 : 1);
    const int s0 = BACK ? segments - 1 : 0;
    float* own = a.own + ((size_t)(slot + s0) * a.heads + h) * KW * VW + (32 * wave + 8 * g) * VW + col;
    const float* m = (BACK ? a.trans_t : a.trans) + ((size_t)(slot + s0) * a.heads + h) * KW * KW +
                     (size_t)(32 * wave + 8 * (c >> 2) + (c & 3)) * KW + 8 * g;
    f32x4 z[2], y[2], rm[KT][2][2];
    Sum<T_TERMS, 8> mf[KT][2];
    auto own_of = [&](f32x4 (&v)[2]) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[b][r] = own[(4 * b + r) * VW];
    };
    auto fetch = [&]() {                                  // the next segment's
        m += mstep;
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const f32x4* const row = reinterpret_cast<const f32x4*>(m + 4 * b * KW + 32 * k);
                rm[k][b][0] = row[0];
                rm[k][b][1] = row[1];
            }
    };
    auto share = [&](int which) {
        Sum<T_TERMS, 8> zf;
        zf.of_summed(joined(z[0], z[1]));
#pragma unroll
        for (int t = 0; t < T_TERMS; ++t) sz[which][wave][t][lane] = zf.term[t];
    };
    own_of(z);
    share(1);
    fetch();
    own += step;
    own_of(y);
    for (int i = 1; i < segments - 1; ++i) {
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
            for (int b = 0; b < 2; ++b) mf[k][b].of_summed(joined(rm[k][b][0], rm[k][b][1]));
        z[0] = y[0];
        z[1] = y[1];
        float* const to = own;
        if (i + 1 < segments - 1) {
            fetch();
            own += step;
            own_of(y);
        }
        __syncthreads();                                  // (the other room is read: its next writer is behind this)
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            Sum<T_TERMS, 8> zf;
#pragma unroll
            for (int t = 0; t < T_TERMS; ++t) zf.term[t] = sz[i & 1][k][t][lane];
            mfmas<true, 2>(z, mf[k], zf);
        }
        share(~i & 1);
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) to[(4 * b + r) * VW] = z[b][r];
    }
}

// ------------------------------------------------------------------------------------------------ the gradients
// A workgroup a chunk and head; a wave 16 of the keys' values.  First what sums over the values' columns: g S^T, y S^T and e X^T
// (transposed), with g, y and e in LDS and a wave's rows of S and X straight from memory, and the 16 x 16 blocks of g e^T and y e^T.
// Then q and k take their place, and H and Z as blocks of terms, which are read by rows for what sums over j and through the
// transposing read for what sums over i.
// 8 x 4,096 moments, 16 heads of 128 in bfloat16 take 750 us (880 where the card clocks lower), their 2.4 GB alone 450: one
// workgroup's 8 waves fill a CU's registers, so that its loads, 112 KB of terms and products follow one another; matrix
// instructions take 25% of the cycles.  (Two workgroups a CU, or one that walks several chunks, spill: slower.  Keys of up to 64
// values with values of more, bfloat16: 4 waves of 308 registers and 117 KB of LDS, one workgroup a CU: 626 us at 64 / 128.)
template <class T, int KT, int VT>
constexpr int grads_room() {                              // 16-bit values of LDS
    using F = DeltaForm<T, true>;
    constexpr int first = (F::X + 2 * F::W) * F::CH * 64 * VT, second = 2 * F::X * F::CH * 32 * KT + F::JB * (F::JB + 1) * F::W * 256;
    constexpr int third = 64 * KT * F::CH, most = first > second ? first : second;
    return most > third ? most : third;
}
// workgroups a CU that LDS lets in, and that registers are left for (waves a SIMD)
template <class T, int KT, int VT>
constexpr int grads_waves() {
    constexpr int fit = 78 * 1024 / grads_room<T, KT, VT>();
    constexpr int most = Form<T>::X == 3 ? 2 : 3;
    return KT == 4 ? 2 : fit < 1 ? 1 : fit > most ? most : fit;
}
template <class T, int KT, int VT>
__global__ __launch_bounds__(128 * KT, (grads_waves<T, KT, VT>())) void k_delta_grads(Delta a) {
    using F = DeltaForm<T, true>;
    constexpr int X = F::X, W = F::W, CH = F::CH, JB = F::JB, KW = 32 * KT, VW = 64 * VT, XP = CH * KW, VP = CH * VW, VN = Vec<T>::N;
    constexpr int WAVES_ = 2 * KT, THREADS = 64 * WAVES_, XC = KW / VN, VC = VW / VN, BLOCKS = JB * (JB + 1) / 2;
    constexpr int BLOCK = W * 256;
    __shared__ __align__(16) bf16 room[grads_room<T, KT, VT>()];
    __shared__ __align__(16) float hi[CH], lo[CH], sb[CH], se[CH], sw[CH], sums[4][CH], red_state[WAVES_];
    bf16 *const sg = room, *const sy = sg + X * VP, *const ser = sy + W * VP;
    bf16 *const sq = room, *const sk = sq + X * XP, *const sh = sk + X * XP;   // sh: [H, Z][block][W][16 i][16 j]
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, c = lane & 15;
    const unsigned block = (unsigned)block_number();
    const int place_in = (int)(block / a.heads), h = (int)(block - (unsigned)place_in * a.heads);
    if (place_in >= a.chunks.slots) return;
    int n, seg, slot;
    long long first, count;
    if (!segment_of(a.chunks, place_in, n, seg, slot, first, count)) return;
    const long long from = (long long)seg * CH, left = count - from;
    const int rows = (int)(left < CH ? left : CH);
    if (rows <= 0) return;
    const long long moment = first + from, out_row = (a.chunks.starts ? 0 : n * a.chunks.n_moments) + moment;
    const size_t mine = (size_t)slot * a.heads + h;
    const float* const f = factors_of<F>(a.prep + mine * F::PREP);
    constexpr int GN = CH * VC, EN = CH * VW / 8, QN = CH * XC;
    constexpr int GV = (GN + THREADS - 1) / THREADS, EV = (EN + THREADS - 1) / THREADS, QV = (QN + THREADS - 1) / THREADS;
    auto nth = [&](int i, int most) { return min(i * THREADS + tid, most - 1); };     // (a share past the last: it once more)
    u32x4 rg[GV], rq[QV], rk[QV];
    f32x4 ry[EV][2], re[EV][2], rs[VW / 32][2], rx[VW / 32][2];
    {                                                     // all at once, in the order that it is used in
        const Chunk<T> go = chunk_of<T>(a, a.go, n, h, moment, rows, a.V);
#pragma unroll
        for (int i = 0; i < GV; ++i) rg[i] = __builtin_bit_cast(u32x4, go(nth(i, GN) / VC, nth(i, GN) % VC * VN));
        const f32x4 *const ys = reinterpret_cast<const f32x4*>(a.ys + mine * CH * VW), *const es = reinterpret_cast<const f32x4*>(a.errors + mine * CH * VW);
#pragma unroll
        for (int i = 0; i < EV; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                ry[i][half] = ys[2 * nth(i, EN) + half];
                re[i][half] = es[2 * nth(i, EN) + half];
            }
        const size_t row = mine * KW * VW + (16 * wave + c) * VW + 8 * g;
#pragma unroll
        for (int b = 0; b < VW / 32; ++b)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                rs[b][half] = *reinterpret_cast<const f32x4*>(a.states + row + 32 * b + 4 * half);
                rx[b][half] = *reinterpret_cast<const f32x4*>(a.grads + row + 32 * b + 4 * half);
            }
    }
    if (tid < CH) {
        se[tid] = f[F_E + tid];
        sw[tid] = f[F_E + 2 * CH + tid];
        sb[tid] = f[F_E + 3 * CH + tid];
        hi[tid] = f[F_E + 4 * CH + tid];
        lo[tid] = f[F_E + 5 * CH + tid];
    }
    f32x4 x1[JB], x2[JB], x3[JB];
    float dot = 0.f;                                      // <S, X>
    constexpr int TASKS = 2 * BLOCKS, MOST = (TASKS + WAVES_ - 1) / WAVES_;
    f32x4 p[MOST];                                        // this wave's blocks of g e^T (task < BLOCKS) and y e^T: rows j, columns i
#pragma unroll
    for (int i = 0; i < JB; ++i) x1[i] = x2[i] = x3[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = 0; m < MOST; ++m) p[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    {
#pragma unroll
        for (int i = 0; i < GV; ++i) {
            const int row = nth(i, GN) / VC, col = nth(i, GN) % VC * VN;
            store_terms<T>(__builtin_bit_cast(uint4, rg[i]), sg + place<VW>(row, col >> 3) + (col & 7), VP);
        }
#pragma unroll
        for (int i = 0; i < EV; ++i) {
            const int at = nth(i, EN), row = at / (VW / 8), col = at % (VW / 8) * 8, to = place<VW>(row, col >> 3);
            const f32x8 y = joined(ry[i][0], ry[i][1]);
            if (a.gv && row < rows && col < a.V) {
                const long long to_v = ((out_row + row) * a.heads + h) * a.V + col;
                typedef T vec8 __attribute__((ext_vector_type(8)));
                if (a.vec && a.share == 1 && sizeof(T) == 2) *reinterpret_cast<vec8*>((T*)a.gv + to_v) = __builtin_convertvector(y, vec8);
                else
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (col + r < a.V) {
                            if (a.share > 1) ((float*)a.gv)[to_v + r] = y[r];
                            else ((T*)a.gv)[to_v + r] = narrow<T>(y[r]);
                        }
            }
            Sum<W, 8> ts, us;
            ts.of(y);
            us.of(joined(re[i][0], re[i][1]));
#pragma unroll
            for (int t = 0; t < W; ++t) {
                *reinterpret_cast<bf16x8*>(sy + to + t * VP) = ts.term[t];
                *reinterpret_cast<bf16x8*>(ser + to + t * VP) = us.term[t];
            }
        }
        __syncthreads();
        {
            const Chunk<T> cq = chunk_of<T>(a, a.q, n, h, moment, rows, a.K), ck = chunk_of<T>(a, a.k, n, h / a.share, moment, rows, a.K);
#pragma unroll
            for (int i = 0; i < QV; ++i) {
                rq[i] = __builtin_bit_cast(u32x4, cq(nth(i, QN) / XC, nth(i, QN) % XC * VN));
                rk[i] = __builtin_bit_cast(u32x4, ck(nth(i, QN) / XC, nth(i, QN) % XC * VN));
            }
        }
#pragma unroll
        for (int b = 0; b < VW / 32; ++b) {
            const f32x8 s = joined(rs[b][0], rs[b][1]), x = joined(rx[b][0], rx[b][1]);
#pragma unroll
            for (int r = 0; r < 8; ++r) dot = fmaf(s[r], x[r], dot);
            Sum<W, 8> st, xt;
            st.of_summed(s);
            xt.of_summed(x);
            const int at = place<VW>(c, g) ^ 32 * b;
#pragma unroll
            for (int i = 0; i < JB; ++i) {
                x1[i] = mfma(st, across<X>(sg + 16 * i * VW + at, VP), x1[i]);
                x2[i] = mfma(st, across<W>(sy + 16 * i * VW + at, VP), x2[i]);
                x3[i] = mfma(xt, across<W>(ser + 16 * i * VW + at, VP), x3[i]);
            }
        }
#pragma unroll
        for (int m = 0; m < MOST; ++m) {
            const int task = WAVES_ * m + wave;
            if (task >= TASKS) break;
            int i, j;
            block_of(task < BLOCKS ? task : task - BLOCKS, i, j);
            const bf16 *const pe = ser + 16 * j * VW, *const pg = sg + 16 * i * VW, *const py = sy + 16 * i * VW;
            if (task < BLOCKS) {
#pragma unroll
                for (int b = 0; b < VW / 32; ++b) {
                    const int at = place<VW>(c, g) ^ 32 * b;
                    p[m] = mfma(across<W>(pe + at, VP), across<X>(pg + at, VP), p[m]);
                }
            } else {
#pragma unroll
                for (int b = 0; b < VW / 32; ++b) {
                    const int at = place<VW>(c, g) ^ 32 * b;
                    p[m] = mfma(across<W>(pe + at, VP), across<W>(py + at, VP), p[m]);
                }
            }
        }
    }
    __syncthreads();                                      // (g, y and e are read)
#pragma unroll
    for (int m = 0; m < MOST; ++m) {
        const int task = WAVES_ * m + wave;
        if (task >= TASKS) break;
        const bool of_z = task >= BLOCKS;
        int i, j;
        block_of(of_z ? task - BLOCKS : task, i, j);
        const int row = 16 * i + c;
        const f32x4 hj = *reinterpret_cast<const f32x4*>(&hi[16 * j + 4 * g]), lj = *reinterpret_cast<const f32x4*>(&lo[16 * j + 4 * g]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int col = 16 * j + 4 * g + r;
            const float d = exp_of(fminf((hi[row] - hj[r]) + (lo[row] - lj[r]), 88.f));
            p[m][r] = of_z ? (row > col ? -d * p[m][r] : 0.f) : (row >= col ? a.c * d * p[m][r] : 0.f);
        }
        Sum<W, 4> t4;
        t4.of_summed(p[m]);
#pragma unroll
        for (int t = 0; t < W; ++t) *reinterpret_cast<bf16x4*>(sh + task * BLOCK + t * 256 + c * 16 + 4 * (g ^ (c >> 2))) = t4.term[t];
    }
#pragma unroll
    for (int i = 0; i < QV; ++i) {
        const int at = nth(i, QN), row = at / XC, col = at % XC * VN, to = place<KW>(row, col >> 3) + (col & 7);
        store_terms<T>(__builtin_bit_cast(uint4, rq[i]), sq + to, XP);
        store_terms<T>(__builtin_bit_cast(uint4, rk[i]), sk + to, XP);
    }
    __syncthreads();
    typedef __attribute__((address_space(3))) s16x4* at_lds;
    // this lane's 4 values of row c; of the transposing read (the shares of row 4n + m exchanged by n: rows 4 apart share banks)
    const bf16* const by_row = sh + c * 16 + 4 * (g ^ (c >> 2));
    const bf16* const turned = sh + (4 * g + (c >> 2)) * 16 + 4 * ((c & 3) ^ g);
    auto number = [](int i, int j) { return i * (i + 1) / 2 + j; };
    // columns i of H (set 0) or Z, summed over moments j of blocks 2jj, 2jj + 1
    auto rows_of = [&](int set, int jj, int i) {
        Sum<W, 8> s;
#pragma unroll
        for (int t = 0; t < W; ++t) {
            bf16x4 v[2] = {};
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (2 * jj + e <= i) v[e] = *reinterpret_cast<const bf16x4*>(by_row + (set * BLOCKS + number(i, 2 * jj + e)) * BLOCK + t * 256);
            s.term[t] = __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return s;
    };
    // columns j of the transpose, summed over moments i of blocks 2ii, 2ii + 1
    auto columns_of = [&](int set, int ii, int j) {
        Sum<W, 8> s;
#pragma unroll
        for (int t = 0; t < W; ++t) {
            bf16x4 v[2] = {};
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (2 * ii + e >= j)
                    v[e] = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (at_lds)(turned + (set * BLOCKS + number(2 * ii + e, j)) * BLOCK + t * 256)));
            s.term[t] = __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return s;
    };
    float dots[4][JB] = {};
    const int krow = place<KW>(c, 2 * wave + (g >> 1)) + 4 * (g & 1), kc = 16 * wave + 4 * g;        // 4 values of row c, from there
#pragma unroll
    for (int i = 0; i < JB; ++i) {
        const float e = se[16 * i + c], w = sw[16 * i + c];
        const f32x4 k4 = widened<X>(sk + 16 * i * KW + krow, XP);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            dots[3][i] = fmaf(k4[r], x3[i][r], dots[3][i]);
            x1[i][r] *= a.c * e;
            x2[i][r] *= -e;
            x3[i][r] *= w;
        }
    }
    // (a step's operands are read before the products of the step before)
    Sum<X, 8> kt[JB / 2], qt[JB / 2];
    Sum<W, 8> kb[JB / 2];                                 // k times its rate
#pragma unroll
    for (int jj = 0; jj < JB / 2; ++jj) {
        const int at = 32 * jj * KW + place<KW>(4 * g + (c >> 2), 2 * wave + (c >> 1 & 1)) + 4 * (c & 1);
        kt[jj] = down<X>(sk + at, 16 * KW, XP);
        qt[jj] = down<X>(sq + at, 16 * KW, XP);
    }
    constexpr int STEPS = 2 * F::PIECES;                  // each piece by rows, then each of the transposes
    Sum<W, 8> hz[2][2];
    auto read_step = [&](int step) {
        const int m = step % F::PIECES, jj = m >= JB, i = jj ? m - JB + 2 : m, ii = m >= 2, j = ii ? m - 2 : m;
        hz[step & 1][0] = step < F::PIECES ? rows_of(0, jj, i) : columns_of(0, ii, j);
        hz[step & 1][1] = step < F::PIECES ? rows_of(1, jj, i) : columns_of(1, ii, j);
    };
    read_step(0);
#pragma unroll
    for (int jj = 0; jj < JB / 2; ++jj)
        kb[jj].of_summed(widened(kt[jj]) * joined(*reinterpret_cast<const f32x4*>(&sb[32 * jj + 4 * g]),
                                                  *reinterpret_cast<const f32x4*>(&sb[32 * jj + 16 + 4 * g])));
#pragma unroll
    for (int step = 0; step < STEPS; ++step) {
        const int m = step % F::PIECES, jj = m >= JB, i = jj ? m - JB + 2 : m, ii = m >= 2, j = ii ? m - 2 : m;
        if (step + 1 < STEPS) read_step(step + 1);
        in_order();
        if (step < F::PIECES) {
            f32x4 two[2] = {x1[i], x2[i]};
            mfmas<false, 2>(two, hz[step & 1], kb[jj]);   // (two sums at a time: no product waits for the one before it)
            x1[i] = two[0];
            x2[i] = two[1];
        } else {
            f32x4 two[2] = {x3[j], f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int t = W - 1; t >= 0; --t)
#pragma unroll
                for (int u = 0; u < X; ++u)
                    if (t + u < W) {
                        two[0] = mfma(qt[ii].term[u], hz[step & 1][0].term[t], two[0]);
                        two[1] = mfma(kt[ii].term[u], hz[step & 1][1].term[t], two[1]);
                    }
            x3[j] = two[0] + two[1];
        }
        in_order();
    }
    typedef T vec4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int i = 0; i < JB; ++i) {
        const f32x4 k4 = widened<X>(sk + 16 * i * KW + krow, XP), q4 = widened<X>(sq + 16 * i * KW + krow, XP);
        const int row = 16 * i + c;
        f32x4 gk;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            dots[0][i] = fmaf(q4[r], x1[i][r], dots[0][i]);
            dots[1][i] = fmaf(k4[r], x2[i][r], dots[1][i]);
            dots[2][i] = fmaf(k4[r], x3[i][r], dots[2][i]);
            gk[r] = fmaf(sb[row], x3[i][r], x2[i][r]);
        }
        if (row >= rows || kc >= a.K) continue;
        const long long at = ((out_row + row) * a.heads + h) * a.K + kc;
        if (a.vec) {
            if (a.gq) *reinterpret_cast<vec4*>((T*)a.gq + at) = __builtin_convertvector(x1[i], vec4);
            if (a.gk && a.share > 1) *reinterpret_cast<f32x4*>((float*)a.gk + at) = gk;
            else if (a.gk) *reinterpret_cast<vec4*>((T*)a.gk + at) = __builtin_convertvector(gk, vec4);
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (kc + r >= a.K) continue;
                if (a.gq) ((T*)a.gq)[at + r] = narrow<T>(x1[i][r]);
                if (a.gk && a.share > 1) ((float*)a.gk)[at + r] = gk[r];
                else if (a.gk) ((T*)a.gk)[at + r] = narrow<T>(gk[r]);
            }
        }
    }
    if (!a.glog_decay && !a.gbeta) return;
    __syncthreads();                                      // (q, k, H and Z are read)
    float* const red = reinterpret_cast<float*>(room);    // [wave][g][4][CH], the 16s of a g exchanged by it
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < JB; ++i) red[(wave * 4 + g) * 4 * CH + ((d * CH + 16 * i + c) ^ (16 * g))] = dots[d][i];
    dot = wave_sum(dot, 64);
    if (lane == 0) red_state[wave] = dot;
    __syncthreads();
    if (tid < 4 * CH) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < 4 * WAVES_; ++w) s += red[w * 4 * CH + (tid ^ (16 * (w & 3)))];
        sums[tid / CH][tid % CH] = s;
    }
    __syncthreads();
    if (wave == 0) {
        float s[4], sx = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES_; ++w) sx += red_state[w];
#pragma unroll
        for (int d = 0; d < 4; ++d) s[d] = lane < CH ? sums[d][lane] : 0.f;
        const float b = lane < CH ? sb[lane] : 0.f;
        float gg = s[0] + s[1] - b * s[2], end = lane < CH ? sw[lane] * b * s[3] : 0.f;
        end = wave_sum(end, 64) + (f[0] + f[1]) * sx;
        for (int m = 1; m < 64; m <<= 1) {
            const float t = __shfl_down(gg, m);
            if (lane + m < 64) gg += t;
        }
        const long long at = (out_row + lane) * a.heads + h;
        if (lane < rows && a.glog_decay) a.glog_decay[at] = gg + end;
        if (lane < rows && a.gbeta) a.gbeta[at] = s[2];
    }
}

// gradients of shared heads: out[m][j][d] = the sum over a key head's query heads of part[m][share j + i][d]; the first `first`
// workgroups those of k, the rest those of v
template <class T>
__global__ __launch_bounds__(256) void k_delta_share(const float* part_k, T* out_k, int K, long long nk, long long first,
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

// Packed moments before the first stretch and after the last one: zeros in each output.  grid (workgroups, outputs)
struct Outside {
    char* out[8];
    long long row[8];                    // bytes a moment
};
__global__ __launch_bounds__(256) void k_delta_outside(Cuts a, Outside z) {
    long long first = 0, rest = a.n_moments, before = 0;
    if (a.n_seq) {
        leaf_of(a, a.n_seq, first, rest);
        before = bound_of(a, 0);
    }
    const long long row = z.row[blockIdx.y];
    auto clear = [&](uintptr_t from, uintptr_t to) {      // (4-byte words, or 2-byte values at the ends)
        for (uintptr_t p = from + 4 * ((uintptr_t)blockIdx.x * 256 + threadIdx.x); p < to; p += 4 * 256 * (uintptr_t)gridDim.x) {
            if (!(from & 3) && p + 4 <= to) *(unsigned*)p = 0;
            else {
                *(unsigned short*)p = 0;
                if (p + 2 < to) *(unsigned short*)(p + 2) = 0;
            }
        }
    };
    const uintptr_t out = (uintptr_t)z.out[blockIdx.y];
    clear(out, out + before * row);
    clear(out + first * row, out + (first + rest) * row);
}

// ------------------------------------------------------------------------------------------------ one moment
// A workgroup takes CB columns of a row's state of one head, CB / 4 lanes a row of it, every (1024 / CB)th row a lane, all a
// lane's loads under way at once.  What the state holds under the key, S^T k, and what the query reads of it, S^T q, are joined over
// rows in one go, as o = c (S^T q + (q . k) beta e) needs no second pass.
// VEC: 16-byte loads and stores of the states (v_dim a multiple of 4, states aligned).  grid (blocks of columns, heads, rows)
template <class T, int CB, bool VEC>
__global__ __launch_bounds__(256) void k_delta_step(fm_delta_step_args a) {
    constexpr int LR = CB / 4, RG = 256 / LR, PER = DELTA_MAX / RG;
    __shared__ float part[4][2 * CB + 1];
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
    float4 s[PER];
    float kr[PER], qr[PER], vv[4];
    // (lanes past the state's rows and columns load its first ones, which nothing uses: branches would make the loads wait for one
    // another: 416 rows, 8 heads of 128 x 128 in bfloat16, 94 us instead of 87)
    auto load = [&](const float* p) {
        if (VEC) return *reinterpret_cast<const float4*>(p + (c0 < N ? c0 : 0));
        return make_float4(p[c0 < N ? c0 : 0], p[c0 + 1 < N ? c0 + 1 : 0], p[c0 + 2 < N ? c0 + 2 : 0], p[c0 + 3 < N ? c0 + 3 : 0]);
    };
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = rg + i * RG;
        const int there = r < K ? r : 0;
        s[i] = load(a.state + at + (size_t)there * N);
        kr[i] = widen(k[there]);
        qr[i] = widen(q[there]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) vv[j] = widen(v[c0 + j < N ? c0 + j : 0]);
    const float log_decay = a.log_decay[n * a.ld_row + h * a.ld_head], beta = a.beta[n * a.be_row + h * a.be_head];
    const Keep keep(log_decay);
    float sum[9] = {};                                    // S^T k, S^T q of 4 columns; q . k
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (rg + i * RG >= K) break;
        s[i] = make_float4(keep(s[i].x), keep(s[i].y), keep(s[i].z), keep(s[i].w));
        const float x[4] = {s[i].x, s[i].y, s[i].z, s[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            sum[j] = fmaf(kr[i], x[j], sum[j]);
            sum[4 + j] = fmaf(qr[i], x[j], sum[4 + j]);
        }
        sum[8] = fmaf(qr[i], kr[i], sum[8]);
    }
#pragma unroll
    for (int m = LR; m < 64; m <<= 1)
#pragma unroll
        for (int j = 0; j < 9; ++j) sum[j] += __shfl_xor(sum[j], m);
    if ((tid & 63) < LR) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            part[tid >> 6][4 * cg + j] = sum[j];
            part[tid >> 6][CB + 4 * cg + j] = sum[4 + j];
        }
        if (cg == 0) part[tid >> 6][2 * CB] = sum[8];
    }
    __syncthreads();
    auto joined_at = [&](int i) { return part[0][i] + part[1][i] + part[2][i] + part[3][i]; };
    float u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        // (a value, key, decay or rate that is not finite: NaN in all that it reaches, also where an infinite decay meets a state of 0
        // or an infinite step a key of any sign)
        u[j] = beta * (vv[j] - joined_at(4 * cg + j));
        if (!(fabsf(u[j]) < INFINITY) || !(log_decay < INFINITY)) u[j] = NAN;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = rg + i * RG;
        if (r >= K) break;
        s[i] = make_float4(fmaf(kr[i], u[0], s[i].x), fmaf(kr[i], u[1], s[i].y), fmaf(kr[i], u[2], s[i].z), fmaf(kr[i], u[3], s[i].w));
        float* p = a.next + at + (size_t)r * N + c0;
        if (VEC) {
            if (c0 < N) *reinterpret_cast<float4*>(p) = s[i];
        } else {
            if (c0 < N) p[0] = s[i].x;
            if (c0 + 1 < N) p[1] = s[i].y;
            if (c0 + 2 < N) p[2] = s[i].z;
            if (c0 + 3 < N) p[3] = s[i].w;
        }
    }
    if (rg == 0) {
        const float qk = joined_at(2 * CB);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (4 * cg + j < cols) o[4 * cg + j] = narrow<T>((float)a.scale * fmaf(qk, u[j], joined_at(CB + 4 * cg + j)));
    }
}

// ------------------------------------------------------------------------------------------------ host
const char* delta_heads_wrong(long long dtype, long long qh, long long kh, long long kd, long long vd) {
    if (dtype < FM_F32 || dtype > FM_F16) return "values of an unknown type";
    if (qh < 1 || kh < 1 || qh % kh || qh > 65535) return "query heads must be a multiple of key heads, at most 65535";
    if (kd < 1 || kd > DELTA_MAX || vd < 1 || vd > DELTA_MAX) return "heads of other than 1 to 128 values";
    return nullptr;
}
bool share_memory(const float* a, const float* b, long long n) {
    return a && b && (uintptr_t)a < (uintptr_t)b + 4 * n && (uintptr_t)b < (uintptr_t)a + 4 * n;
}
const char* delta_wrong(const fm_delta_args& a, bool bwd, bool sizes_only = false) {
    if (const char* e = delta_heads_wrong(a.dtype, a.q_heads, a.k_heads, a.k_dim, a.v_dim)) return e;
    if (a.n_seq < 0 || a.n_seq > 16384) return "other than 0 to 16384 stretches";
    if (a.n_moments < 0 || a.n_moments > 1LL << 31) return "other than 0 to 2^31 moments";
    if ((double)a.n_moments * (a.starts ? 1 : (double)a.n_seq) * (double)a.q_heads > 8e9) return "more than 8e9 heads of moments";
    if (sizes_only) return nullptr;
    const bool any = a.n_seq && a.n_moments;
    if (any && (!a.q.data || !a.k.data || !a.v.data || !a.log_decay || !a.beta)) return "a null tensor";
    if (!bwd && a.n_moments && (a.n_seq || a.starts) && !a.o) return "a null tensor";
    if (!bwd && share_memory(a.state, a.state_out, a.n_seq * a.q_heads * a.k_dim * a.v_dim)) return "state_out must not be state";
    if (bwd && any && (!a.go.data || !a.saved)) return "a null tensor";
    return nullptr;
}

int chunk_length(long long dtype) { return dtype == FM_BF16 ? Form<bf16>::CHUNK : Form<float>::CHUNK; }
template <bool BWD>
long long prep_bytes_of(long long dtype) {
    return dtype == FM_BF16 ? DeltaForm<bf16, BWD>::PREP : dtype == FM_F16 ? DeltaForm<f16, BWD>::PREP : DeltaForm<float, BWD>::PREP;
}
long long prep_bytes(long long dtype, bool bwd) { return bwd ? prep_bytes_of<true>(dtype) : prep_bytes_of<false>(dtype); }
long long chunk_slots(const fm_delta_args& a) {
    const long long C = chunk_length(a.dtype), most = (a.n_moments + C - 1) / C;
    if (!a.n_seq || !a.n_moments) return 0;
    return a.starts && most > 1 ? a.n_moments / C + a.n_seq : a.n_seq * most;
}
// Segments: a walk takes a workgroup for 64 columns and a CU for itself, so that few chains leave most CUs without work.  Cut
// into segments of L moments, these are walked at the same time, for more work: their own end states, with M (K more columns) but
// for the first, then those joined one after another, then the walk.  The choice is by an estimate whose constants are fitted, in
// units of about a microsecond: a chunk takes a walk `chunk`, four fifths of it where only the own state is wanted, a join `join`, the
// launches 12; workgroups go 256 at a time.  (Whole walks of bfloat16 took 3.0 us a chunk at heads of 64, 4.0 at 128, up to 6.2 where
// chunks are kept and all CUs walk, a join 2.6: the longer the walks, the more joins and launches weigh beside them.  The half in
// `rounds` for heads of up to 64 is the fit's: registers and LDS let a second workgroup into a CU for some of binary16's walks and
// float32's own states, for none of bfloat16's.  Whether gradients are wanted is not asked: M serves both, and both are cut alike.)
// Packed stretches, whose lengths only the device knows, are taken to be of any length up to twice the middle one.
// Fitted to 84 calls measured with 1 to 64 segments: each type, heads of 64 and 128, 1 to 37 stretches of 1,024 to 32,768 moments,
// with gradients and without.  In that same table, interpolated between the counts measured, the choice takes 1.02 times the best
// one's time in the middle, 1.18 at most, walks without segments 2.4 in the middle, 18 at most: 1 x 4 heads of 128 x 16,384 of bfloat16
// 1,012 us whole and 183 in 16 segments; 16 x 8 x 1,024 108 and 172 in two.  Calls outside the table were not timed.
long long segment_length(const fm_delta_args& p) {
    const long long C = chunk_length(p.dtype), whole = (p.n_moments + C - 1) / C * C;
    if (!p.n_seq || whole <= C) return whole ? whole : C;
    const bool packed = p.starts && p.n_seq > 1, deep = p.k_dim > 64;
    const double chunk = p.dtype == FM_F32 ? 3.4 : 2.4, join = deep ? 2.5 : 0.8, BV = p.v_dim <= 64 ? 1 : 2, BK = deep ? 2 : 1;
    const double middle = (double)p.n_moments / (packed ? p.n_seq : 1), longest = packed ? fmin(2 * middle, (double)p.n_moments) : middle;
    const double chains = (double)p.n_seq * p.q_heads, chunks = ceil(longest / C);
    auto rounds = [deep](double groups) {
        const double x = groups / 256;
        return fmax(1.0, deep ? ceil(x) : (x + ceil(x)) / 2);
    };
    double best = chunk * fmax(chunks, chains * BV * ceil(middle / C) / 256);
    long long L = whole;
    for (int nseg = 2; nseg <= 256; nseg += nseg < 16 ? 1 : nseg / 8) {
        const double each = ceil(chunks / nseg);
        if (each < 1 || each >= chunks) continue;
        const double mean = packed ? middle / (each * C) + 0.5 : ceil(chunks / each);            // segments a chain
        const double t = rounds(chains * BV * mean) * each * chunk +
                         rounds(chains * (BV * fmax(0.0, mean - 1) + BK * fmax(0.0, mean - 2))) * each * 0.8 * chunk +
                         fmax(0.0, ceil(chunks / each) - 2) * join + 12;
        if (t < best) {
            best = t;
            L = (long long)each * C;
        }
        if (each == 1) break;
    }
    return L;
}
long long segment_slots(const fm_delta_args& p) {
    const long long L = segment_length(p), most = (p.n_moments + L - 1) / L;
    return p.starts && most > 1 ? p.n_moments / L + p.n_seq : p.n_seq * (most > 1 ? most : 1);
}
bool in_segments(const fm_delta_args& p) { return p.n_seq && p.n_moments > segment_length(p); }
Cuts cuts_of(const fm_delta_args& p, long long L, int slots) {
    const long long most = (p.n_moments + L - 1) / L;
    return Cuts{p.starts, p.n_moments, L, L, (int)p.wide, (int)p.n_seq, (int)(most > 1 ? most : 1), slots};
}
// floats of a state or of a chunk's rows, padded as the kernels hold them
long long state_floats(const fm_delta_args& a) { return (a.k_dim <= 64 ? 64 : 128) * (a.v_dim <= 64 ? 64LL : 128); }
long long row_floats(const fm_delta_args& a) { return chunk_length(a.dtype) * (a.v_dim <= 64 ? 64LL : 128); }
// floats of segments' states, of their M
long long cut_floats(const fm_delta_args& a) { return in_segments(a) ? segment_slots(a) * a.q_heads * state_floats(a) : 0; }
long long move_floats(const fm_delta_args& a) {
    const long long KW = a.k_dim <= 64 ? 64 : 128;
    return in_segments(a) ? segment_slots(a) * a.q_heads * KW * KW : 0;
}
long long kept_floats(const fm_delta_args& a) { return chunk_slots(a) * a.q_heads * (state_floats(a) + row_floats(a)); }
long long turned_bytes(const fm_delta_args& a) { return chunk_slots(a) * a.q_heads * prep_bytes(a.dtype, true); }
long long delta_saved_bytes(const fm_delta_args& a) { return 4 * (kept_floats(a) + move_floats(a)) + turned_bytes(a); }
// float32 parts of shared key / value heads' gradients
long long delta_part_floats(const fm_delta_args& a, bool of_v) {
    const long long moments = a.n_moments * (a.starts ? 1 : a.n_seq);
    return a.q_heads > a.k_heads ? (moments * a.q_heads * (of_v ? a.v_dim : a.k_dim) + 3) / 4 * 4 : 0;
}
// whether the kernels can load these tensors as they are: heads of whole 16-byte units, aligned, a chunk's rows within 2^30 bytes
bool in_whole_units(const fm_delta_args& p, bool bwd) {
    const int size = p.dtype == FM_F32 ? 4 : 2;
    if (p.k_dim * size % 16 || p.v_dim * size % 16) return false;
    for (const fm_view* v : {&p.q, &p.k, bwd ? &p.go : &p.v})
        if (!aligned16(*v, size) || v->moment < 0 || v->moment >= STRIDE_MOST) return false;
    return true;
}
// Whether dense tensors of these sizes have moments too far apart for that: their copies' room is then counted for any strides, so that
// what a call takes goes by sizes alone wherever tensors are dense or aligned as in_whole_units wants them (the output's gradient
// need not be known when room is asked for).
bool far_apart(const fm_delta_args& p, bool bwd) {
    const long long third = (bwd ? p.q_heads : p.k_heads) * p.v_dim, row = p.q_heads * p.k_dim;
    return (row > third ? row : third) >= STRIDE_MOST;
}
// bytes of their copies: queries, keys, and values or (gradient) the output's gradient
long long pack_bytes(const fm_delta_args& p, bool bwd, int which) {
    const int size = p.dtype == FM_F32 ? 4 : 2;
    const long long moments = p.n_moments * (p.starts ? 1 : p.n_seq), K = (p.k_dim * size + 15) / 16, V = (p.v_dim * size + 15) / 16;
    return 16 * moments * (which == 0 ? p.q_heads * K : which == 1 ? p.k_heads * K : (bwd ? p.q_heads : p.k_heads) * V);
}
bool whole_stores(const fm_delta_args& p) {
    const int size = p.dtype == FM_F32 ? 4 : 2;
    return p.k_dim * size % 16 == 0 && p.v_dim * size % 16 == 0 &&
           !(((uintptr_t)p.o | (uintptr_t)p.gq | (uintptr_t)p.gk | (uintptr_t)p.gv) & 15);
}

long long delta_workspace_bytes(const fm_delta_args& a, bool bwd) {
    long long n = (bwd ? 0 : chunk_slots(a) * a.q_heads * prep_bytes(a.dtype, false)) + 4 * cut_floats(a);
    n += 4 * (bwd ? kept_floats(a) + delta_part_floats(a, false) + delta_part_floats(a, true) : move_floats(a));
    if (chunk_slots(a) && (!in_whole_units(a, bwd) || far_apart(a, bwd)))
        for (int i = 0; i < 3; ++i) n += pack_bytes(a, bwd, i);
    return n;
}


Delta delta_of(const fm_delta_args& p, bool bwd) {
    Delta a{};
    a.q = p.q;
    a.k = p.k;
    a.v = p.v;
    a.go = p.go;
    a.log_decay = p.log_decay;
    a.beta = p.beta;
    a.ld_seq = p.ld_seq;
    a.ld_moment = p.ld_moment;
    a.ld_head = p.ld_head;
    a.be_seq = p.be_seq;
    a.be_moment = p.be_moment;
    a.be_head = p.be_head;
    const long long C = chunk_length(p.dtype);
    a.chunks = cuts_of(p, C, (int)chunk_slots(p));
    const long long L = segment_length(p);
    a.segs = cuts_of(p, L, (int)segment_slots(p));
    a.heads = (int)p.q_heads;
    a.share = (int)(p.q_heads / p.k_heads);
    a.K = (int)p.k_dim;
    a.V = (int)p.v_dim;
    a.c = (float)p.scale;
    a.vec = whole_stores(p);
    const long long states = chunk_slots(p) * p.q_heads * state_floats(p);
    a.states = (float*)p.saved;
    a.errors = a.states ? a.states + states : nullptr;
    a.turned = a.errors ? (char*)(a.errors + chunk_slots(p) * p.q_heads * row_floats(p) + move_floats(p)) : nullptr;
    a.prep = bwd ? a.turned : (char*)p.workspace;
    float* room = (float*)((char*)p.workspace + (bwd ? 0 : chunk_slots(p) * p.q_heads * prep_bytes(p.dtype, false)));
    a.own = room;
    room += cut_floats(p);
    a.trans_t = a.errors ? a.errors + chunk_slots(p) * p.q_heads * row_floats(p) : nullptr;
    if (bwd) {
        a.grads = room;
        a.ys = a.grads + states;
    } else {
        a.trans = room;
    }
    a.init = p.state;
    a.fin = p.state_out;
    a.o = p.o;
    a.gfin = p.gstate_out;
    a.ginit = p.gstate;
    a.gq = p.gq;
    a.gk = p.gk;
    a.gv = p.gv;
    a.glog_decay = p.glog_decay;
    a.gbeta = p.gbeta;
    return a;
}

// a launch of the walks: 8 segments' blocks of columns at a time
dim3 walks_of(const Delta& a, int blocks) { return blocks_of(((long long)a.segs.slots * a.heads + 7) / 8 * 8 * blocks); }
template <class T, int KT>
void delta_fwd(const Delta& a, hipStream_t st) {
    const int BV = (a.V + 63) / 64;
    const dim3 chunks = a.chunks.slots ? blocks_of((long long)a.chunks.slots * a.heads) : dim3(1);
    if (a.chunks.slots && a.turned) k_delta_prep<T, KT, true><<<chunks, 256, 0, st>>>(a);
    else if (a.chunks.slots) k_delta_prep<T, KT, false><<<chunks, 256, 0, st>>>(a);
    if (a.segs.nseg > 1) {
        k_delta_scan<T, KT, OWN><<<walks_of(a, BV + KT / 2), 256, 0, st>>>(a);
        if (a.segs.nseg > 2) k_delta_join<KT, false><<<dim3(4 * BV * a.heads, a.segs.n_seq), 64 * KT, 0, st>>>(a);
    }
    if (a.states) k_delta_scan<T, KT, KEEP><<<walks_of(a, BV), 256, 0, st>>>(a);
    else k_delta_scan<T, KT, PLAY><<<walks_of(a, BV), 256, 0, st>>>(a);
}
template <class T, int KT>
void delta_bwd(const Delta& a, hipStream_t st) {
    const int BV = (a.V + 63) / 64;
    if (a.segs.nseg > 1) {
        k_delta_back<T, KT, OWN><<<walks_of(a, BV), 256, 0, st>>>(a);
        if (a.segs.nseg > 2) k_delta_join<KT, true><<<dim3(4 * BV * a.heads, a.segs.n_seq), 64 * KT, 0, st>>>(a);
    }
    k_delta_back<T, KT, KEEP><<<walks_of(a, BV), 256, 0, st>>>(a);
    if (!a.chunks.slots || !(a.gq || a.gk || a.gv || a.glog_decay || a.gbeta)) return;
    const dim3 chunks = blocks_of((long long)a.chunks.slots * a.heads);
    if (a.V <= 64) k_delta_grads<T, KT, 1><<<chunks, 128 * KT, 0, st>>>(a);
    else k_delta_grads<T, KT, 2><<<chunks, 128 * KT, 0, st>>>(a);
}

template <class T>
void delta_of_type(const fm_delta_args& p, bool bwd, hipStream_t st) {
    Delta a = delta_of(p, bwd);
    if (p.starts && p.n_moments) {
        const int size = sizeof(T);
        Outside z{};
        int n = 0;
        auto add = [&](void* out, long long row) {
            if (!out) return;
            z.out[n] = (char*)out;
            z.row[n++] = row;
        };
        if (!bwd) add(p.o, p.q_heads * p.v_dim * size);
        else {
            const int ks = a.share > 1 && p.n_seq ? 0 : size;             // (shared heads: their parts, below)
            add(p.gq, p.q_heads * p.k_dim * size);
            if (ks) add(p.gk, p.k_heads * p.k_dim * size);
            if (ks) add(p.gv, p.k_heads * p.v_dim * size);
            add(p.glog_decay, p.q_heads * 4);
            add(p.gbeta, p.q_heads * 4);
        }
        if (bwd && a.share > 1 && p.n_seq) {
            float* part = a.grads + chunk_slots(p) * p.q_heads * (state_floats(p) + row_floats(p));
            if (p.gk) add(part, p.q_heads * p.k_dim * 4);
            if (p.gv) add(part + delta_part_floats(p, false), p.q_heads * p.v_dim * 4);
        }
        if (n) k_delta_outside<<<dim3(256, n), 256, 0, st>>>(a.chunks, z);
    }
    if (!p.n_seq) return;
    if (a.chunks.slots && !in_whole_units(p, bwd)) {
        Packs k{};
        char* to = (char*)p.workspace + delta_workspace_bytes(p, bwd);
        fm_view* const views[3] = {&a.q, &a.k, bwd ? &a.go : &a.v};
        k.n_moments = p.n_moments;
        k.moments = p.n_moments * (p.starts ? 1 : p.n_seq);
        for (int i = 2; i >= 0; --i) {
            to -= pack_bytes(p, bwd, i);
            k.from[i] = *views[i];
            k.to[i] = to;
            k.heads[i] = i == 0 || (i == 2 && bwd) ? a.heads : (int)p.k_heads;
            k.width[i] = i == 2 ? a.V : a.K;
            const long long row = (k.width[i] + Vec<T>::N - 1) / Vec<T>::N * Vec<T>::N;
            *views[i] = fm_view{to, p.n_moments * k.heads[i] * row, k.heads[i] * row, row};
        }
        k_delta_pack<T><<<dim3(2048, 3), 256, 0, st>>>(k);
    }
    float *part_k = nullptr, *part_v = nullptr;
    if (bwd && a.share > 1) {
        part_k = a.grads + chunk_slots(p) * p.q_heads * (state_floats(p) + row_floats(p));
        part_v = part_k + delta_part_floats(p, false);
        a.gk = p.gk ? part_k : nullptr;
        a.gv = p.gv ? part_v : nullptr;
    }
    if (bwd) p.k_dim <= 64 ? delta_bwd<T, 2>(a, st) : delta_bwd<T, 4>(a, st);
    else p.k_dim <= 64 ? delta_fwd<T, 2>(a, st) : delta_fwd<T, 4>(a, st);
    if (!part_k) return;
    const long long rows = p.n_moments * (p.starts ? 1 : p.n_seq) * p.k_heads;
    const long long nk = p.gk ? rows * p.k_dim : 0, nv = p.gv ? rows * p.v_dim : 0;
    const long long bk = (nk + 255) / 256, bv = (nv + 255) / 256;
    if (bk + bv)
        k_delta_share<T><<<blocks_of(bk + bv), 256, 0, st>>>(part_k, (T*)p.gk, (int)p.k_dim, nk, bk, part_v, (T*)p.gv,
                                                             (int)p.v_dim, nv, a.share);
}

int delta(const fm_delta_args* args, bool bwd, void* stream) {
    const std::string name = bwd ? "fm_delta_bwd: " : "fm_delta: ";
    clear_error();
    if (!args) return fail((name + "no arguments").c_str());
    if (const char* e = delta_wrong(*args, bwd)) return fail((name + e).c_str());
    const long long need = delta_workspace_bytes(*args, bwd);
    if (need && (!args->workspace || args->workspace_bytes < need)) return fail((name + "the workspace is too small").c_str());
    const long long kept = delta_saved_bytes(*args);
    if (kept && args->saved && args->saved_bytes < kept) return fail((name + "saved is too small").c_str());
    hipStream_t st = (hipStream_t)stream;
    if (args->dtype == FM_F32) delta_of_type<float>(*args, bwd, st);
    else if (args->dtype == FM_BF16) delta_of_type<bf16>(*args, bwd, st);
    else delta_of_type<f16>(*args, bwd, st);
    FG_CHECK(hipGetLastError(), -1);
    return 0;
}

// 32 columns a workgroup, or 64 where that makes two workgroups a CU or more and leaves no half of one idle.  With 32 and 64 columns,
// us: 416 rows, 8 heads of 128 x 128 in bfloat16 87 and 81, of 64 x 48 in float32 21 and 16, of 64 x 96 28 and 32; 64 rows of 64 x 64
// 6.1 and 5.5; 16 rows of 128 x 128 5.4 and 6.3, one 4.0 and 5.0.  (16 columns: 117 and 3.8, 128: 88 and 6.3, 416 rows and one.)
template <class T, int CB>
void launch_delta_step(const fm_delta_step_args& a, hipStream_t st) {
    const dim3 grid((unsigned)((a.v_dim + CB - 1) / CB), (unsigned)a.q_heads, (unsigned)a.n);
    if (a.v_dim % 4 || (((uintptr_t)a.state | (uintptr_t)a.next) & 15)) k_delta_step<T, CB, false><<<grid, 256, 0, st>>>(a);
    else k_delta_step<T, CB, true><<<grid, 256, 0, st>>>(a);
}
template <class T>
void delta_step_of_type(const fm_delta_step_args& a, hipStream_t st) {
    const long long blocks = (a.v_dim + 31) / 32;
    if (blocks % 2 == 0 && a.n * a.q_heads * blocks >= 1024) launch_delta_step<T, 64>(a, st);
    else launch_delta_step<T, 32>(a, st);
}

}  // namespace fg

using namespace fg;

extern "C" {

long long fm_delta_workspace(const fm_delta_args* a, int backward) {
    return a && !delta_wrong(*a, false, true) ? delta_workspace_bytes(*a, backward) : 0;
}
long long fm_delta_saved(const fm_delta_args* a) { return a && !delta_wrong(*a, false, true) ? delta_saved_bytes(*a) : 0; }
int fm_delta(const fm_delta_args* a, void* stream) { return delta(a, false, stream); }
int fm_delta_bwd(const fm_delta_args* a, void* stream) { return delta(a, true, stream); }

int fm_delta_step(const fm_delta_step_args* a, void* stream) {
    clear_error();
    if (!a) return fail("fm_delta_step: no arguments");
    if (const char* e = delta_heads_wrong(a->dtype, a->q_heads, a->k_heads, a->k_dim, a->v_dim))
        return fail((std::string("fm_delta_step: ") + e).c_str());
    if (a->n < 0 || a->n > 65535 || a->n_states < 0) return fail("fm_delta_step: other than 0 to 65535 rows");
    if (!a->n) return 0;
    if (!a->q.data || !a->k.data || !a->v.data || !a->log_decay || !a->beta || !a->state || !a->next || !a->o)
        return fail("fm_delta_step: a null tensor");
    if (!a->slots && a->n_states < a->n) return fail("fm_delta_step: fewer states than rows");
    if (a->next != a->state && share_memory(a->state, a->next, a->n_states * a->q_heads * a->k_dim * a->v_dim))
        return fail("fm_delta_step: next must be state or lie outside it");
    if (a->dtype == FM_F32) delta_step_of_type<float>(*a, (hipStream_t)stream);
    else if (a->dtype == FM_BF16) delta_step_of_type<bf16>(*a, (hipStream_t)stream);
    else delta_step_of_type<f16>(*a, (hipStream_t)stream);
    FG_CHECK(hipGetLastError(), -1);
    return 0;
}

}  // extern "C"
