// Linear attention with a decay for each head (include/flyguy_memory.h: fm_attention, fm_attention_bwd, fm_step).
//
// One scan computes everything: with x, y, v of K, K, N values a moment, a state Z [K][N] and l = exp(log_decay),
//   Z_i = l Z_{i-1} + cz y_i v_i^T,   out_i = co x_i Z_i.
// The forward is the scan of (q, k, v); the gradient of q that of (go, v, k), with the start state transposed; the
// gradients of k and v those of (v, go, q) and (k, q, go) over the moments backwards, from the end state's gradient, which
// the last moment's term does not decay; the second one's end state, decayed once more, is the start state's gradient.
#include <hip/hip_runtime.h>

#include "memory.h"

namespace fg {

constexpr int ATT_MAX = 128;             // values of a head

struct Scan {
    fm_view x, y, v;
    int xs, ys, vs;                      // query heads per head of x, y, v (1, or q_heads / k_heads)
    void* out;                           // dense [moments][heads][N]; 0: no output
    const float* init;                   // start state [n_seq][heads][K][N] (transposed: [N][K]); 0: zeros
    float* fin;                          // end state [n_seq][heads][K][N]; 0: not wanted
    int K, N, transposed, backwards;
    float co, cz;
};

struct Scans {
    Scan s[3];
    const float* log_decay;
    const void* starts;
    long long n_moments;
    int wide, heads;
};

// the moments of stretch n: [first, first + count) of the views
__device__ __forceinline__ void stretch_of(const Scans& a, int n, long long& first, long long& count) {
    if (!a.starts) {
        first = 0;
        count = a.n_moments;
        return;
    }
    long long b = index_at(a.starts, n, a.wide), e = index_at(a.starts, n + 1, a.wide);
    b = b < 0 ? 0 : b > a.n_moments ? a.n_moments : b;
    e = e < b ? b : e > a.n_moments ? a.n_moments : e;
    first = b;
    count = e - b;
}

// Moment by moment: a workgroup holds 32 columns of a head's state, 4 columns and every 32nd row a lane.
// grid (blocks of columns, heads, stretches x scans)
template <class T, class TO>
__global__ __launch_bounds__(256) void k_scan_simple(Scans a, int n_seq) {
    __shared__ float xs[ATT_MAX], ys[ATT_MAX], part[4][32];
    const Scan& s = a.s[blockIdx.z / n_seq];
    const int n = blockIdx.z % n_seq, h = blockIdx.y, tid = threadIdx.x, cg = tid & 7, rg = tid >> 3;
    const int c0 = blockIdx.x * 32 + 4 * cg, K = s.K, N = s.N;
    if (blockIdx.x * 32 >= N) return;
    long long first, count;
    stretch_of(a, n, first, count);
    const T* x = (const T*)s.x.data + (a.starts ? 0 : n * s.x.seq) + (h / s.xs) * s.x.head;
    const T* y = (const T*)s.y.data + (a.starts ? 0 : n * s.y.seq) + (h / s.ys) * s.y.head;
    const T* v = (const T*)s.v.data + (a.starts ? 0 : n * s.v.seq) + (h / s.vs) * s.v.head;
    TO* out = (TO*)s.out + ((a.starts ? first : n * a.n_moments) * a.heads + h) * N;
    const Keep keep(a.log_decay[h]);
    float z[4][4] = {};
    const size_t at = ((size_t)n * a.heads + h) * K * N;
    if (s.init)
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j) {
                const int k = rg + 32 * i, c = c0 + j;
                if (k < K && c < N) z[i][j] = s.init[at + (s.transposed ? (size_t)c * K + k : (size_t)k * N + c)];
            }
    for (long long i = 0; i < count; ++i) {
        const long long t = s.backwards ? count - 1 - i : i;
        __syncthreads();
        for (int k = tid; k < K; k += 256) {
            xs[k] = s.out ? widen(x[(first + t) * s.x.moment + k]) : 0.f;
            ys[k] = widen(y[(first + t) * s.y.moment + k]);
        }
        __syncthreads();
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float vv[4];
        for (int j = 0; j < 4; ++j) vv[j] = c0 + j < N ? s.cz * widen(v[(first + t) * s.v.moment + c0 + j]) : 0.f;
        const bool first_back = s.backwards && i == 0;
        for (int r = 0; r < 4; ++r) {
            const int k = rg + 32 * r;
            if (k >= K) break;
            for (int j = 0; j < 4; ++j) z[r][j] = (first_back ? z[r][j] : keep(z[r][j])) + ys[k] * vv[j];
            fma4(xs[k], make_float4(z[r][0], z[r][1], z[r][2], z[r][3]), o);
        }
        for (int m = 8; m < 64; m <<= 1) {
            o.x += __shfl_xor(o.x, m);
            o.y += __shfl_xor(o.y, m);
            o.z += __shfl_xor(o.z, m);
            o.w += __shfl_xor(o.w, m);
        }
        if ((tid & 63) < 8) *(float4*)&part[tid >> 6][4 * cg] = o;
        __syncthreads();
        if (s.out && tid < 32 && blockIdx.x * 32 + tid < N)
            out[t * a.heads * N + blockIdx.x * 32 + tid] =
                narrow<TO>(s.co * (part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid]));
    }
    if (a.starts && s.out) {             // moments of no stretch: those before the first one and after the last
        TO* all = (TO*)s.out + (size_t)h * N + blockIdx.x * 32 + (tid & 31);
        if (blockIdx.x * 32 + (tid & 31) < N) {
            if (n == 0)
                for (long long t = tid >> 5; t < first; t += 8) all[t * a.heads * N] = narrow<TO>(0.f);
            if (n == n_seq - 1)
                for (long long t = first + count + (tid >> 5); t < a.n_moments; t += 8) all[t * a.heads * N] = narrow<TO>(0.f);
        }
    }
    if (s.fin)
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j) {
                const int k = rg + 32 * i, c = c0 + j;
                if (k < K && c < N) s.fin[at + (size_t)k * N + c] = s.backwards && count ? keep(z[i][j]) : z[i][j];
            }
}

// gradients of shared heads: out[m][j][d] = the sum over a key head's `share` query heads of part[m][share j + i][d]
template <class T>
__global__ __launch_bounds__(256) void k_share(const float* __restrict__ part, T* __restrict__ out, int share, int D,
                                               long long n) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const long long row = i / D;
    const int d = (int)(i % D);
    float s = 0.f;
    for (int j = 0; j < share; ++j) s += part[(row * share + j) * D + d];
    out[i] = narrow<T>(s);
}

// One moment: a workgroup takes 32 columns of a row's state of one head.  grid (blocks of columns, heads, rows)
template <class T>
__global__ __launch_bounds__(256) void k_step(fm_step_args a) {
    __shared__ float part[4][32];
    const int tid = threadIdx.x, cg = tid & 7, rg = tid >> 3, h = blockIdx.y, K = (int)a.k_dim, N = (int)a.v_dim;
    const int c0 = blockIdx.x * 32 + 4 * cg;
    const long long n = blockIdx.z, slot = a.slots ? a.slots[n] : n;
    T* o = (T*)a.o + (n * a.q_heads + h) * N;
    if (slot < 0 || slot >= a.n_states) {
        if (tid < 32 && blockIdx.x * 32 + tid < N) o[blockIdx.x * 32 + tid] = narrow<T>(slot < 0 ? 0.f : NAN);
        return;
    }
    const int hk = h / (int)(a.q_heads / a.k_heads);
    const T* q = (const T*)a.q.data + n * a.q.seq + h * a.q.head;
    const T* k = (const T*)a.k.data + n * a.k.seq + hk * a.k.head;
    const T* v = (const T*)a.v.data + n * a.v.seq + hk * a.v.head;
    const size_t at = ((size_t)slot * a.q_heads + h) * K * N;
    const Keep keep(a.log_decay[h]);
    float acc[4] = {};
    for (int r = rg; r < K; r += 32)
        for (int j = 0; j < 4; ++j)
            if (c0 + j < N) {
                const float s = keep(a.state[at + (size_t)r * N + c0 + j]) + widen(k[r]) * widen(v[c0 + j]);
                a.next[at + (size_t)r * N + c0 + j] = s;
                acc[j] += widen(q[r]) * s;
            }
    for (int j = 0; j < 4; ++j) {
        for (int m = 8; m < 64; m <<= 1) acc[j] += __shfl_xor(acc[j], m);
        if ((tid & 63) < 8) part[tid >> 6][4 * cg + j] = acc[j];
    }
    __syncthreads();
    if (tid < 32 && blockIdx.x * 32 + tid < N)
        o[blockIdx.x * 32 + tid] = narrow<T>((float)a.scale * (part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid]));
}

// ------------------------------------------------------------------------------------------------ host
const char* heads_wrong(long long dtype, long long qh, long long kh, long long kd, long long vd) {
    if (dtype < FM_F32 || dtype > FM_F16) return "values of an unknown type";
    if (qh < 1 || kh < 1 || qh % kh || qh > 65535) return "query heads must be a multiple of key heads, at most 65535";
    if (kd < 1 || kd > ATT_MAX || vd < 1 || vd > ATT_MAX) return "heads of other than 1 to 128 values";
    return nullptr;
}

const char* attention_wrong(const fm_attention_args& a, bool bwd) {
    if (const char* e = heads_wrong(a.dtype, a.q_heads, a.k_heads, a.k_dim, a.v_dim)) return e;
    if (a.n_seq < 0 || a.n_seq > 16384) return "other than 0 to 16384 stretches";
    if (a.n_moments < 0 || a.n_moments > 1LL << 31) return "other than 0 to 2^31 moments";
    if (!a.log_decay) return "no decays";
    const bool any = a.n_seq && a.n_moments;
    if (any && (!a.q.data || !a.k.data || !a.v.data)) return "a null tensor";
    if (!bwd && any && !a.o) return "a null tensor";
    if (!bwd && a.state && a.state_out == a.state) return "state_out must not be state";
    if (bwd && any && !a.go.data) return "a null tensor";
    return nullptr;
}

// float32 partial gradients of shared key / value heads
long long shared_floats(const fm_attention_args& a, bool of_v) {
    const long long moments = a.n_moments * (a.starts ? 1 : a.n_seq);
    return a.q_heads > a.k_heads ? moments * a.q_heads * (of_v ? a.v_dim : a.k_dim) : 0;
}

template <class T, class TO>
void launch_scans(const Scans& a, int count, int n_seq, hipStream_t st) {
    if (!n_seq || !count) return;
    int widest = 0;
    for (int i = 0; i < count; ++i) widest = a.s[i].N > widest ? a.s[i].N : widest;
    k_scan_simple<T, TO><<<dim3((widest + 31) / 32, a.heads, n_seq * count), 256, 0, st>>>(a, n_seq);
}

template <class T>
void attention_fwd(const fm_attention_args& p, hipStream_t st) {
    const int share = (int)(p.q_heads / p.k_heads);
    Scans a{};
    a.log_decay = p.log_decay;
    a.starts = p.starts;
    a.n_moments = p.n_moments;
    a.wide = (int)p.wide;
    a.heads = (int)p.q_heads;
    a.s[0] = Scan{p.q, p.k, p.v, 1, share, share, p.o, p.state, p.state_out, (int)p.k_dim, (int)p.v_dim, 0, 0,
                  (float)p.scale, 1.f};
    launch_scans<T, T>(a, 1, (int)p.n_seq, st);
}

template <class T>
void attention_bwd(const fm_attention_args& p, hipStream_t st) {
    const int share = (int)(p.q_heads / p.k_heads), K = (int)p.k_dim, V = (int)p.v_dim;
    const float c = (float)p.scale;
    float* part_k = (float*)p.workspace;
    float* part_v = part_k + shared_floats(p, false);
    Scans a{};
    a.log_decay = p.log_decay;
    a.starts = p.starts;
    a.n_moments = p.n_moments;
    a.wide = (int)p.wide;
    a.heads = (int)p.q_heads;
    int n = 0;
    if (p.gq) a.s[n++] = Scan{p.go, p.v, p.k, 1, share, share, p.gq, p.state, nullptr, V, K, 1, 0, c, 1.f};
    const int own = share == 1;
    if (own && p.gk) a.s[n++] = Scan{p.v, p.go, p.q, share, 1, 1, p.gk, p.gstate_out, nullptr, V, K, 1, 1, 1.f, c};
    if (own && (p.gv || p.gstate)) a.s[n++] = Scan{p.k, p.q, p.go, share, 1, 1, p.gv, p.gstate_out, p.gstate, K, V, 0, 1, 1.f, c};
    launch_scans<T, T>(a, n, (int)p.n_seq, st);
    if (own) return;
    n = 0;
    if (p.gk) a.s[n++] = Scan{p.v, p.go, p.q, share, 1, 1, part_k, p.gstate_out, nullptr, V, K, 1, 1, 1.f, c};
    if (p.gv || p.gstate)
        a.s[n++] = Scan{p.k, p.q, p.go, share, 1, 1, p.gv ? part_v : nullptr, p.gstate_out, p.gstate, K, V, 0, 1, 1.f, c};
    launch_scans<T, float>(a, n, (int)p.n_seq, st);
    const long long rows = p.n_moments * (p.starts ? 1 : p.n_seq) * p.k_heads;
    if (rows && p.gk) k_share<T><<<(unsigned)((rows * K + 255) / 256), 256, 0, st>>>(part_k, (T*)p.gk, share, K, rows * K);
    if (rows && p.gv) k_share<T><<<(unsigned)((rows * V + 255) / 256), 256, 0, st>>>(part_v, (T*)p.gv, share, V, rows * V);
}

}  // namespace fg

using namespace fg;

extern "C" {

long long fm_attention_workspace(const fm_attention_args* a, int backward) {
    return backward ? 4 * (shared_floats(*a, false) + shared_floats(*a, true)) : 0;
}

int fm_attention(const fm_attention_args* a, void* stream) {
    clear_error();
    if (!a) return fail("fm_attention: no arguments");
    if (const char* e = attention_wrong(*a, false)) return fail((std::string("fm_attention: ") + e).c_str());
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
    if (const char* e = heads_wrong(a->dtype, a->q_heads, a->k_heads, a->k_dim, a->v_dim)) return fail((std::string("fm_step: ") + e).c_str());
    if (a->n < 0 || a->n > 65535 || a->n_states < 0) return fail("fm_step: other than 0 to 65535 rows");
    if (!a->n) return 0;
    if (!a->q.data || !a->k.data || !a->v.data || !a->log_decay || !a->state || !a->next || !a->o) return fail("fm_step: a null tensor");
    if (!a->slots && a->n_states < a->n) return fail("fm_step: fewer states than rows");
    const dim3 grid((unsigned)((a->v_dim + 31) / 32), (unsigned)a->q_heads, (unsigned)a->n);
    if (a->dtype == FM_F32) k_step<float><<<grid, 256, 0, (hipStream_t)stream>>>(*a);
    else if (a->dtype == FM_BF16) k_step<bf16><<<grid, 256, 0, (hipStream_t)stream>>>(*a);
    else k_step<f16><<<grid, 256, 0, (hipStream_t)stream>>>(*a);
    FG_CHECK(hipGetLastError(), -1);
    return 0;
}

}  // extern "C"
