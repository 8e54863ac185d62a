// distill.hip -- distillation of a ranker's top list over a flat index, forward and backward (rag_flat_distill_dev).
//
// Query q_i (d values), rows x_j of the index, beta = 1 / temperature.  Student logits
//     s_ij = beta <q_i, x_j>  (inner product)     or     -beta ||q_i - x_j||^2  (L2).
// Teacher: k row numbers t_ik (-1: no entry) with scores z_ik; p_i = softmax(z_i / teacher temperature) over the
// entries.  P_i = softmax(s_i) over every row of the index ("index") or over the entries of the list ("list").
//     loss_i = sum_k p_ik (log p_ik - s_i,t_ik) + log sum_j exp(s_ij)
//     dq_i   = w_i g beta (sum_j P_ij x_j - sum_k p_ik x_t_ik)          g = 1 (inner product), 2 (L2)
// (L2: the term in q_i has the factor sum_j P_ij - sum_k p_ik = 0.)  Gradient and loss need the same weights of the
// same rows, so both come out of ONE pass: a running maximum m, the sum l of exp(s - m) and the row sum
// o = sum_j exp(s_ij - m) x_j, rescaled when m grows.  The index is split over workgroups; a join kernel adds the parts.
// All sums, statistics and the row sum are fp32; dq is rounded once, to the type of q.
#include "common.h"
#include "distill_rows.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

namespace {

using namespace rag;

using distill::f32x4;
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));

constexpr int THREADS = 256;
constexpr int WAVES = THREADS / 64;

__device__ __forceinline__ float bf_to_f(unsigned short v) { return __uint_as_float((unsigned)v << 16); }
// round to nearest even; NaN stays NaN
__device__ __forceinline__ unsigned short f_to_bf(float f) {
    const unsigned u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (unsigned short)((u >> 16) | 0x40);
    return (unsigned short)((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
}
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const unsigned short* p) { return bf_to_f(*p); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(unsigned short* p, float v) { *p = f_to_bf(v); }

// A 16-byte piece of a row: E = 4 floats or 8 bfloat16.
template <typename T> struct Piece;
template <> struct Piece<float> {
    static constexpr int E = 4;
    static __device__ __forceinline__ void load(const float* p, float* v) {
        const f32x4 t = *reinterpret_cast<const f32x4*>(p);
        for (int i = 0; i < 4; ++i) v[i] = t[i];
    }
};
template <> struct Piece<unsigned short> {
    static constexpr int E = 8;
    static __device__ __forceinline__ void load(const unsigned short* p, float* v) {
        const u16x8 t = *reinterpret_cast<const u16x8*>(p);
        for (int i = 0; i < 8; ++i) v[i] = bf_to_f(t[i]);
    }
};

__device__ __forceinline__ float wave_sum(float v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
// over a workgroup of W waves, for every thread; `red` holds W floats
template <int W>
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
    for (int w = 0; w < W; ++w) s += red[w];
    return s;
}
template <int W>
__device__ __forceinline__ float block_max(float v, float* red) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = red[0];
    for (int w = 1; w < W; ++w) s = fmaxf(s, red[w]);
    return s;
}

struct Call {
    const void* x;            // rows, n x ld
    const float* norms;       // L2, over the index
    long long n, m;
    int ld, d, k, l2;
    const void* q;
    long long ldq;
    const long long* ids;     // m x k
    const float* scores;
    float beta, beta_t;
    const float* weights;     // m or NULL (1)
    float* loss;
    void* dq;                 // m x d or NULL
    long long lddq;
    // workspace of the "index" form: the parts of the index' shares
    float* part_ml;           // splits x m x 2: maximum in units of the product (L2: 2 <q,x> - ||x||^2), sum
    float* part_o;            // splits x m x ld
    int splits;
    long long rows_per_split;
};

// The teacher's side of one query, by each wave for itself (lists are short, a barrier costs more): the maximum and the sum
// of its softmax.  Returns 1, or 0 (no entry of finite score) or NaN (a row number outside the index).
__device__ __forceinline__ float teacher(const Call& c, const long long* ids, const float* z, float* zmax, float* zsum) {
    const int lane = threadIdx.x & 63;
    float top = -INFINITY;
    bool any = false, bad = false;
    for (int k = lane; k < c.k; k += 64) {
        const long long id = ids[k];
        const float v = z[k] * c.beta_t;
        bad |= id < -1 || id >= c.n;
        if (id >= 0) {
            top = fmaxf(top, v);
            any |= !(v == -INFINITY);
        }
    }
    if (__any(bad)) return NAN;
    if (!__any(any)) return 0.f;
    top = wave_max(top);
    float sum = 0.f;
    for (int k = lane; k < c.k; k += 64) sum += ids[k] >= 0 ? expf(z[k] * c.beta_t - top) : 0.f;
    *zmax = top;
    *zsum = wave_sum(sum);
    return 1.f;
}
// p and p (log p - s) of an entry
__device__ __forceinline__ float prob(const Call& c, float z, float zmax, float zsum) { return expf(z * c.beta_t - zmax) / zsum; }
__device__ __forceinline__ float cross(const Call& c, float z, float p, float s, float zmax, float log_zsum) {
    return p != 0.f ? p * (z * c.beta_t - zmax - log_zsum - s) : 0.f;   // (NaN enters)
}

// over = the list: one workgroup per query.  LPR lanes hold a row (NP pieces of 16 bytes each) and their columns of the query and of
// two sums, sum exp(s - m) x and sum p x: every row is read once, the next two are on their way while one is used.
// Bound by the gather of the rows: 4096 lists of 50 to 100 rows x 768 bfloat16 out of 300k, 470 MB in 114 us = 4.1 TB/s.
template <typename T, int LPR, int NP, bool GRAD>
__global__ __launch_bounds__(512) void list_rows_kernel(Call c) {
    typedef distill::RowPiece<T> P;
    typedef typename P::raw raw;
    constexpr int E = P::E, RPW = 64 / LPR;
    extern __shared__ __align__(16) char raw_lds[];
    long long* ids = reinterpret_cast<long long*>(raw_lds);         // k
    float* z = reinterpret_cast<float*>(ids + c.k);            // k
    float* p_of = z + c.k;                                     // k
    float* lds = p_of + c.k;                                   // GRAD: waves x ld
    __shared__ float mlh[8][3];
    const long long i = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6, li = lane % LPR;
    const int group = wave * RPW + lane / LPR, groups = waves * RPW;
    const T* x = static_cast<const T*>(c.x);
    const T* qp = static_cast<const T*>(c.q) + i * c.ldq;
    for (int k = tid; k < c.k; k += blockDim.x) {
        ids[k] = c.ids[i * c.k + k];
        z[k] = c.scores[i * c.k + k];
    }
    T* dq = GRAD ? static_cast<T*>(c.dq) + i * c.lddq : nullptr;
    int col[NP];
    bool mine[NP];
#pragma unroll
    for (int a = 0; a < NP; ++a) {
        col[a] = (li + LPR * a) * E;
        mine[a] = col[a] < c.ld;
        if (!mine[a]) col[a] = c.ld - E;
    }
    raw next[2][NP];
    auto fetch = [&](int k, raw* to) {        // (an entry that is none takes row 0, if there is one; it is not used)
        long long id = k < c.k ? ids[k] : 0;
        id = id >= 0 && id < c.n ? id : 0;
#pragma unroll
        for (int a = 0; a < NP; ++a) to[a] = *reinterpret_cast<const raw*>(x + id * c.ld + col[a]);
    };
    __syncthreads();
    if (c.n > 0) {
        fetch(group, next[0]);
        fetch(group + groups, next[1]);
    }
    float zmax, zsum;
    const float live = teacher(c, ids, z, &zmax, &zsum);
    if (!(live == 1.f)) {                     // (uniform) nothing to learn from, or a row number outside the index
        if (tid == 0) c.loss[i] = live;
        if (GRAD)
            for (int j = tid; j < c.d; j += blockDim.x) store1(dq + j, live);
        return;
    }
    const float log_zsum = logf(zsum);
    for (int k = tid; k < c.k; k += blockDim.x) p_of[k] = ids[k] >= 0 ? prob(c, z[k], zmax, zsum) : 0.f;
    float q[NP * E];
#pragma unroll
    for (int a = 0; a < NP; ++a)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float v = load1(qp + min(col[a] + e, c.d - 1));
            q[a * E + e] = mine[a] && col[a] + e < c.d ? v : 0.f;
        }
    __syncthreads();
    // m is a reference that moves when a logit lies more than 2^40 above it (weights up to there lose nothing)
    const float k2 = 1.44269504f;
    float m = -INFINITY, l = 0.f, head = 0.f, o[GRAD ? NP * E : 1] = {}, w[GRAD ? NP * E : 1] = {};
    for (int k = group; k - group < c.k; k += groups) {      // (every group goes round equally often)
        raw now[NP];
#pragma unroll
        for (int a = 0; a < NP; ++a) {
            now[a] = next[0][a];
            next[0][a] = next[1][a];
        }
        if (k - group + 2 * groups < c.k) fetch(k + 2 * groups, next[1]);
        const int at = k < c.k ? k : 0;
        const bool real = k < c.k && ids[at] >= 0;
        const float p = p_of[at];
        float v[NP * E], part[2] = {0.f, 0.f};
#pragma unroll
        for (int a = 0; a < NP; ++a) P::widen(now[a], v + a * E);
#pragma unroll
        for (int j = 0; j < NP * E; ++j) {
            if (c.l2) {
                const float t = mine[j / E] ? q[j] - v[j] : 0.f;     // (pad columns are zero on both sides)
                part[j & 1] = fmaf(t, t, part[j & 1]);
            } else {
                part[j & 1] = fmaf(q[j], v[j], part[j & 1]);
            }
        }
        const float dot = distill::group_sum<LPR>(part[0] + part[1]);
        const float s = real ? (c.l2 ? -c.beta * dot : c.beta * dot) : -INFINITY;
        if (real) head += cross(c, z[at], p, s, zmax, log_zsum);
        const bool lift = (s - m) * k2 > 40.f;
        if (__any(lift)) {
            const float scale = lift ? __builtin_amdgcn_exp2f((m - s) * k2) : 1.f;
            m = lift ? s : m;
            l *= scale;
            if (GRAD)
#pragma unroll
                for (int j = 0; j < NP * E; ++j) o[j] *= scale;
        }
        if (real) {
            const float e = __builtin_amdgcn_exp2f((s - (m == -INFINITY ? 0.f : m)) * k2);
            l += e;
            if (GRAD)
#pragma unroll
                for (int j = 0; j < NP * E; ++j) {
                    o[j] = fmaf(e, v[j], o[j]);
                    w[j] = fmaf(p, v[j], w[j]);
                }
        }
    }
    // the groups of a wave, then the waves
    float all = m;
#pragma unroll
    for (int d = LPR; d < 64; d *= 2) all = fmaxf(all, __shfl_xor(all, d));
    float mass = l * expf(m - (all == -INFINITY ? 0.f : all));
#pragma unroll
    for (int d = LPR; d < 64; d *= 2) {
        mass += __shfl_xor(mass, d);
        head += __shfl_xor(head, d);
    }
    if (lane == 0) {
        mlh[wave][0] = all;
        mlh[wave][1] = mass;
        mlh[wave][2] = head;
    }
    __syncthreads();
    float top = -INFINITY;
    for (int a = 0; a < waves; ++a) top = fmaxf(top, mlh[a][0]);
    const float base = top == -INFINITY ? 0.f : top;
    mass = head = 0.f;
    for (int a = 0; a < waves; ++a) {
        mass = fmaf(mlh[a][1], expf(mlh[a][0] - base), mass);
        head += mlh[a][2];
    }
    if (tid == 0) c.loss[i] = head + top + logf(mass);
    if (!GRAD) return;
    const float share = expf(m - base) / mass;
#pragma unroll
    for (int j = 0; j < NP * E; ++j) {
        o[GRAD ? j : 0] = fmaf(o[GRAD ? j : 0], share, -w[GRAD ? j : 0]);
#pragma unroll
        for (int d = LPR; d < 64; d *= 2) o[GRAD ? j : 0] += __shfl_xor(o[GRAD ? j : 0], d);
    }
    if (lane < LPR)
#pragma unroll
        for (int a = 0; a < NP; ++a)
            if (mine[a])
#pragma unroll
                for (int e = 0; e < E; ++e) lds[wave * c.ld + col[a] + e] = o[GRAD ? a * E + e : 0];
    __syncthreads();
    const float f = (c.weights ? c.weights[i] : 1.f) * c.beta * (c.l2 ? 2.f : 1.f);
    for (int j = tid; j < c.d; j += blockDim.x) {
        float sum = 0.f;
        for (int a = 0; a < waves; ++a) sum += lds[a * c.ld + j];
        store1(dq + j, f * sum);
    }
}

// s_of[k]: the student's logits of the list's entries, four entries a wave; qs holds the query.
template <typename T, int W>
__device__ __forceinline__ void list_logits(const Call& c, const long long* ids, const float* qs, float* s_of) {
    constexpr int E = Piece<T>::E;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15;
    for (int k = wave * 4 + (lane >> 4); k - (lane >> 4) < c.k; k += 4 * W) {
        const long long id = k < c.k ? ids[k] : -1;
        const T* row = static_cast<const T*>(c.x) + (id >= 0 ? id : 0) * c.ld;
        float acc = 0.f;
        if (id >= 0)
#pragma unroll 8
            for (int j = li * E; j < c.ld; j += 16 * E) {
                float v[E];
                Piece<T>::load(row + j, v);
                for (int e = 0; e < E; ++e) {
                    if (c.l2) {
                        const float t = qs[j + e] - v[e];
                        acc = fmaf(t, t, acc);
                    } else {
                        acc = fmaf(qs[j + e], v[e], acc);
                    }
                }
            }
        acc = distill::group_sum<16>(acc);
        if (li == 0 && k < c.k) s_of[k] = c.l2 ? -c.beta * acc : c.beta * acc;
    }
    __syncthreads();
}

// over = the list, any row length: one workgroup per query; the rows are read twice.
template <typename T>
__global__ __launch_bounds__(THREADS) void list_any_kernel(Call c) {
    constexpr int E = Piece<T>::E;
    extern __shared__ float sh[];
    float* qs = sh;               // ld
    float* s_of = qs + c.ld;      // k
    float* w_of = s_of + c.k;     // k
    __shared__ float red[WAVES];
    const long long i = blockIdx.x;
    const int tid = threadIdx.x;
    const T* x = static_cast<const T*>(c.x);
    const long long* ids = c.ids + i * c.k;
    const float* z = c.scores + i * c.k;
    const T* q = static_cast<const T*>(c.q) + i * c.ldq;
    T* dq = c.dq ? static_cast<T*>(c.dq) + i * c.lddq : nullptr;
    float zmax, zsum;
    const float live = teacher(c, ids, z, &zmax, &zsum);
    if (!(live == 1.f)) {         // (uniform)
        if (tid == 0) c.loss[i] = live;
        if (dq)
            for (int j = tid; j < c.d; j += THREADS) store1(dq + j, live);
        return;
    }
    for (int j = tid; j < c.ld; j += THREADS) qs[j] = j < c.d ? load1(q + j) : 0.f;
    __syncthreads();
    list_logits<T, WAVES>(c, ids, qs, s_of);
    float smax = -INFINITY, mass = 0.f, head = 0.f;
    for (int k = tid; k < c.k; k += THREADS)
        if (ids[k] >= 0) smax = fmaxf(smax, s_of[k]);
    smax = block_max<WAVES>(smax, red);
    for (int k = tid; k < c.k; k += THREADS)
        if (ids[k] >= 0) {
            mass += expf(s_of[k] - smax);
            head += cross(c, z[k], prob(c, z[k], zmax, zsum), s_of[k], zmax, logf(zsum));
        }
    mass = block_sum<WAVES>(mass, red);
    head = block_sum<WAVES>(head, red);
    if (tid == 0) c.loss[i] = head + smax + logf(mass);
    if (!dq) return;
    for (int k = tid; k < c.k; k += THREADS)
        w_of[k] = ids[k] >= 0 ? expf(s_of[k] - smax) / mass - prob(c, z[k], zmax, zsum) : 0.f;
    __syncthreads();
    const float f = (c.weights ? c.weights[i] : 1.f) * c.beta * (c.l2 ? 2.f : 1.f);
    for (int j = tid * E; j < c.ld; j += THREADS * E) {
        float acc[E] = {};
#pragma unroll 4
        for (int k = 0; k < c.k; ++k) {
            const long long id = ids[k];
            if (id < 0) continue;
            float v[E];
            Piece<T>::load(x + id * c.ld + j, v);
            for (int e = 0; e < E; ++e) acc[e] = fmaf(w_of[k], v[e], acc[e]);
        }
        for (int e = 0; e < E; ++e)
            if (j + e < c.d) store1(dq + j + e, f * acc[e]);
    }
}

// Any row length: one workgroup per (split of the rows, query), 32 rows at a time; a wave computes eight dot products,
// then every thread adds its columns of the 32 rows.  For rows that the other kernels' registers do not hold (over 1536 values):
// the rows are read twice, the second time from L2.  As in the matrix form, m is a reference that moves when a logit lies more than
// 2^LIFT above it, and the sums are put down then and every WINDOW steps: added to the share's part in HBM, and begun again.  (All
// rows of a large batch's one share in one float32 lost 2^-7 of the sum at 300000 rows.)  64 queries x 2048 bfloat16, 200k rows: 15.1 ms.
constexpr int ANY_ROWS = 32;
template <typename T, bool GRAD>
__global__ __launch_bounds__(THREADS) void index_any_kernel(Call c) {
    constexpr int E = Piece<T>::E, COLS = (8192 / E + THREADS - 1) / THREADS;
    extern __shared__ float qs[];   // ld
    __shared__ float s_of[ANY_ROWS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long long i = blockIdx.y, r0 = blockIdx.x * c.rows_per_split, r1 = min(c.n, r0 + c.rows_per_split);
    const T* x = static_cast<const T*>(c.x);
    const T* q = static_cast<const T*>(c.q) + i * c.ldq;
    for (int j = tid; j < c.ld; j += THREADS) qs[j] = j < c.d ? load1(q + j) : 0.f;
    __syncthreads();
    float m = -INFINITY, l = 0.f, o[COLS][E] = {};
    float m_part = 0.f, l_part = 0.f;      // of what is put down
    bool fresh = true;
    const long long at = blockIdx.x * c.m + i;
    auto put_down = [&]() {
        const float before = fresh ? 0.f : expf((m_part - (m == -INFINITY ? 0.f : m)) * c.beta);
        l_part = fmaf(l_part, before, l);
        l = 0.f;
        m_part = m;
        if (GRAD)
            for (int b = 0; b < COLS; ++b) {
                const int j = (b * THREADS + tid) * E;
                if (j >= c.ld) break;
                for (int e = 0; e < E; e += 4) {
                    f32x4* to = reinterpret_cast<f32x4*>(c.part_o + at * c.ld + j + e);
                    f32x4 v = {o[b][e], o[b][e + 1], o[b][e + 2], o[b][e + 3]};
                    if (!fresh) v += *to * before;
                    *to = v;
                    for (int k = 0; k < 4; ++k) o[b][e + k] = 0.f;
                }
            }
        fresh = false;
    };
    int step = 0;
    for (long long r = r0; r < r1; r += ANY_ROWS, ++step) {
        for (int a = wave; a < ANY_ROWS; a += WAVES) {
            float acc = 0.f;
            if (r + a < r1) {
                const T* row = x + (r + a) * c.ld;
                for (int j = lane * E; j < c.ld; j += 64 * E) {
                    float v[E];
                    Piece<T>::load(row + j, v);
                    for (int e = 0; e < E; ++e) acc = fmaf(qs[j + e], v[e], acc);
                }
                acc = wave_sum(acc);
                if (c.l2) acc = fmaf(2.f, acc, -c.norms[r + a]);
            } else {
                acc = -INFINITY;
            }
            if (lane == 0) s_of[a] = acc;
        }
        __syncthreads();
        float t = -INFINITY;
        for (int a = 0; a < ANY_ROWS; ++a) t = fmaxf(t, s_of[a]);
        const bool lift = (t - m) * c.beta > distill::LIFT * 0.69314718f;      // (uniform; m = -inf: nothing has been added)
        if ((lift && m != -INFINITY) || (step > 0 && step % distill::WINDOW == 0)) put_down();
        if (lift) m = t;
        const float base = m == -INFINITY ? 0.f : m;
        for (int a = 0; a < ANY_ROWS && r + a < r1; ++a) {
            const float p = expf((s_of[a] - base) * c.beta);
            l += p;
            if (!GRAD) continue;
            for (int b = 0; b < COLS; ++b) {
                const int j = (b * THREADS + tid) * E;
                if (j >= c.ld) break;
                float v[E];
                Piece<T>::load(x + (r + a) * c.ld + j, v);
                for (int e = 0; e < E; ++e) o[b][e] = fmaf(p, v[e], o[b][e]);
            }
        }
        __syncthreads();
    }
    put_down();
    if (tid == 0) {
        c.part_ml[2 * at] = m_part;
        c.part_ml[2 * at + 1] = l_part;
    }
}

// Adds the shares' parts and takes the teacher's side off: one workgroup per query and 64 columns, each wave adds every
// JOIN_WAVES-th share and list entry; one more workgroup per query computes the loss.  Latency-bound where there are few queries (512
// shares x 384, 1 query: 11 us with 16 waves of one column a lane), else by the parts' bytes (1024 queries, 32 shares: 95 us).
template <typename T, int JOIN_WAVES, int CPL>
__global__ __launch_bounds__(64 * JOIN_WAVES) void join_kernel(Call c) {
    constexpr int JOIN_THREADS = 64 * JOIN_WAVES;
    extern __shared__ float sh[];
    __shared__ float red[JOIN_WAVES];
    __shared__ float cols[JOIN_WAVES][64 * CPL][2];
    const long long i = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool loss = blockIdx.y == 0;
    const long long* ids = c.ids + i * c.k;
    const float* z = c.scores + i * c.k;
    const T* q = static_cast<const T*>(c.q) + i * c.ldq;
    T* dq = c.dq ? static_cast<T*>(c.dq) + i * c.lddq : nullptr;
    const int col = (((int)blockIdx.y - 1) * 64 + lane) * CPL;
    float zmax, zsum;
    const float live = teacher(c, ids, z, &zmax, &zsum);
    if (!(live == 1.f)) {             // (uniform)
        if (tid == 0 && loss) c.loss[i] = live;
        if (!loss && wave == 0)
            for (int e = 0; e < CPL; ++e)
                if (col + e < c.d) store1(dq + col + e, live);
        return;
    }
    // the shares' references and sums
    float m = -INFINITY, l = 0.f;
#pragma unroll 2
    for (int s = tid; s < c.splits; s += JOIN_THREADS) {
        const float ms = c.part_ml[2 * (s * c.m + i)], ls = c.part_ml[2 * (s * c.m + i) + 1], top = fmaxf(m, ms);
        if (top != -INFINITY) l = l * expf((m - top) * c.beta) + ls * expf((ms - top) * c.beta);
        else l += ls;                     // (nothing, or NaN)
        m = top;
    }
    const float mine = m;
    m = block_max<JOIN_WAVES>(m, red);
    l = block_sum<JOIN_WAVES>(mine == -INFINITY ? l : l * expf((mine - m) * c.beta), red);
    if (loss) {
        float* s_of = sh;                 // k
        float* qs = s_of + c.k;           // ld
        float qq = 0.f, head = 0.f;
        for (int j = tid; j < c.ld; j += JOIN_THREADS) {
            const float v = j < c.d ? load1(q + j) : 0.f;
            qs[j] = v;
            qq = fmaf(v, v, qq);
        }
        qq = block_sum<JOIN_WAVES>(qq, red);
        list_logits<T, JOIN_WAVES>(c, ids, qs, s_of);
        const float log_zsum = logf(zsum);
        for (int k = tid; k < c.k; k += JOIN_THREADS)
            if (ids[k] >= 0) head += cross(c, z[k], prob(c, z[k], zmax, zsum), s_of[k], zmax, log_zsum);
        head = block_sum<JOIN_WAVES>(head, red);
        if (tid == 0) c.loss[i] = head + c.beta * (c.l2 ? m - qq : m) + logf(l);
        return;
    }
    float o[CPL] = {}, a[CPL] = {};
    const int at = min(col, c.ld - CPL);     // (rows are padded to 16 bytes; columns behind the end are not stored)
#pragma unroll 8
    for (int s = wave; s < c.splits; s += JOIN_WAVES) {
        const float ms = c.part_ml[2 * (s * c.m + i)], f = ms == -INFINITY ? 0.f : expf((ms - m) * c.beta);
        float v[CPL];
        __builtin_memcpy(v, __builtin_assume_aligned(c.part_o + (s * c.m + i) * c.ld + at, CPL * 4), CPL * 4);
#pragma unroll
        for (int e = 0; e < CPL; ++e) o[e] = fmaf(f, v[e], o[e]);
    }
#pragma unroll 8
    for (int k = wave; k < c.k; k += JOIN_WAVES) {
        const long long id = ids[k];
        T v[CPL];
        __builtin_memcpy(v, __builtin_assume_aligned(static_cast<const T*>(c.x) + max(id, 0ll) * c.ld + at, CPL * sizeof(T)), CPL * sizeof(T));
        const float p = id >= 0 ? prob(c, z[k], zmax, zsum) : 0.f;
#pragma unroll
        for (int e = 0; e < CPL; ++e) a[e] = fmaf(p, id >= 0 ? load1(v + e) : 0.f, a[e]);
    }
#pragma unroll
    for (int e = 0; e < CPL; ++e) {
        cols[wave][lane * CPL + e][0] = o[e];
        cols[wave][lane * CPL + e][1] = a[e];
    }
    __syncthreads();
    const float f = (c.weights ? c.weights[i] : 1.f) * c.beta * (c.l2 ? 2.f : 1.f);
    for (int j = tid; j < 64 * CPL; j += JOIN_THREADS) {
        const int to = ((int)blockIdx.y - 1) * 64 * CPL + j;
        if (to >= c.d) break;
        float so = 0.f, sa = 0.f;
        for (int w = 0; w < JOIN_WAVES; ++w) {
            so += cols[w][j][0];
            sa += cols[w][j][1];
        }
        store1(dq + to, f * (so / l - sa));
    }
}

// How a call is split; depends on the number of queries and the row length, not on the number of rows (the
// workspace may be allocated before rows are added).
struct Plan {
    distill::TilePlan tile;
    int splits;
    size_t ml_off, o_off, bytes;
};

int elem_ld(int d, int bf16) { return bf16 ? (d + 7) & ~7 : (d + 3) & ~3; }

Plan make_plan(long long m, int d, int bf16, int over, bool grad) {
    Plan p{};
    if (over == RAG_OVER_LIST || m == 0) return p;
    const size_t ld = elem_ld(d, bf16);
    if (distill::tile_plan(m, (int)ld, bf16 != 0, grad, &p.tile)) p.splits = p.tile.splits;
    else p.splits = (int)std::max<long long>(1, std::min<long long>(1024, 2048 / m));
    auto take = [&](size_t floats) {
        const size_t at = p.bytes;
        p.bytes += (floats * sizeof(float) + 255) & ~(size_t)255;
        return at;
    };
    p.ml_off = take((size_t)p.splits * m * 2);
    p.o_off = take(grad ? (size_t)p.splits * m * ld : 0);
    return p;
}

struct Ctx {
    Call c;
    Plan p;
    int over;
    char* ws;
    hipStream_t st;
};

template <int V> using Int = std::integral_constant<int, V>;

template <typename T>
int launch(Ctx& x) {
    Call& c = x.c;
    if (x.over == RAG_OVER_LIST) {
        constexpr int E = Piece<T>::E;
        auto rows = [&](auto lpr, auto np) {
            if (lpr.value * np.value * E < c.ld) return false;
            // waves: enough for the list's rows, but fewer (two rows or more each) where the queries fill the card
            const int need = (c.k * lpr.value + 63) / 64, waves = std::max(1, std::min(c.m >= 1024 ? 4 : 8, need));
            const size_t bytes = (size_t)c.k * 16 + (c.dq ? (size_t)waves * c.ld * sizeof(float) : 0);
            if (c.dq) list_rows_kernel<T, lpr.value, np.value, true><<<(unsigned)c.m, 64 * waves, bytes, x.st>>>(c);
            else list_rows_kernel<T, lpr.value, np.value, false><<<(unsigned)c.m, 64 * waves, bytes, x.st>>>(c);
            return true;
        };
        bool served = rows(Int<16>(), Int<1>()) || rows(Int<16>(), Int<2>()) || rows(Int<32>(), Int<2>()) || rows(Int<32>(), Int<3>()) ||
                      rows(Int<32>(), Int<4>());
        if constexpr (E == 4) served = served || rows(Int<32>(), Int<6>()) || rows(Int<32>(), Int<8>());
        if (!served) list_any_kernel<T><<<(unsigned)c.m, THREADS, ((size_t)c.ld + 2 * c.k) * sizeof(float), x.st>>>(c);
        RAG_HIP(hipGetLastError());
        return RAG_OK;
    }
    const int step = x.p.tile.rows > 0 ? x.p.tile.rows : ANY_ROWS;     // shares are whole tiles; the last may be shorter
    const long long per = (c.n + x.p.splits - 1) / x.p.splits;
    c.rows_per_split = std::max<long long>(1, (per + step - 1) / step) * step;
    c.splits = (int)((c.n + c.rows_per_split - 1) / c.rows_per_split);
    c.part_ml = reinterpret_cast<float*>(x.ws + x.p.ml_off);
    c.part_o = reinterpret_cast<float*>(x.ws + x.p.o_off);
    if (c.splits > 0 && x.p.tile.rows > 0) {
        distill::TileCall t{};
        t.x = c.x;
        t.norms = c.l2 ? c.norms : nullptr;
        t.q = c.q;
        t.part_ml = c.part_ml;
        t.part_o = c.part_o;
        t.n = c.n;
        t.m = c.m;
        t.ldq = c.ldq;
        t.rows_per_split = c.rows_per_split;
        t.ld = c.ld;
        t.d = c.d;
        t.splits = c.splits;
        t.q_tiles = x.p.tile.q_tiles;
        t.k2 = (float)((double)c.beta * 1.4426950408889634074);
        const int rc = distill::tile_launch(x.p.tile, t, c.dq != nullptr, x.st);
        if (rc) return rc;
    } else if (c.splits > 0) {
        const dim3 grid((unsigned)c.splits, (unsigned)c.m);
        if (c.dq) index_any_kernel<T, true><<<grid, THREADS, c.ld * sizeof(float), x.st>>>(c);
        else index_any_kernel<T, false><<<grid, THREADS, c.ld * sizeof(float), x.st>>>(c);
        RAG_HIP(hipGetLastError());
    }
    // (few queries have many shares each, and leave the card to them; many share a workgroup's chain of loads over more columns)
    const size_t bytes = ((size_t)c.k + c.ld) * sizeof(float);
    auto grid = [&](int cols) { return dim3((unsigned)c.m, c.dq ? 1u + (unsigned)((c.d + cols - 1) / cols) : 1u); };
    if (c.m <= 64) join_kernel<T, 16, 1><<<grid(64), 64 * 16, bytes, x.st>>>(c);
    else join_kernel<T, 8, 4><<<grid(256), 64 * 8, bytes, x.st>>>(c);
    RAG_HIP(hipGetLastError());
    return RAG_OK;
}

int with_rows(const FlatRows& r, void* ctx) {
    Ctx& x = *static_cast<Ctx*>(ctx);
    x.c.x = r.arena;
    x.c.norms = r.norms;
    x.c.n = r.n_rows;
    x.c.ld = r.ld;
    x.c.d = r.d;
    x.c.l2 = r.metric == RAG_METRIC_L2;
    return r.bf16 ? launch<unsigned short>(x) : launch<float>(x);
}

int check_shape(const char* who, rag_flat_t* h, int64_t nq, int k, int over) {
    if (!h) return fail(RAG_ERR_INVALID_ARG, "%s: bad handle", who);
    if (nq < 0 || nq > RAG_DISTILL_MAX_NQ)
        return fail(RAG_ERR_INVALID_ARG, "%s: nq=%lld out of range [0,%d]", who, (long long)nq, RAG_DISTILL_MAX_NQ);
    if (k < 0 || k > RAG_DISTILL_MAX_K)
        return fail(RAG_ERR_INVALID_ARG, "%s: k=%d out of range [0,%d]", who, k, RAG_DISTILL_MAX_K);
    if (over != RAG_OVER_INDEX && over != RAG_OVER_LIST)
        return fail(RAG_ERR_INVALID_ARG, "%s: over=%d is neither RAG_OVER_INDEX(0) nor RAG_OVER_LIST(1)", who, over);
    return RAG_OK;
}

}  // namespace

extern "C" {

int rag_flat_distill_ws_bytes(rag_flat_t* h, int64_t nq, int k, int over, int want_grad, int64_t* bytes) {
    RAG_REQUIRE_INIT();
    const int rc = check_shape("rag_flat_distill_ws_bytes", h, nq, k, over);
    if (rc) return rc;
    if (!bytes) return fail(RAG_ERR_INVALID_ARG, "rag_flat_distill_ws_bytes: bytes is NULL");
    const FlatShape s = flat_shape(h);
    *bytes = (int64_t)make_plan(nq, s.d, s.bf16, over, want_grad != 0).bytes;
    return RAG_OK;
}

int rag_flat_distill_dev(rag_flat_t* h, int64_t nq, const void* q_dev, int64_t ldq, int k, const int64_t* ids_dev,
                         const float* scores_dev, double temperature, double teacher_temperature, int over,
                         const float* weights_dev, float* loss_dev, void* dq_dev, int64_t lddq, void* ws_dev,
                         int64_t ws_bytes, void* stream) {
    const char* who = "rag_flat_distill_dev";
    RAG_REQUIRE_INIT();
    int rc = check_shape(who, h, nq, k, over);
    if (rc) return rc;
    if (!(temperature > 0) || !(teacher_temperature > 0) || !std::isfinite(temperature) || !std::isfinite(teacher_temperature) ||
        !std::isfinite((float)(2.0 / temperature)) || !std::isfinite((float)(1.0 / teacher_temperature)))   // (2: the factors below)
        return fail(RAG_ERR_INVALID_ARG, "%s: temperatures must be positive and finite (%g, %g)", who, temperature,
                    teacher_temperature);
    if (nq == 0) return RAG_OK;
    const FlatShape s = flat_shape(h);
    if (!q_dev || !loss_dev || (k > 0 && (!ids_dev || !scores_dev)))
        return fail(RAG_ERR_INVALID_ARG, "%s: NULL buffer", who);
    if (ldq < s.d || (dq_dev && lddq < s.d))
        return fail(RAG_ERR_INVALID_ARG, "%s: row strides %lld / %lld are below d=%d", who, (long long)ldq, (long long)lddq, s.d);
    Ctx x{};
    x.p = make_plan(nq, s.d, s.bf16, over, dq_dev != nullptr);
    if (x.p.bytes > 0 && (!ws_dev || ws_bytes < (int64_t)x.p.bytes || ((uintptr_t)ws_dev & 255)))
        return fail(RAG_ERR_INVALID_ARG, "%s: needs a workspace of %lld bytes, aligned to 256 (rag_flat_distill_ws_bytes)", who,
                    (long long)x.p.bytes);
    x.over = over;
    x.ws = static_cast<char*>(ws_dev);
    x.st = (hipStream_t)stream;
    x.c.m = nq;
    x.c.k = k;
    x.c.q = q_dev;
    x.c.ldq = ldq;
    x.c.ids = reinterpret_cast<const long long*>(ids_dev);
    x.c.scores = scores_dev;
    x.c.beta = (float)(1.0 / temperature);
    x.c.beta_t = (float)(1.0 / teacher_temperature);
    x.c.weights = weights_dev;
    x.c.loss = loss_dev;
    x.c.dq = dq_dev;
    x.c.lddq = lddq;
    DeviceScope dev;
    return flat_rows_on_stream(h, s.metric == RAG_METRIC_L2 && over == RAG_OVER_INDEX, x.st, who, with_rows, &x);
}

}  // extern "C"
