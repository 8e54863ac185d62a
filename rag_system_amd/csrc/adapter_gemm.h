// adapter_gemm.h -- the matrix kernels of the query adapters (adapter.hip).
//
// Requests are met in the order of their slots (perm, slot_at: position -> request, slot), so that 16 neighbours mostly share an
// adapter.  Every product is written transposed, (weights' rows) x (requests): a request is ONE lane of every result
// (lane & 15), so slots are told apart per lane, and rows of x and of W, A, B are read along the summed index, 16 bytes a
// lane, straight into MFMA operands (16x16x4 float32, 16x16x32 bfloat16).
//     down:  U^T = c A_s X^T      (rank x requests)       float32, in sorted order, rank padded to Rp with zeros
//     up:    Y^T = W X^T + B_s U^T
// The backward is the same two with the transposed matrices: V = c B_s^T dY, dX = dY W + V A_s.
// U keeps float32: for bfloat16 weights its product is made of three, with the three bfloat16 that hold U's 24 bits (two would lose up
// to 2^-16 of it, which shows where y is small beside what W and the adapter add to it).
#pragma once
#include "distill_tile.h"

#include <type_traits>

namespace rag {
namespace adapter {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16;

__device__ __forceinline__ u16 f_to_bf(float f) { return __builtin_bit_cast(u16, (__bf16)f); }
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const u16* p) { return __uint_as_float((unsigned)*p << 16); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(u16* p, float v) { *p = f_to_bf(v); }

// The bank as a product sees it (forward: W, A, B; backward: their transposes).
struct Bank {
    const void *w, *a, *b;      // d_out x d_in, slots x rank x d_in, slots x d_out x rank
    const float* scale;         // slots
    int d_in, d_out, rank, rp;  // rp: row length of U
    int live;                   // of the rank: rows of A behind it are filled-up copies, whose U is zero whatever x and scale are
    bool vec_in, vec_rank;      // 16-byte loads along d_in (x, W, A) and along rank (B)
};
struct Order {
    const int* perm;            // NULL: position = request
    const int* slot_at;         // NULL: from slots
    const long long* slots;
    long long n;
    int n_slots;
    // position -> slot: >= 0, -1 (none), -2 (outside the bank: NaN)
    __device__ __forceinline__ int slot(long long pos) const {
        if (slot_at) return slot_at[pos];
        const long long s = slots[pos];
        return s >= -1 && s < n_slots ? (int)s : -2;
    }
    __device__ __forceinline__ long long request(long long pos) const { return perm ? perm[pos] : pos; }
};

template <typename T> struct Mma;
template <> struct Mma<float> {
    static constexpr int E = 4;
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
        return c;
    }
};
template <> struct Mma<u16> {
    static constexpr int E = 8;
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};

// Where the piece of a row of `end` values at `col` begins.  Rows of any length and alignment are read 16 bytes at a time too (the
// hardware takes any address): the piece that would pass the end is the row's LAST one, without the values before `col`.
template <int E>
__device__ __forceinline__ int begin_of(int col, int end) { return end < E ? col : min(col, end - E); }
// E values of `row` from there on (behind the end: the last one again).
template <bool VEC, typename T>
__device__ __forceinline__ u32x4 whole_piece(const T* row, int begin, int end) {
    constexpr int E = Mma<T>::E;
    if (VEC) return *reinterpret_cast<const u32x4*>(row + begin);
    u32x4 r;
    if (end >= E) {                     // (uniform)
        __builtin_memcpy(&r, row + begin, 16);
    } else {
        T v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = row[min(begin + e, end - 1)];
        __builtin_memcpy(&r, v, 16);
    }
    return r;
}
// That piece of `row`: what is in memory, and kept of it: zeros in the place of values before `col` and behind the end.  Two rows'
// pieces at the same place hold matching values, which is all that a sum over them needs.  VEC: rows are 16-byte aligned and end
// with a piece.  (Apart, since a loop that loads ahead may not touch the values until it uses them: it would wait for them.)
template <bool VEC, typename T>
__device__ __forceinline__ u32x4 raw_piece(const T* row, int col, int end) {
    constexpr int E = Mma<T>::E;
    return whole_piece<VEC>(row, VEC ? min(col, end - E) : begin_of<E>(col, end), end);
}
template <bool VEC, int E>
__device__ __forceinline__ u32x4 kept(u32x4 r, int col, int end) {
    if (VEC) {
        const unsigned keep = col < end ? ~0u : 0u;
        return u32x4{r[0] & keep, r[1] & keep, r[2] & keep, r[3] & keep};
    }
    const int begin = begin_of<E>(col, end), skip = col - begin, stop = end - begin;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (E == 8) r[e] &= (2 * e >= skip && 2 * e < stop ? 0xffffu : 0u) | (2 * e + 1 >= skip && 2 * e + 1 < stop ? 0xffff0000u : 0u);
        else r[e] &= e >= skip && e < stop ? ~0u : 0u;
    }
    return r;
}
template <bool VEC, typename T>
__device__ __forceinline__ u32x4 piece(const T* row, int col, int end) {
    return kept<VEC, Mma<T>::E>(raw_piece<VEC>(row, col, end), col, end);
}
// U's values that go with piece<VEC, T>(b, col, rank), E of them.  (Behind the rank U holds zeros.)
template <bool VEC, int E>
__device__ __forceinline__ void piece_of_u(const float* u, int col, int rank, float* v) {
    const int begin = VEC ? col : begin_of<E>(col, rank), skip = col - begin;
    __builtin_memcpy(v, VEC ? static_cast<const float*>(__builtin_assume_aligned(u + begin, 16)) : u + begin, E * 4);
    if (!VEC)
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = e >= skip ? v[e] : 0.f;
}

// Element e of a piece, as a float.
template <typename T>
__device__ __forceinline__ float element(u32x4 p, int e) {
    if (sizeof(T) == 4) return __uint_as_float(p[e & 3]);
    return __uint_as_float(e & 1 ? p[e >> 1] & 0xffff0000u : p[e >> 1] << 16);
}

// Up to two products of this kind in a launch (blockIdx.y): U, and V in a backward.
struct Down {
    Bank bank[2];
    const void* x[2];
    long long ldx[2];
    float* u[2];
};

// U (or V) of 32 positions: four waves take every fourth step along d_in, their sums meet in LDS.  (65536 x 768 bf16, rank 64: 60 us
// for 134 MB; each workgroup's chain of loads bounds it: 64 positions, which read A half as often, take as long.)
constexpr int DOWN_TOKENS = 32, DOWN_WAVES = 4;
template <typename T, int RT, bool VEC>
__global__ __launch_bounds__(64 * DOWN_WAVES) void down_kernel(Down d, Order ord) {
    const Bank& k = d.bank[blockIdx.y];
    const long long ldx = d.ldx[blockIdx.y];
    float* u = d.u[blockIdx.y];
    typedef Mma<T> M;
    constexpr int E = M::E;
    __shared__ float part[DOWN_WAVES][2 * RT][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, kl = lane >> 4;
    // neighbours, which share a slot's A, on ONE of the eight dies (65536 requests of 256 slots x 64 x 768 bf16: 300 -> 134 MB read)
    const long long p0 = ((long long)(blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3)) * DOWN_TOKENS;
    if (p0 >= ord.n) return;
    const T* x = static_cast<const T*>(d.x[blockIdx.y]);
    const T* row[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) row[t] = x + ord.request(min(p0 + t * 16 + li, ord.n - 1)) * ldx;
    const int mine = p0 + (lane & 31) < ord.n ? ord.slot(p0 + (lane & 31)) : -3;   // of position lane & 31
    unsigned todo = (unsigned)__ballot(mine >= 0);
    const int steps = (k.d_in + 4 * E - 1) / (4 * E);
    // positions without an adapter: zeros, outside the bank: NaN
    if (__ballot(mine == -1 || mine == -2))            // (rp is a multiple of 16: every lane goes round as often)
        for (int j = threadIdx.x; j < DOWN_TOKENS * k.rp; j += 64 * DOWN_WAVES) {
            const int s = __shfl(mine, j / k.rp);
            if (s == -1 || s == -2) u[(p0 + j / k.rp) * k.rp + j % k.rp] = s == -2 ? NAN : 0.f;
        }
    while (todo) {                    // (uniform over the workgroup: every wave has the same slots)
        const int s = __shfl(mine, __ffs(todo) - 1);
        const unsigned with = (unsigned)__ballot(mine == s) & todo;
        todo &= ~with;
        const T* a = static_cast<const T*>(k.a) + (long long)s * k.rank * k.d_in;
        f32x4 acc[2][RT];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < RT; ++r) acc[t][r] = f32x4{0.f, 0.f, 0.f, 0.f};
        u32x4 xp[2][2], ap[2][RT];
        auto load = [&](int st, u32x4* xt, u32x4* at) __attribute__((always_inline)) {
            const int col = (st * 4 + kl) * E;
#pragma unroll
            for (int t = 0; t < 2; ++t) xt[t] = raw_piece<VEC>(row[t], col, k.d_in);
#pragma unroll
            for (int r = 0; r < RT; ++r) at[r] = raw_piece<VEC>(a + (long long)min(r * 16 + li, k.rank - 1) * k.d_in, col, k.d_in);
            __builtin_amdgcn_sched_barrier(0);
        };
        auto use = [&](int st, u32x4* xt, u32x4* at) __attribute__((always_inline)) {
            if ((st + 1) * 4 * E > k.d_in) {         // (uniform; behind the end: zeros)
                const int col = (st * 4 + kl) * E;
#pragma unroll
                for (int t = 0; t < 2; ++t) xt[t] = kept<VEC, E>(xt[t], col, k.d_in);
#pragma unroll
                for (int r = 0; r < RT; ++r) at[r] = kept<VEC, E>(at[r], col, k.d_in);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < RT; ++r) acc[t][r] = M::mma(at[r], xt[t], acc[t][r]);
        };
        load(wave, xp[0], ap[0]);
        for (int st = wave; st < steps; st += 2 * DOWN_WAVES) {
            load(st + DOWN_WAVES, xp[1], ap[1]);
            use(st, xp[0], ap[0]);
            load(st + 2 * DOWN_WAVES, xp[0], ap[0]);
            use(st + DOWN_WAVES, xp[1], ap[1]);
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < RT; ++r) *reinterpret_cast<f32x4*>(&part[wave][t * RT + r][lane * 4]) = acc[t][r];
        __syncthreads();
        const float scale = k.scale[s];
        for (int j = wave; j < 2 * RT; j += DOWN_WAVES) {
            f32x4 sum = *reinterpret_cast<const f32x4*>(&part[0][j][lane * 4]);
#pragma unroll
            for (int w = 1; w < DOWN_WAVES; ++w) sum += *reinterpret_cast<const f32x4*>(&part[w][j][lane * 4]);
            const int t = j / RT, r0 = j % RT * 16 + 4 * kl;
            if ((with >> (t * 16 + li)) & 1) {
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = r0 + i < k.live ? sum[i] * scale : 0.f;
                if (r0 < k.rp) *reinterpret_cast<f32x4*>(u + (p0 + t * 16 + li) * k.rp + r0) = sum;
            }
        }
    }
}

// Four values of U from r0 on of one position (in lanes 0 to 3): one wave, 16 bytes a lane of x and of each of A's four rows.
template <typename T, bool VEC>
__device__ __forceinline__ float down_rows(const Bank& k, const T* x, int s, int r0) {
    constexpr int E = Mma<T>::E;
    const int lane = threadIdx.x & 63;
    const T* a = static_cast<const T*>(k.a) + (long long)s * k.rank * k.d_in;
    float acc[4] = {};
    for (int c = lane * E; c < k.d_in; c += 64 * E) {
        const u32x4 xp = piece<VEC>(x, c, k.d_in);
        u32x4 ap[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) ap[r] = piece<VEC>(a + (long long)min(r0 + r, k.rank - 1) * k.d_in, c, k.d_in);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float xe = element<T>(xp, e);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r] = fmaf(element<T>(ap[r], e), xe, acc[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        for (int o = 32; o > 0; o >>= 1) acc[r] += __shfl_xor(acc[r], o);
    const float v = lane == 0 ? acc[0] : lane == 1 ? acc[1] : lane == 2 ? acc[2] : acc[3];
    return r0 + lane < k.live ? v * k.scale[s] : 0.f;
}

// U where slots have few requests each: a workgroup per position, a wave per four rows of A_s.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void down_each_kernel(Down d, Order ord) {
    const Bank& k = d.bank[blockIdx.y];
    float* u = d.u[blockIdx.y];
    const long long p = blockIdx.x;
    const int s = ord.slot(p), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (s < 0) {
        for (int r = threadIdx.x; r < k.rp; r += 256) u[p * k.rp + r] = s == -2 ? NAN : 0.f;
        return;
    }
    const T* x = static_cast<const T*>(d.x[blockIdx.y]) + ord.request(p) * d.ldx[blockIdx.y];
    for (int r0 = wave * 4; r0 < k.rp; r0 += 16) {
        const float v = down_rows<T, VEC>(k, x, s, r0);
        if (lane < 4) u[p * k.rp + r0 + lane] = v;
    }
}

// += B_s U^T for a tile of 16 output columns (from o0) and the 16 positions from p: the first two slots by matrix products, slot
// by slot; where there are more, each lane takes its own position's.  share of shares: every shares-th step of the rank.
template <typename T, bool VEC>
__device__ __forceinline__ f32x4 up(const Bank& k, const float* u, long long p, long long n, int my_slot, int o0, f32x4 acc, int share = 0,
                                    int shares = 1) {
    typedef Mma<T> M;
    constexpr int E = M::E;
    const int lane = threadIdx.x & 63, li = lane & 15, kl = lane >> 4;
    unsigned todo = (unsigned)__ballot(my_slot >= 0) & 0xffffu;
    const float* ur = u + min(p + li, n - 1) * k.rp;
    for (int turn = 0; todo; ++turn) {
        if (turn == 2) {
            if ((todo >> li) & 1) {
                const T* b = static_cast<const T*>(k.b) + (long long)my_slot * k.d_out * k.rank;
                for (int r = share * E; r < k.rank; r += shares * E) {
                    float v[E];
                    piece_of_u<VEC, E>(ur, r, k.rank, v);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const u32x4 bv = piece<VEC>(b + (long long)min(o0 + 4 * kl + i, k.d_out - 1) * k.rank, r, k.rank);
#pragma unroll
                        for (int e = 0; e < E; ++e) acc[i] = fmaf(element<T>(bv, e), v[e], acc[i]);
                    }
                }
            }
            break;
        }
        const int s = __shfl(my_slot, __ffs(todo) - 1);
        const unsigned with = (unsigned)__ballot(my_slot == s) & todo;
        todo &= ~with;
        const T* b = static_cast<const T*>(k.b) + ((long long)s * k.d_out + min(o0 + li, k.d_out - 1)) * k.rank;
        // (others' lanes keep what they have: a zero times this slot's infinity would not be one)
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        for (int r = share * 4 * E; r < k.rank; r += shares * 4 * E) {
            const u32x4 bv = piece<VEC>(b, r + kl * E, k.rank);
            float v[E];
            piece_of_u<VEC, E>(ur, r + kl * E, k.rank, v);
            if constexpr (E == 4) {
                u32x4 uv;
                __builtin_memcpy(&uv, v, 16);
                sum = M::mma(bv, uv, sum);
            } else {
                u32x4 part[3];
                distill::three_parts<true>(v, part);
#pragma unroll
                for (int a = 2; a >= 0; --a) sum = M::mma(bv, part[a], sum);
            }
        }
        if ((with >> li) & 1) acc += sum;
    }
    return acc;
}

// A tile of Y^T to memory: lane = position, four columns.
template <typename T>
__device__ __forceinline__ void put(const Bank& k, void* y, long long ldy, long long request, int o, int slot, f32x4 v) {
    T* to = static_cast<T*>(y) + request * ldy + o;
    if (slot == -2) v = f32x4{NAN, NAN, NAN, NAN};
    if (o + 4 <= k.d_out) {             // (of any alignment)
        if constexpr (sizeof(T) == 4) {
            __builtin_memcpy(to, &v, 16);
        } else {
            typedef u16 u16x4 __attribute__((ext_vector_type(4)));
            typedef unsigned long long any64 __attribute__((aligned(2), may_alias));
            *reinterpret_cast<any64*>(to) = __builtin_bit_cast(unsigned long long, u16x4{f_to_bf(v[0]), f_to_bf(v[1]), f_to_bf(v[2]), f_to_bf(v[3])});
        }
        return;
    }
    for (int i = 0; i < 4; ++i)
        if (o + i < k.d_out) store1(to + i, v[i]);
}

// Y for a few requests: a workgroup has OT x 16 output columns and TT x 16 positions, its waves every WAVES-th step along d_in,
// straight from memory (each byte is used by one wave, LDS would only add a trip); their sums meet in LDS, a wave finishes a tile.
// WHOLE: U too, by each workgroup for itself, into `own` in LDS (at most 16 requests).
template <typename T, int OT, int TT, int WAVES, bool VEC, bool WHOLE = false>
__device__ __forceinline__ void up_direct(const Bank& k, const Order& ord, const void* xv, long long ldx, const float* u, void* y,
                                          long long ldy, int block, float* own = nullptr) {
    typedef Mma<T> M;
    constexpr int E = M::E;
    __shared__ float part[WAVES][OT * TT][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, kl = lane >> 4;
    const int outs = (k.d_out + 16 * OT - 1) / (16 * OT);        // (neighbours share their requests' rows)
    const long long p0 = (long long)(block / outs) * TT * 16;
    const int o0 = block % outs * OT * 16;
    const T* x = static_cast<const T*>(xv);
    const T* row[TT];
    const T* w[OT];
#pragma unroll
    for (int t = 0; t < TT; ++t) row[t] = x + ord.request(min(p0 + t * 16 + li, ord.n - 1)) * ldx;
#pragma unroll
    for (int o = 0; o < OT; ++o) w[o] = static_cast<const T*>(k.w) + (long long)min(o0 + o * 16 + li, k.d_out - 1) * k.d_in;
    f32x4 acc[OT][TT];
#pragma unroll
    for (int o = 0; o < OT; ++o)
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[o][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int steps = (k.d_in + 4 * E - 1) / (4 * E);
    u32x4 xp[2][TT], wp[2][OT];
    auto load = [&](int st, u32x4* xt, u32x4* wt) __attribute__((always_inline)) {
        const int col = (st * 4 + kl) * E;
#pragma unroll
        for (int t = 0; t < TT; ++t) xt[t] = raw_piece<VEC>(row[t], col, k.d_in);
#pragma unroll
        for (int o = 0; o < OT; ++o) wt[o] = raw_piece<VEC>(w[o], col, k.d_in);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto use = [&](int st, u32x4* xt, u32x4* wt) __attribute__((always_inline)) {
        if ((st + 1) * 4 * E > k.d_in) {             // (uniform; behind the end: zeros)
            const int col = (st * 4 + kl) * E;
#pragma unroll
            for (int t = 0; t < TT; ++t) xt[t] = kept<VEC, E>(xt[t], col, k.d_in);
#pragma unroll
            for (int o = 0; o < OT; ++o) wt[o] = kept<VEC, E>(wt[o], col, k.d_in);
        }
#pragma unroll
        for (int o = 0; o < OT; ++o)
#pragma unroll
            for (int t = 0; t < TT; ++t) acc[o][t] = M::mma(wt[o], xt[t], acc[o][t]);
    };
    load(wave, xp[0], wp[0]);
    for (int st = wave; st < steps; st += 2 * WAVES) {
        load(st + WAVES, xp[1], wp[1]);
        use(st, xp[0], wp[0]);
        load(st + 2 * WAVES, xp[0], wp[0]);
        use(st + WAVES, xp[1], wp[1]);
    }
#pragma unroll
    for (int o = 0; o < OT; ++o)
#pragma unroll
        for (int t = 0; t < TT; ++t) *reinterpret_cast<f32x4*>(&part[wave][o * TT + t][lane * 4]) = acc[o][t];
    if (WHOLE) {
        const int quads = k.rp / 4;
        for (int j = wave; j < (int)ord.n * quads; j += WAVES) {
            const int p = j / quads, s = ord.slot(p), r0 = j % quads * 4;
            const float v = s >= 0 && r0 < k.rank ? down_rows<T, VEC>(k, x + ord.request(p) * ldx, s, r0) : 0.f;
            if (lane < 4) own[p * k.rp + r0 + lane] = v;
        }
        u = own;
        __syncthreads();
    }
    // the adapters' side: the waves of a tile share the steps of the rank
    constexpr int TILES = OT * TT, SHARES = WAVES > TILES ? WAVES / TILES : 1;
    static_assert(WAVES % TILES == 0 || TILES % WAVES == 0, "waves of a tile");
    for (int j = wave % TILES; j < TILES; j += WAVES) {
        const long long p = p0 + j % TT * 16, pos = p + li;
        const int slot = pos < ord.n ? ord.slot(pos) : -3, o = o0 + j / TT * 16;
        f32x4* mine = reinterpret_cast<f32x4*>(&part[wave][j][lane * 4]);
        if (k.vec_rank) *mine = up<T, true>(k, u, p, ord.n, slot, o, *mine, wave / TILES, SHARES);
        else *mine = up<T, false>(k, u, p, ord.n, slot, o, *mine, wave / TILES, SHARES);
    }
    __syncthreads();
    for (int j = wave; j < TILES; j += WAVES) {
        f32x4 sum = *reinterpret_cast<const f32x4*>(&part[0][j][lane * 4]);
#pragma unroll
        for (int v = 1; v < WAVES; ++v) sum += *reinterpret_cast<const f32x4*>(&part[v][j][lane * 4]);
        const int o = o0 + j / TT * 16;
        const long long pos = p0 + j % TT * 16 + li;
        const int slot = pos < ord.n ? ord.slot(pos) : -3;
        if (pos < ord.n && o + 4 * kl < k.d_out) put<T>(k, y, ldy, ord.request(pos), o + 4 * kl, slot, sum);
    }
}

template <typename T, int OT, int TT, int WAVES, bool VEC>
__global__ __launch_bounds__(64 * WAVES) void up_direct_kernel(Bank k, Order ord, const void* xv, long long ldx, const float* u, void* y,
                                                               long long ldy, int first) {
    up_direct<T, OT, TT, WAVES, VEC>(k, ord, xv, ldx, u, y, ldy, first + (int)blockIdx.x);
}

// Both products of a few requests in one launch, while what every workgroup does again is little (768 wide, rank 16: 8 requests 15.5 us
// with two launches, 12.6 with one; 16 requests 15, 17.8).
constexpr long long WHOLE_PRODUCTS = 100000;
template <typename T, bool VEC>
__global__ __launch_bounds__(512) void whole_kernel(Bank k, Order ord, const void* xv, long long ldx, void* y, long long ldy) {
    __shared__ __align__(16) float own[16 * 128];
    up_direct<T, 1, 1, 8, VEC, true>(k, ord, xv, ldx, nullptr, y, ldy, blockIdx.x, own);
}

// Y for many requests: a workgroup has 128 output columns x POS positions (256, or 64 where that would leave CUs idle), each of its
// eight waves 64 x 64 (an operand read for every two products; 32 x 32: for every one), 128 bytes of every row a stage, three stages
// by LDS-DMA.  (Two waves on a SIMD, since an LDS-DMA instruction holds its wave for 60 to 180 cycles: four waves of 64 x 128 read
// less and took 30 us more.)  Rows of 16-byte pieces only.
// 65536 x 768 x 768 bf16, rank 64: 147 us = 526 TFLOP/s (the library's product alone, without adapters: 67), matrix pipes busy for
// 32 % of the time.  One workgroup fits on a CU, so what it does before its first and behind its last product, some 10 us of each 23, is not hidden by another's products.
// RS: 64-byte steps of the rank that a wave keeps of its slot's B rows while neighbours share the slot.
constexpr int TILED_OUTS = 128;
constexpr int tiled_lds_bytes(int pos) { return 3 * (TILED_OUTS + pos) * 128; }
template <typename T, int RS, int POS>
__global__ __launch_bounds__(512, 1) void up_tiled_kernel(Bank k, Order ord, const void* xv, long long ldx, unsigned x_bytes, const float* u, void* y,
                                                          long long ldy) {
    typedef Mma<T> M;
    constexpr int E = M::E, ESZ = sizeof(T), ROWS = TILED_OUTS + POS, STAGE = ROWS * 128, LOADS = ROWS / 8 / 8;
    constexpr int WP = POS / 64 >= 4 ? 4 : 2, WO = 8 / WP, TO = 8 / WO, TP = POS / 16 / WP;   // waves, and tiles of a wave
    extern __shared__ __align__(16) char tiled_lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, kl = lane >> 4;
    const int outs = (k.d_out + TILED_OUTS - 1) / TILED_OUTS;
    // the workgroups of the same positions follow each other on ONE of the eight dies, whose L2 then has their rows
    const unsigned turn = blockIdx.x >> 3;
    const long long p0 = (long long)((blockIdx.x & 7) + 8 * (turn / outs)) * POS;
    const int o0 = turn % outs * TILED_OUTS;
    if (p0 >= ord.n) return;
    const int stages = (k.d_in * ESZ + 127) / 128;
    const int lr = lane >> 3, lp = (lane & 7) ^ lr;
    // a wave's instructions: every eighth group of eight rows, W's first
    unsigned from[LOADS];
#pragma unroll
    for (int a = 0; a < LOADS; ++a) {
        const int row = (a * 8 + wave) * 8 + lr;
        from[a] = a * 64 < TILED_OUTS ? (unsigned)min(o0 + row, k.d_out - 1) * (unsigned)(k.d_in * ESZ)
                                      : (unsigned)(ord.request(min(p0 + row - TILED_OUTS, ord.n - 1)) * ldx * ESZ);
    }
    const unsigned w_bytes = (unsigned)k.d_out * k.d_in * ESZ;
    auto fetch1 = [&](int t, int b, int a) __attribute__((always_inline)) {
        const int col = min(t * 128 + lp * 16, k.d_in * ESZ - 16);       // (behind the end: masked)
        distill::lds_dma16(a * 64 < TILED_OUTS ? k.w : xv, a * 64 < TILED_OUTS ? w_bytes : x_bytes, from[a] + col,
                           tiled_lds + b * STAGE + (a * 8 + wave) * 1024);
    };
    f32x4 acc[TO][TP];
#pragma unroll
    for (int o = 0; o < TO; ++o)
#pragma unroll
        for (int t = 0; t < TP; ++t) acc[o][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int wo = wave % WO * TO * 16, wp = wave / WO * TP * 16, ob = o0 + wo;
    int off[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) off[h] = li * 128 + (((h * 4 + kl) ^ (li & 7)) << 4);
    auto stage = [&](int t, int b, int b2, bool tail) __attribute__((always_inline)) {
        const char* ws = tiled_lds + b * STAGE + wo * 128;
        const char* xs = tiled_lds + b * STAGE + (TILED_OUTS + wp) * 128;
        u32x4 a[2][TO], v[2][TP];
        auto read = [&](int h) __attribute__((always_inline)) {
#pragma unroll
            for (int o = 0; o < TO; ++o) a[h][o] = *reinterpret_cast<const u32x4*>(ws + o * 2048 + off[h]);
#pragma unroll
            for (int p = 0; p < TP; ++p) v[h][p] = *reinterpret_cast<const u32x4*>(xs + p * 2048 + off[h]);
            if (tail) {                     // (both: an infinity times zero is none)
                const unsigned keep = t * 128 + (h * 4 + kl) * 16 < k.d_in * ESZ ? ~0u : 0u;
#pragma unroll
                for (int o = 0; o < TO; ++o) a[h][o] = u32x4{a[h][o][0] & keep, a[h][o][1] & keep, a[h][o][2] & keep, a[h][o][3] & keep};
#pragma unroll
                for (int p = 0; p < TP; ++p) v[h][p] = u32x4{v[h][p][0] & keep, v[h][p][1] & keep, v[h][p][2] & keep, v[h][p][3] & keep};
            }
        };
        read(0);
        read(1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int o = 0; o < TO; ++o) {
#pragma unroll
                for (int p = 0; p < TP; ++p) acc[o][p] = M::mma(a[h][o], v[h][p], acc[o][p]);
#pragma unroll
                for (int f = (h * TO + o) * LOADS / (2 * TO); f < (h * TO + o + 1) * LOADS / (2 * TO); ++f) fetch1(t + 2 < stages ? t + 2 : 0, b2, f);
                __builtin_amdgcn_sched_barrier(0);
            }
    };
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int a = 0; a < LOADS; ++a) fetch1(b < stages ? b : 0, b, a);
    // what the adapters need of the wave's positions, on its way beside the products
    int slot0, request0, b_slot = -1;
    auto look = [&](int p, int* slot, int* request) __attribute__((always_inline)) {
        const long long pos = p0 + wp + p * 16 + li;
        *slot = pos < ord.n ? ord.slot(pos) : -3;
        *request = (int)ord.request(min(pos, ord.n - 1));
    };
    look(0, &slot0, &request0);
    u32x4 bv[TO][RS];
    f32x4 un[RS][E / 4];
    auto load_u = [&](int p, f32x4 (*to)[E / 4]) __attribute__((always_inline)) {
        const float* ur = u + min(p0 + wp + p * 16 + li, ord.n - 1) * k.rp;
#pragma unroll
        for (int r = 0; r < RS; ++r)
#pragma unroll
            for (int h = 0; h < E / 4; ++h) to[r][h] = *reinterpret_cast<const f32x4*>(ur + min((r * 4 + kl) * E + 4 * h, k.rp - 4));
    };
    auto load_b = [&](int s) __attribute__((always_inline)) {
        if (s == b_slot) return;                  // (uniform)
        const T* bs = static_cast<const T*>(k.b) + (long long)s * k.d_out * k.rank;
#pragma unroll
        for (int o = 0; o < TO; ++o)
#pragma unroll
            for (int r = 0; r < RS; ++r)
                bv[o][r] = piece<true>(bs + (long long)min(ob + o * 16 + li, k.d_out - 1) * k.rank, (r * 4 + kl) * E, k.rank);
        b_slot = s;
    };
    constexpr int PARTS = E == 8 ? 3 : 1;
    auto narrow = [&](const f32x4 (*from)[E / 4], u32x4 (*part)[PARTS]) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < RS; ++r) {
            if constexpr (E == 4) {
                part[r][0] = __builtin_bit_cast(u32x4, from[r][0]);
            } else {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = from[r][e >> 2][e & 3];
                distill::three_parts<true>(v, part[r]);
            }
        }
    };
    load_u(0, un);
    int b = 0;
    for (int t = 0; t + 1 < stages; ++t) {
        distill::wait_meet<LOADS>();
        stage(t, b, b > 0 ? b - 1 : 2, false);
        b = b < 2 ? b + 1 : 0;
    }
    distill::wait_meet<LOADS>();
    stage(stages - 1, b, b > 0 ? b - 1 : 2, true);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // no LDS-DMA outlives the workgroup
    // The tiles go through LDS (the ring is done with) into a loop over the positions: the adapters' cases are too much code to
    // stand here eight times.  A tile's U is loaded while the tile before it is finished, B's rows stay while the slot does.
    __syncthreads();
    char* tiles = tiled_lds + wave * TO * TP * 1024 + lane * 16;
#pragma unroll
    for (int p = 0; p < TP; ++p)
#pragma unroll
        for (int o = 0; o < TO; ++o) *reinterpret_cast<f32x4*>(tiles + (p * TO + o) * 1024) = acc[o][p];
    const bool kept_form = k.rank <= RS * 4 * E && k.vec_rank;      // (uniform)
    int next_slot = slot0, next_request = request0;
#pragma unroll 1
    for (int p = 0; p < TP; ++p) {
        const long long q = p0 + wp + p * 16;
        const int slot = next_slot, request = next_request;
        u32x4 part[RS][PARTS];
        narrow(un, part);
        if (p < TP - 1) {
            look(p + 1, &next_slot, &next_request);
            load_u(p + 1, un);
        }
        f32x4 v[TO];
#pragma unroll
        for (int o = 0; o < TO; ++o) v[o] = *reinterpret_cast<const f32x4*>(tiles + (p * TO + o) * 1024);
        unsigned todo = (unsigned)__ballot(slot >= 0) & 0xffffu;
        if (kept_form)
            for (int turn = 0; todo && turn < 2; ++turn) {
                const int s = __shfl(slot, __ffs(todo) - 1);
                const unsigned with = (unsigned)__ballot(slot == s) & todo;
                todo &= ~with;
                load_b(s);
#pragma unroll
                for (int o = 0; o < TO; ++o) {
                    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int r = 0; r < RS; ++r)
#pragma unroll
                        for (int a = PARTS - 1; a >= 0; --a) sum = M::mma(bv[o][r], part[r][a], sum);
                    if ((with >> li) & 1) v[o] += sum;          // (others' lanes keep what they have)
                }
            }
        if (todo) {                             // more slots in a tile, or rows of B in no whole pieces
            const int rest = (todo >> li) & 1 ? slot : -3;
#pragma unroll
            for (int o = 0; o < TO; ++o)
                v[o] = k.vec_rank ? up<T, true>(k, u, q, ord.n, rest, ob + o * 16, v[o]) : up<T, false>(k, u, q, ord.n, rest, ob + o * 16, v[o]);
        }
        if (slot > -3) {
#pragma unroll
            for (int o = 0; o < TO; ++o)
                if (ob + o * 16 + 4 * kl < k.d_out) put<T>(k, y, ldy, request, ob + o * 16 + 4 * kl, slot, v[o]);
        }
    }
}

}  // namespace adapter
}  // namespace rag
