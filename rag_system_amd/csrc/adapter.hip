// adapter.hip -- low-rank adapters of many requests beside a shared projection (rag_adapter_apply_dev / _grad_dev).
//
// Request t has an embedding x_t and a slot s = slots[t] (-1: no adapter) of a bank A (slots x R x d_in),
// B (slots x d_out x R), scale c (slots):
//     u_t = c_s A_s x_t                 y_t = W x_t + B_s u_t
// and, with dy the gradient of y (W is frozen),
//     v_t = c_s B_s^T dy_t              dx_t = W^T dy_t + A_s^T v_t
//     dA_s = sum_t v_t x_t^T            dB_s = sum_t dy_t u_t^T      over the requests of slot s.
// u, v, dA, dB and every sum are fp32; y and dx are rounded once, to the type of x.
#include "adapter_gemm.h"

#include <algorithm>

namespace {

using namespace rag;
using namespace rag::adapter;

// ---- order: requests sorted by slot, in the order they came within a slot ------------------------------------------
//
// A counting sort over bins 0 .. slots - 1, slots (none), slots + 1 (outside the bank).  A wave counts a chunk of requests,
// every bin's counts are summed over the chunks, and the wave puts its requests where the sums say: no atomics, so equal
// calls give equal orders.  For the gradients a slot's requests are dealt out as items of `len` (an empty slot is one item,
// which writes zeros).
struct Item {
    int slot, begin, end, part;   // part: -1, or the partial sum it writes (its slot has several items)
};
struct Sort {
    const long long* slots;
    int n, n_slots, bits, chunk, chunks, len;
    int *perm, *slot_at, *counts;           // counts: chunks x (slots + 2)
    int2* parts;                            // per slot: first partial, number of partials (0: none)
    int* n_items;
    Item* items;
};
__device__ __forceinline__ int bin_of(const Sort& s, int t) {
    const long long v = s.slots[t];
    return v >= 0 && v < s.n_slots ? (int)v : v == -1 ? s.n_slots : s.n_slots + 1;
}
// lane's place among the lanes of its bin, and their number: the lanes that agree in every bit of the bin
__device__ __forceinline__ int place_in_wave(int bits, int bin, bool live, int* of) {
    unsigned long long with = __ballot(live);
    for (int b = 0; b < bits; ++b) {
        const unsigned long long set = __ballot((bin >> b) & 1);
        with &= (bin >> b) & 1 ? set : ~set;
    }
    *of = __popcll(with);
    return __popcll(with & ((1ull << (threadIdx.x & 63)) - 1));
}
// What a lane has written is there for the others of its wave, and is not written before they have read what was.
__device__ __forceinline__ void wave_meets() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// f(request, bin, live) for 64 requests of the chunk at a time, eight lots of slots on their way at once.
template <typename F>
__device__ __forceinline__ void each_of_chunk(const Sort& s, int c, F f) {
    const int lane = threadIdx.x & 63, end = min(s.n, (c + 1) * s.chunk);
    for (int t0 = c * s.chunk; t0 < end; t0 += 512) {
        int bin[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) bin[j] = bin_of(s, min(t0 + j * 64 + lane, s.n - 1));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (t0 + j * 64 >= end) break;      // (uniform)
            f(t0 + j * 64 + lane, bin[j], t0 + j * 64 + lane < end);
            wave_meets();
        }
    }
}
// counts[] += this wave's chunk; the last lane of a bin adds for all of them (one writer, no atomics)
__device__ __forceinline__ void count_chunk(const Sort& s, int c, int* counts) {
    each_of_chunk(s, c, [&](int, int bin, bool live) {
        int of = 0;
        const int at = place_in_wave(s.bits, bin, live, &of);
        if (live && at == of - 1) counts[bin] += of;
    });
}
__device__ __forceinline__ void place_chunk(const Sort& s, int c, int* next) {
    each_of_chunk(s, c, [&](int t, int bin, bool live) {
        int of = 0;
        const int at = place_in_wave(s.bits, bin, live, &of);
        const int to = live ? next[bin] + at : 0;
        wave_meets();
        if (live && at == of - 1) next[bin] = to + 1;
        if (live) {
            s.perm[to] = t;
            s.slot_at[to] = bin < s.n_slots ? bin : bin == s.n_slots ? -1 : -2;
        }
    });
}
// From the bins' totals (in LDS) where each bin starts (there), and, if it shall write, the list of items.  A workgroup of 1024.
__device__ __forceinline__ void starts_and_items(const Sort& s, int* totals, int* tmp, bool write) {
    const int bins = s.n_slots + 2, per = (bins + 1023) / 1024, b0 = threadIdx.x * per;
    // three sums over the bins at a time: requests, items, partials
    int sum[3] = {0, 0, 0};
    auto items_of = [&](int b) { return b >= s.n_slots || !s.items ? 0 : max(1, (totals[b] + s.len - 1) / s.len); };
    for (int b = b0; b < min(bins, b0 + per); ++b) {
        const int it = items_of(b);
        sum[0] += totals[b];
        sum[1] += it;
        sum[2] += it > 1 ? it : 0;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int upto[3] = {sum[0], sum[1], sum[2]};         // within the wave, then over the waves
    for (int d = 1; d < 64; d *= 2)
        for (int a = 0; a < 3; ++a) {
            const int v = __shfl_up(upto[a], d);
            upto[a] += lane >= d ? v : 0;
        }
    if (lane == 63)
        for (int a = 0; a < 3; ++a) tmp[a * 16 + wave] = upto[a];
    __syncthreads();
    int all_items = 0;
    for (int w = 0; w < 16; ++w) {
        all_items += tmp[16 + w];
        if (w < wave)
            for (int a = 0; a < 3; ++a) upto[a] += tmp[a * 16 + w];
    }
    int at = upto[0] - sum[0], item = upto[1] - sum[1], part = upto[2] - sum[2];
    if (threadIdx.x == 0 && write && s.items) *s.n_items = all_items;
    for (int b = b0; b < min(bins, b0 + per); ++b) {
        const int total = totals[b], it = items_of(b);
        totals[b] = at;
        if (it > 0 && write) {
            s.parts[b] = int2{part, it > 1 ? it : 0};
            for (int j = 0; j < it; ++j)
                s.items[item + j] = Item{b, at + j * s.len, min(at + total, at + (j + 1) * s.len), it > 1 ? part + j : -1};
            item += it;
            part += it > 1 ? it : 0;
        }
        at += total;
    }
    __syncthreads();
}

// The place of every wave's first request of every bin, from the counts of all chunks: this workgroup's `waves` chunks from c0 on
// (next: waves x bins).  Every workgroup adds up the counts for itself, which is less than a launch to do it once.  tmp: 2048.
__device__ __forceinline__ void places(const Sort& s, int c0, int waves, int* next, int* totals, int* tmp) {
    const int bins = s.n_slots + 2;
    // several threads a bin where there are few, each for a run of the chunks
    const int width = min(1024, (bins + 63) / 64 * 64), teams = 1024 / width;
    const int team = threadIdx.x / width, run = (s.chunks + teams - 1) / teams, from = team * run, to = team < teams ? min(s.chunks, from + run) : 0;
    for (int b0 = 0; b0 < bins; b0 += width) {
        const int b = b0 + threadIdx.x % width;
        int all = 0, before = 0;
        if (b < bins)
            for (int c = from; c < to; c += 16) {           // (sixteen on their way at once)
                int v[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = s.counts[min(c + j, to - 1) * bins + b];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    all += c + j < to ? v[j] : 0;
                    before += c + j < min(to, c0) ? v[j] : 0;
                }
            }
        tmp[threadIdx.x] = all;
        tmp[1024 + threadIdx.x] = before;
        __syncthreads();
        if (b < bins && team == 0) {
            for (int t = 1; t < teams; ++t) {
                all += tmp[t * width + threadIdx.x];
                before += tmp[1024 + t * width + threadIdx.x];
            }
            totals[b] = all;
            for (int w0 = 0; w0 < waves; w0 += 4) {
                int v[4];
#pragma unroll
                for (int w = 0; w < 4; ++w) v[w] = s.counts[min(c0 + w0 + w, s.chunks - 1) * bins + b];
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    next[(w0 + w) * bins + b] = before;
                    before += v[w];               // (behind the last chunk: not used)
                }
            }
        }
        __syncthreads();
    }
    starts_and_items(s, totals, tmp, blockIdx.x == 0);
    for (int j = threadIdx.x; j < waves * bins; j += 1024) next[j] += totals[j % bins];
    __syncthreads();
}
__global__ __launch_bounds__(1024) void place_kernel(Sort s, int waves) {
    extern __shared__ int lds[];
    const int bins = s.n_slots + 2, wave = threadIdx.x >> 6, c0 = blockIdx.x * waves;
    int* totals = lds + waves * bins;
    places(s, c0, waves, lds, totals, totals + bins);
    if (wave < waves && c0 + wave < s.chunks) place_chunk(s, c0 + wave, lds + wave * bins);
}

// ---- transposes of the bank for the backward ---------------------------------------------------------------------------
struct Turn {
    const void* from[3];
    void* to[3];
    int rows[3], cols[3], count[3];   // count matrices of rows x cols, dense
    int to_rows[3], to_cols[3];       // of the transposes: cols and rows, or more, filled up with zeros
    int first[4];                     // first workgroup of each kind
};
// One 64 x 64 tile by WAVES waves.
template <typename T, int WAVES>
__device__ __forceinline__ void turn_tile(const Turn& j, int block, T (*tile)[66]) {
    int kind = 0;
    while (kind < 2 && block >= j.first[kind + 1]) ++kind;
    const int rows = j.rows[kind], cols = j.cols[kind], to_rows = j.to_rows[kind], to_cols = j.to_cols[kind];
    const int tr = (to_cols + 63) / 64, tc = (to_rows + 63) / 64;
    const int b = block - j.first[kind], m = b / (tr * tc), r0 = b / tc % tr * 64, c0 = b % tc * 64;
    const T* from = static_cast<const T*>(j.from[kind]) + (long long)m * rows * cols;
    T* to = static_cast<T*>(j.to[kind]) + (long long)m * to_rows * to_cols;
    const int lane = threadIdx.x & 63;
    for (int r = threadIdx.x >> 6; r < 64; r += WAVES)
        tile[r][lane] = r0 + r < rows && c0 + lane < cols ? from[(long long)(r0 + r) * cols + c0 + lane] : (T)0;
    __syncthreads();
    for (int c = threadIdx.x >> 6; c < 64; c += WAVES)
        if (c0 + c < to_rows && r0 + lane < to_cols) to[(long long)(c0 + c) * to_cols + r0 + lane] = tile[lane][c];
}

// ---- rows in whole pieces ------------------------------------------------------------------------------------------------
//
// The tiled product wants rows that begin and end with a 16-byte piece.  For a batch that it serves, matrices whose rows do not are
// copied, filled up with zeros (16001 x 767 x 765 bf16, 64 slots of rank 33: 398 us without the copies, 106 with them).
struct Pad {
    const void* from[4];
    void* to[4];
    long long ld[4];                            // between rows of `from`, whose matrices follow each other
    int rows[4], cols[4], to_rows[4], to_cols[4];
    unsigned first[5];                          // first piece of each kind
};
template <typename T>
__global__ __launch_bounds__(256) void pad_kernel(Pad j) {
    constexpr int E = Mma<T>::E;
    for (unsigned at = blockIdx.x * 256 + threadIdx.x; at < j.first[4]; at += gridDim.x * 256) {
        int kind = 0;
        while (kind < 3 && at >= j.first[kind + 1]) ++kind;
        const unsigned i = at - j.first[kind], pieces = j.to_cols[kind] / E, row = i / pieces, m = row / j.to_rows[kind], r = row % j.to_rows[kind];
        const int cols = j.cols[kind], col = (int)(i % pieces) * E;
        u32x4 v = {0, 0, 0, 0};
        if (r < (unsigned)j.rows[kind]) {
            const T* from = static_cast<const T*>(j.from[kind]) + ((long long)m * j.rows[kind] + r) * j.ld[kind];
            if (col + E <= cols) {
                __builtin_memcpy(&v, from + col, 16);
            } else {
                T e[E] = {};
                for (int k = 0; k < E; ++k)
                    if (col + k < cols) e[k] = from[col + k];
                __builtin_memcpy(&v, e, 16);
            }
        }
        *reinterpret_cast<u32x4*>(static_cast<T*>(j.to[kind]) + (long long)i * E) = v;
    }
}

// All of it in one workgroup: sixteen waves, sixteen chunks, counts in LDS.
constexpr int SMALL_BINS = 1026, SMALL_N = 4096;
__device__ __forceinline__ void order_small(const Sort& s, int* lds) {
    const int bins = s.n_slots + 2, wave = threadIdx.x >> 6;
    int* counts = lds;                 // 16 x bins
    int* totals = counts + 16 * bins;  // bins
    int* tmp = totals + bins;          // 48
    for (int j = threadIdx.x; j < 16 * bins; j += 1024) counts[j] = 0;
    __syncthreads();
    count_chunk(s, wave, counts + wave * bins);
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += 1024) {
        int sum = 0;
        for (int w = 0; w < 16; ++w) {
            const int v = counts[w * bins + b];
            counts[w * bins + b] = sum;
            sum += v;
        }
        totals[b] = sum;
    }
    __syncthreads();
    starts_and_items(s, totals, tmp, true);
    for (int j = threadIdx.x; j < 16 * bins; j += 1024) counts[j] += totals[j % bins];
    __syncthreads();
    place_chunk(s, wave, counts + wave * bins);
}
// The first workgroup sorts, the others turn the bank's matrices (none for a forward): a launch fewer.
template <typename T>
__global__ __launch_bounds__(1024) void prepare_kernel(Sort s, Turn j) {
    extern __shared__ __align__(16) int prepare_lds[];
    if (blockIdx.x == 0) order_small(s, prepare_lds);
    else turn_tile<T, 16>(j, blockIdx.x - 1, reinterpret_cast<T(*)[66]>(prepare_lds));
}
// More requests: chunks counted by a wave each, beside the turning; place_kernel follows (16001 requests of 64 slots:
// one workgroup 30 us, the two launches 22).
template <typename T>
__global__ __launch_bounds__(256) void count_kernel(Sort s, Turn j, unsigned groups) {
    extern __shared__ __align__(16) int count_lds[];
    if (blockIdx.x >= groups) {
        turn_tile<T, 4>(j, blockIdx.x - groups, reinterpret_cast<T(*)[66]>(count_lds));
        return;
    }
    const int bins = s.n_slots + 2, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 4 + wave;
    int* counts = count_lds + wave * bins;
    for (int b = lane; b < bins; b += 64) counts[b] = 0;
    __syncthreads();
    if (c < s.chunks) count_chunk(s, c, counts);
    __syncthreads();
    if (c < s.chunks)
        for (int b = lane; b < bins; b += 64) s.counts[(long long)c * bins + b] = counts[b];
}

// ---- gradients of the bank -----------------------------------------------------------------------------------------------
//
// dA_s = sum_t v_t x_t^T and dB_s = sum_t dy_t u_t^T over the requests of an item.  MFMA 16x16x4 in float32 (u and v are float32,
// and the sums are small beside W's products): the A operand is u or v (16 of the rank x 4 requests), the B operand x or dy.
// A lane loads 16 bytes of a request's row, E columns, and gives one of them to each of E products: product e has the columns
// li * E + e (the last lane's: the row's last E columns).  Nothing is staged; a wave has 16 E columns and up to 64 of the rank.
struct SlotGrad {
    Sort s;
    const float *u, *v;
    const void *x, *dy;
    long long ldx, lddy;
    float *da, *db, *part;   // part: partials x rank x (d_in + d_out)
    int d_in, d_out, rank, rp;
    int row_x, row_dy;       // values in a row of x and dy: d_in and d_out, or with zeros up to a whole piece
    bool vec_x, vec_dy;
};
// Four waves share an item and a unit, 64 requests at a time each; their sums meet in LDS.  (They take the same branches:
// every wave of the workgroup comes to the barriers.)
template <typename T, int RT>
__device__ __forceinline__ void slot_grad(const SlotGrad& g, int item, int unit, float (*part)[4][256]) {
    constexpr int E = Mma<T>::E, LOT = RT >= 4 ? 4 : 8;       // steps whose operands are on their way at once
    const int lane = threadIdx.x & 63, li = lane & 15, kl = lane >> 4, team = threadIdx.x >> 6 & 3;
    const int rcs = (g.rank + RT * 16 - 1) / (RT * 16);
    const int cols_a = (g.d_in + 16 * E - 1) / (16 * E), cols_b = (g.d_out + 16 * E - 1) / (16 * E);
    const bool live = item < *g.s.n_items && unit < (cols_a + cols_b) * rcs;
    const Item it = live ? g.s.items[item] : Item{0, 0, 0, -1};
    const bool is_b = unit >= cols_a * rcs;
    if (is_b) unit -= cols_a * rcs;
    const int r0 = unit % rcs * RT * 16, c0 = unit / rcs * 16 * E + li * E, d = is_b ? g.d_out : g.d_in;
    const int row_d = is_b ? g.row_dy : g.row_x, begin = begin_of<E>(c0, row_d);
    const T* src = static_cast<const T*>(is_b ? g.dy : g.x);
    const long long ld = is_b ? g.lddy : g.ldx;
    const float* cf = (is_b ? g.u : g.v) + r0;
    const bool vec = is_b ? g.vec_dy : g.vec_x;
    f32x4 acc[RT][E];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[r][e] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int t0 = it.begin + team * 64; t0 < it.end; t0 += 256) {
        const int mine = g.s.perm[min(t0 + lane, it.end - 1)];
        const int steps = (min(64, it.end - t0) + 3) / 4;
        for (int s0 = 0; s0 < steps; s0 += LOT) {
            u32x4 xv[LOT];
            float a[LOT][RT];
#pragma unroll
            for (int j = 0; j < LOT; ++j) {
                const int t = t0 + (s0 + j) * 4 + kl;
                const T* row = src + (long long)__shfl(mine, min((s0 + j) * 4 + kl, 63)) * ld;
                xv[j] = vec ? whole_piece<true>(row, begin, row_d) : whole_piece<false>(row, begin, row_d);
#pragma unroll
                for (int r = 0; r < RT; ++r) a[j][r] = cf[(long long)min(t, it.end - 1) * g.rp + min(r * 16 + li, g.rp - 1 - r0)];
            }
#pragma unroll
            for (int j = 0; j < LOT; ++j) {
                const unsigned keep = t0 + (s0 + j) * 4 + kl < it.end ? ~0u : 0u;
#pragma unroll
                for (int e = 0; e < 4; ++e) xv[j][e] &= keep;
#pragma unroll
                for (int r = 0; r < RT; ++r) a[j][r] = __uint_as_float(__float_as_uint(a[j][r]) & keep);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float b = element<T>(xv[j], e);
#pragma unroll
                    for (int r = 0; r < RT; ++r) acc[r][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j][r], b, acc[r][e], 0, 0, 0);
                }
            }
        }
    }
    const long long size_a = (long long)g.rank * g.d_in, size_b = (long long)g.rank * g.d_out;
    float* to = it.part >= 0 ? g.part + it.part * (size_a + size_b) + (is_b ? size_a : 0)
                             : is_b ? g.db + it.slot * size_b : g.da + it.slot * size_a;
    // four tiles at a time: each wave adds up one of them
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e0 = 0; e0 < E; e0 += 4) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 4; ++e) *reinterpret_cast<f32x4*>(&part[team][e][lane * 4]) = acc[r][e0 + e];
            __syncthreads();
            f32x4 sum = *reinterpret_cast<const f32x4*>(&part[0][team][lane * 4]);
#pragma unroll
            for (int w = 1; w < 4; ++w) sum += *reinterpret_cast<const f32x4*>(&part[w][team][lane * 4]);
            const int rr = r0 + r * 16 + 4 * kl, cc = begin + e0 + team;
            if (live && cc >= c0 && cc < d)       // (columns before c0 are another lane's)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (rr + i < g.rank) to[is_b ? (long long)cc * g.rank + rr + i : (long long)(rr + i) * g.d_in + cc] = sum[i];
        }
}
template <typename T, int RT>
__global__ __launch_bounds__(256) void slot_grad_kernel(SlotGrad g) {
    __shared__ float part[4][4][256];
    slot_grad<T, RT>(g, blockIdx.x, blockIdx.y, part);
}
// dx of a few requests and the bank's gradients, which do not depend on each other: a launch fewer, and neither waits for the
// other's last workgroups.
template <typename T, int RT, bool VEC>
__global__ __launch_bounds__(512) void up_and_slot_kernel(Bank k, Order ord, const void* xv, long long ldx, const float* u, void* y, long long ldy,
                                                          unsigned up_first, unsigned slot_first, unsigned slot_groups, SlotGrad g, unsigned unit_groups) {
    __shared__ float part[2][4][4][256];
    const unsigned b = blockIdx.x - slot_first, half = threadIdx.x >> 8;
    if (b >= slot_groups) {              // (also below slot_first: unsigned)
        up_direct<T, 1, 2, 8, VEC>(k, ord, xv, ldx, u, y, ldy, blockIdx.x - up_first);
        return;
    }
    slot_grad<T, RT>(g, b / unit_groups, b % unit_groups * 2 + half, part[half]);
}
// The slots of several items: their partials, in order.
__global__ __launch_bounds__(256) void slot_join_kernel(SlotGrad g) {
    const int2 parts = g.s.parts[blockIdx.x];
    if (parts.y == 0) return;
    const long long size_a = (long long)g.rank * g.d_in, size = size_a + (long long)g.rank * g.d_out;
    for (long long j = (long long)blockIdx.y * 256 + threadIdx.x; j < size; j += (long long)gridDim.y * 256) {
        float sum = 0.f;
#pragma unroll 8
        for (int p = 0; p < parts.y; ++p) sum += g.part[(parts.x + p) * size + j];
        if (j < size_a) g.da[blockIdx.x * size_a + j] = sum;
        else g.db[blockIdx.x * (size - size_a) + j - size_a] = sum;
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
struct Plan {
    bool sorted, each;
    bool pad;                // rows filled up to whole pieces
    int rp, chunk, chunks, len, max_items, max_parts;
    int in, out, rank;       // row lengths then: d_in, d_out, rank otherwise
    size_t xp, wp, ap, bp, dyp, u, v, perm, slot_at, counts, parts, n_items, items, wt, at, bt, part, bytes;
};

constexpr long long MAX_THREADS = 1ll << 31;      // of a launch (the runtime refuses 2^32)

// Positions of a workgroup of the tiled product, or 0: too few of them to fill the card, the direct one takes it.
int tiled_positions(long long n, long long ldx, int d_out, size_t esz) {
    if ((unsigned long long)n * ldx * esz >= (1ull << 32)) return 0;      // (rows are found by 32-bit offsets)
    const long long outs = (d_out + TILED_OUTS - 1) / TILED_OUTS;
    return (n + 255) / 256 * outs >= 128 ? 256 : (n + 63) / 64 * outs >= 128 ? 64 : 0;
}

Plan make_plan(int dtype, long long n, int d_in, int d_out, int n_slots, int rank, bool grad) {
    Plan p{};
    const size_t esz = dtype == RAG_DTYPE_BF16 ? 2 : 4;
    const int unit = dtype == RAG_DTYPE_BF16 ? 32 : 16;
    auto take = [&](size_t bytes) {
        const size_t at = p.bytes;
        p.bytes += (bytes + 255) & ~(size_t)255;
        return at;
    };
    p.rp = (rank + unit - 1) / unit * unit;
    // Few requests a slot (on average: the host does not see them): U request by request.  A matrix tile of 32 neighbours would go
    // over its slots one after the other (64 requests of 64 slots, 768 wide: 85 us against 4 us); each A_s is read once per
    // request, so only while that stays in the caches.
    p.each = n_slots > 2 && n <= (grad ? 16ll : 32ll) * n_slots && n * rank * std::max(d_in, d_out) * (long long)esz <= (256ll << 20);
    // Then nothing needs an order, and it costs a launch, 7 us for 1000 requests; nor do one or two slots.
    p.sorted = grad || (n > 64 && n_slots > 2 && !p.each);
    p.u = take((size_t)n * p.rp * 4);
    const int e = (int)(16 / esz), in = (d_in + e - 1) / e * e, out = (d_out + e - 1) / e * e, whole_rank = (rank + e - 1) / e * e;
    // pieces of all copies (pad_kernel counts them in 32 bits: a backward with a long x and a short dy has more, and does without)
    const long long pieces = ((long long)n_slots * whole_rank * in + (in > d_in ? n * in : 0) +
                              (grad ? (out > d_out ? n * out : 0)
                                    : (in > d_in ? (long long)d_out * in : 0) + (whole_rank > rank ? (long long)n_slots * d_out * whole_rank : 0))) / e;
    p.pad = (in > d_in || whole_rank > rank || (grad && out > d_out)) && pieces < 1ll << 31 &&
            (grad ? tiled_positions(n, out, d_in, esz) : tiled_positions(n, in, d_out, esz)) > 0;
    p.in = p.pad ? in : d_in;
    p.out = p.pad ? out : d_out;
    p.rank = p.pad ? whole_rank : rank;
    if (p.pad) {
        p.xp = take((size_t)n * in * esz);
        p.ap = take((size_t)n_slots * whole_rank * in * esz);
        if (grad) {
            p.dyp = take((size_t)n * out * esz);
        } else {
            p.wp = take((size_t)d_out * in * esz);
            p.bp = take((size_t)n_slots * d_out * whole_rank * esz);
        }
    }
    if (p.sorted) {
        const bool small = n <= SMALL_N && n_slots + 2 <= SMALL_BINS;
        // (every workgroup of place_kernel reads all counts: fewer chunks where there are many bins)
        const long long most = n_slots + 2 <= SMALL_BINS ? 256 : 64;
        p.chunk = small ? (int)((n + 16 * 64 - 1) / (16 * 64) * 64) : (int)std::max<long long>(256, ((n + most - 1) / most + 63) / 64 * 64);
        p.chunks = small ? 0 : (int)((n + p.chunk - 1) / p.chunk);
        p.perm = take((size_t)n * 4);
        p.slot_at = take((size_t)n * 4);
        p.counts = take((size_t)p.chunks * (n_slots + 2) * 4);
    }
    if (grad) {
        // One item a slot saves the launch that joins partials, 1.4 us; items of 512 shorten the longest chain.  So one item up to a
        // mean of 512 a slot, and up to 2048 requests, since all of them may have the same slot (x 384 float32, items of 512 against
        // one item: 1024 requests of one slot 37 and 48 us, of two 39 and 37, of four 33 and 32; 2000 of four 46 and 45, of sixteen 48
        // and 47; 3000 of two 53 and 76).
        p.len = n <= 512ll * std::min(n_slots, 4) ? (int)std::max<long long>(1, n) : (int)std::max<long long>(512, (n + 255) / 256);
        p.max_items = n_slots + (int)(n / p.len) + 1;
        p.max_parts = 2 * (int)(n / p.len) + 2;
        p.v = take((size_t)n * p.rp * 4);
        p.parts = take((size_t)n_slots * sizeof(int2));
        p.n_items = take(4);
        p.items = take((size_t)p.max_items * sizeof(Item));
        p.wt = take((size_t)d_in * p.out * esz);
        p.at = take((size_t)n_slots * d_in * p.rank * esz);
        p.bt = take((size_t)n_slots * p.rank * p.out * esz);
        p.part = take((size_t)p.max_parts * rank * ((size_t)d_in + d_out) * 4);
    }
    return p;
}

struct Call {
    int dtype, d_in, d_out, n_slots, rank;
    long long n, ldx, ldy, lddy, lddx;
    const void *x, *w, *a, *b, *dy;
    const float* scale;
    const long long* slots;
    void *y, *dx;
    float *da, *db;
    char* ws;
    hipStream_t st;
};

bool aligned16(const void* p, long long ld, size_t esz) { return ((uintptr_t)p & 15) == 0 && ld * (long long)esz % 16 == 0; }

template <typename T>
int run_order(const Call& c, const Plan& p, Sort* out, const Turn* turn) {      // turn: with the list of items, for the backward
    Sort s{};
    s.slots = c.slots;
    s.n = (int)c.n;
    s.n_slots = c.n_slots;
    while ((c.n_slots + 1) >> s.bits) ++s.bits;
    s.chunk = p.chunk;
    s.chunks = p.chunks;
    s.len = p.len;
    s.perm = reinterpret_cast<int*>(c.ws + p.perm);
    s.slot_at = reinterpret_cast<int*>(c.ws + p.slot_at);
    s.counts = reinterpret_cast<int*>(c.ws + p.counts);
    if (turn) {
        s.parts = reinterpret_cast<int2*>(c.ws + p.parts);
        s.n_items = reinterpret_cast<int*>(c.ws + p.n_items);
        s.items = reinterpret_cast<Item*>(c.ws + p.items);
    }
    *out = s;
    const size_t bins = c.n_slots + 2;
    const unsigned tiles = turn ? (unsigned)turn->first[3] : 0;
    if (p.chunks == 0) {
        const size_t lds = std::max<size_t>((17 * bins + 48) * 4, 64 * 66 * sizeof(T));
        if (lds > 48 * 1024)
            RAG_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(prepare_kernel<T>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        prepare_kernel<T><<<1 + tiles, 1024, lds, c.st>>>(s, turn ? *turn : Turn{});
        RAG_HIP(hipGetLastError());
        return RAG_OK;
    }
    const int waves = c.n_slots + 2 <= SMALL_BINS ? 16 : 4;
    const unsigned groups = (unsigned)(p.chunks + 3) / 4;
    const size_t count_lds = std::max<size_t>(4 * bins * 4, 64 * 66 * sizeof(T)), place_lds = ((waves + 1) * bins + 2048) * 4;
    if (count_lds > 48 * 1024)
        RAG_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(count_kernel<T>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)count_lds));
    if (place_lds > 48 * 1024)
        RAG_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(place_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)place_lds));
    count_kernel<T><<<groups + tiles, 256, count_lds, c.st>>>(s, turn ? *turn : Turn{}, groups);
    RAG_HIP(hipGetLastError());
    place_kernel<<<(unsigned)((p.chunks + waves - 1) / waves), 1024, place_lds, c.st>>>(s, waves);
    RAG_HIP(hipGetLastError());
    return RAG_OK;
}

// One matrix more to copy: `count` of rows x cols, or of to_rows x to_cols.
template <typename T>
void pad_more(Pad* j, int* kinds, const void* from, long long ld, void* to, long long count, int rows, int cols, int to_rows, int to_cols) {
    const int i = (*kinds)++;
    j->from[i] = from;
    j->to[i] = to;
    j->ld[i] = ld;
    j->rows[i] = rows;
    j->cols[i] = cols;
    j->to_rows[i] = to_rows;
    j->to_cols[i] = to_cols;
    // (below 2^31 in all: make_plan)
    for (int k = i; k < 4; ++k) j->first[k + 1] = j->first[i] + (unsigned)(count * to_rows * (to_cols / Mma<T>::E));
}
template <typename T>
int launch_pad(const Pad& j, hipStream_t st) {
    if (j.first[4] == 0) return RAG_OK;
    pad_kernel<T><<<(unsigned)std::min<long long>((j.first[4] + 255) / 256, (long long)num_cus() * 32), 256, 0, st>>>(j);
    RAG_HIP(hipGetLastError());
    return RAG_OK;
}

// U of one bank, or U and V of two at once
template <typename T, bool VEC>
int launch_down(const Plan& p, const Down& d, const Order& o, unsigned kinds, hipStream_t st) {
    const Bank& k = d.bank[0];
    if (p.each) {
        down_each_kernel<T, VEC><<<dim3((unsigned)o.n, kinds), 256, 0, st>>>(d, o);
        RAG_HIP(hipGetLastError());
        return RAG_OK;
    }
    const dim3 groups((unsigned)(((o.n + DOWN_TOKENS - 1) / DOWN_TOKENS + 7) / 8 * 8), kinds);
    if (k.rp <= 16) down_kernel<T, 1, VEC><<<groups, 64 * DOWN_WAVES, 0, st>>>(d, o);
    else if (k.rp <= 32) down_kernel<T, 2, VEC><<<groups, 64 * DOWN_WAVES, 0, st>>>(d, o);
    else if (k.rp <= 64) down_kernel<T, 4, VEC><<<groups, 64 * DOWN_WAVES, 0, st>>>(d, o);
    else down_kernel<T, 8, VEC><<<groups, 64 * DOWN_WAVES, 0, st>>>(d, o);
    RAG_HIP(hipGetLastError());
    return RAG_OK;
}

template <typename T, bool VEC>
int launch_up(const Bank& k, const Order& o, const void* x, long long ldx, const float* u, void* y, long long ldy, hipStream_t st) {
    const int pos = VEC ? tiled_positions(o.n, ldx, k.d_out, sizeof(T)) : 0;
    if (pos > 0) {
        const unsigned tiles = (unsigned)(((o.n + pos - 1) / pos + 7) / 8 * 8 * ((k.d_out + TILED_OUTS - 1) / TILED_OUTS));
        const bool short_rank = k.rank <= 4 * Mma<T>::E;
        auto fn = pos == 256 ? (short_rank ? up_tiled_kernel<T, 1, 256> : up_tiled_kernel<T, 2, 256>)
                             : (short_rank ? up_tiled_kernel<T, 1, 64> : up_tiled_kernel<T, 2, 64>);
        RAG_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, tiled_lds_bytes(pos)));
        fn<<<tiles, 512, tiled_lds_bytes(pos), st>>>(k, o, x, ldx, (unsigned)((unsigned long long)o.n * ldx * sizeof(T)), u, y, ldy);
        RAG_HIP(hipGetLastError());
        return RAG_OK;
    }
    auto grid = [&](int ot, int tt) { return (k.d_out + 16 * ot - 1) / (16 * ot) * ((o.n + 16 * tt - 1) / (16 * tt)); };
    auto launch = [&](auto fn, int ot, int tt, int threads) {
        const long long groups = grid(ot, tt), most = MAX_THREADS / threads;
        for (long long first = 0; first < groups; first += most)
            fn<<<(unsigned)std::min(most, groups - first), threads, 0, st>>>(k, o, x, ldx, u, y, ldy, (int)first);
    };
    if (grid(2, 4) >= 1024) launch(up_direct_kernel<T, 2, 4, 4, VEC>, 2, 4, 256);
    else if (grid(1, 4) >= 512) launch(up_direct_kernel<T, 1, 4, 8, VEC>, 1, 4, 512);
    else if (grid(1, 2) >= 512) launch(up_direct_kernel<T, 1, 2, 8, VEC>, 1, 2, 512);
    else launch(up_direct_kernel<T, 1, 1, 8, VEC>, 1, 1, 512);
    RAG_HIP(hipGetLastError());
    return RAG_OK;
}

Bank make_bank(const Call& c, const Plan& p, const void* w, const void* a, const void* b, int d_in, int d_out) {
    const int e = c.dtype == RAG_DTYPE_BF16 ? 8 : 4;
    Bank k{w, a, b, c.scale, d_in, d_out, p.rank, p.rp, c.rank, false, false};
    k.vec_in = d_in % e == 0 && (((uintptr_t)w | (uintptr_t)a) & 15) == 0;
    k.vec_rank = p.rank % e == 0 && ((uintptr_t)b & 15) == 0;
    return k;
}

template <typename T>
int run_apply(const Call& c, const Plan& p) {
    Order o{nullptr, nullptr, c.slots, c.n, c.n_slots};
    if (p.sorted) {
        Sort s;
        const int rc = run_order<T>(c, p, &s, nullptr);
        if (rc) return rc;
        o.perm = s.perm;
        o.slot_at = s.slot_at;
    }
    const void *x = c.x, *w = c.w, *a = c.a, *b = c.b;
    long long ldx = c.ldx;
    if (p.pad) {
        Pad j{};
        int kinds = 0;
        pad_more<T>(&j, &kinds, a, c.d_in, c.ws + p.ap, c.n_slots, c.rank, c.d_in, p.rank, p.in);
        a = c.ws + p.ap;
        if (p.in > c.d_in) {
            pad_more<T>(&j, &kinds, x, ldx, c.ws + p.xp, 1, (int)c.n, c.d_in, (int)c.n, p.in);
            pad_more<T>(&j, &kinds, w, c.d_in, c.ws + p.wp, 1, c.d_out, c.d_in, c.d_out, p.in);
            x = c.ws + p.xp;
            w = c.ws + p.wp;
            ldx = p.in;
        }
        if (p.rank > c.rank) {
            pad_more<T>(&j, &kinds, b, c.rank, c.ws + p.bp, c.n_slots, c.d_out, c.rank, c.d_out, p.rank);
            b = c.ws + p.bp;
        }
        const int rc = launch_pad<T>(j, c.st);
        if (rc) return rc;
    }
    const Bank k = make_bank(c, p, w, a, b, p.in, c.d_out);
    const bool vec = k.vec_in && aligned16(x, ldx, sizeof(T));
    if (c.n <= 16 && c.n * c.rank * c.d_in <= WHOLE_PRODUCTS) {
        const unsigned groups = (unsigned)(c.d_out + 15) / 16;
        if (vec) whole_kernel<T, true><<<groups, 512, 0, c.st>>>(k, o, x, ldx, c.y, c.ldy);
        else whole_kernel<T, false><<<groups, 512, 0, c.st>>>(k, o, x, ldx, c.y, c.ldy);
        RAG_HIP(hipGetLastError());
        return RAG_OK;
    }
    float* u = reinterpret_cast<float*>(c.ws + p.u);
    const Down d{{k, k}, {x, nullptr}, {ldx, 0}, {u, nullptr}};
    if (vec) {
        const int rc = launch_down<T, true>(p, d, o, 1, c.st);
        return rc ? rc : launch_up<T, true>(k, o, x, ldx, u, c.y, c.ldy, c.st);
    }
    const int rc = launch_down<T, false>(p, d, o, 1, c.st);
    return rc ? rc : launch_up<T, false>(k, o, x, ldx, u, c.y, c.ldy, c.st);
}

template <typename T>
int run_grad(const Call& c, const Plan& p) {
    // the transposed bank: B always (v), W and A for dx
    Turn t{};
    const void* from[3] = {c.b, c.w, c.a};
    void* to[3] = {c.ws + p.bt, c.ws + p.wt, c.ws + p.at};
    const int rows[3] = {c.d_out, c.d_out, c.rank}, cols[3] = {c.rank, c.d_in, c.d_in}, count[3] = {c.n_slots, 1, c.n_slots};
    for (int i = 0; i < 3; ++i) {
        t.from[i] = from[i];
        t.to[i] = to[i];
        t.rows[i] = rows[i];
        t.cols[i] = cols[i];
        t.to_rows[i] = i == 0 ? p.rank : c.d_in;
        t.to_cols[i] = i == 2 ? p.rank : p.out;
        t.first[i + 1] = t.first[i] + (c.n > 0 && (i == 0 || c.dx) ? count[i] * ((t.to_rows[i] + 63) / 64) * ((t.to_cols[i] + 63) / 64) : 0);
    }
    Sort s;
    int rc = run_order<T>(c, p, &s, &t);
    if (rc) return rc;
    constexpr int E = Mma<T>::E;
    const Order o{s.perm, s.slot_at, c.slots, c.n, c.n_slots};
    float* u = reinterpret_cast<float*>(c.ws + p.u);
    float* v = reinterpret_cast<float*>(c.ws + p.v);
    const void *x = c.x, *a = c.a, *dy = c.dy;
    long long ldx = c.ldx, lddy = c.lddy;
    if (p.pad) {
        Pad j{};
        int kinds = 0;
        pad_more<T>(&j, &kinds, a, c.d_in, c.ws + p.ap, c.n_slots, c.rank, c.d_in, p.rank, p.in);
        a = c.ws + p.ap;
        if (p.in > c.d_in) {
            pad_more<T>(&j, &kinds, x, ldx, c.ws + p.xp, 1, (int)c.n, c.d_in, (int)c.n, p.in);
            x = c.ws + p.xp;
            ldx = p.in;
        }
        if (p.out > c.d_out) {
            pad_more<T>(&j, &kinds, dy, lddy, c.ws + p.dyp, 1, (int)c.n, c.d_out, (int)c.n, p.out);
            dy = c.ws + p.dyp;
            lddy = p.out;
        }
        rc = launch_pad<T>(j, c.st);
        if (rc) return rc;
    }
    const SlotGrad g{s, u, v, x, dy, ldx, lddy, c.da, c.db, reinterpret_cast<float*>(c.ws + p.part), c.d_in, c.d_out, c.rank, p.rp,
                     p.in, p.out, p.in % E == 0 && aligned16(x, ldx, sizeof(T)), p.out % E == 0 && aligned16(dy, lddy, sizeof(T))};
    const Bank fore = make_bank(c, p, c.w, a, c.b, p.in, c.d_out), back = make_bank(c, p, to[1], to[0], to[2], p.out, c.d_in);
    const bool vec = fore.vec_in && g.vec_x && back.vec_in && g.vec_dy;
    if (c.n > 0) {
        const Down d{{fore, back}, {x, dy}, {ldx, lddy}, {u, v}};
        rc = vec ? launch_down<T, true>(p, d, o, 2, c.st) : launch_down<T, false>(p, d, o, 2, c.st);
        if (rc) return rc;
    }
    const long long ups = (long long)((c.d_in + 15) / 16) * ((c.n + 31) / 32);
    const bool together = c.n > 0 && c.dx && !(vec && tiled_positions(c.n, lddy, c.d_in, sizeof(T)) > 0) && ups * 512 <= MAX_THREADS;
    if (c.n > 0 && c.dx && !together) {
        rc = vec ? launch_up<T, true>(back, o, dy, lddy, v, c.dx, c.lddx, c.st)
                 : launch_up<T, false>(back, o, dy, lddy, v, c.dx, c.lddx, c.st);
        if (rc) return rc;
    }
    auto launch = [&](auto rt) {
        constexpr int RT = rt.value;
        const int units = ((c.d_in + 16 * E - 1) / (16 * E) + (c.d_out + 16 * E - 1) / (16 * E)) * ((c.rank + 16 * RT - 1) / (16 * RT));
        if (!together) {
            slot_grad_kernel<T, RT><<<dim3((unsigned)p.max_items, (unsigned)units), 256, 0, c.st>>>(g);
            return;
        }
        const unsigned groups = (unsigned)((units + 1) / 2);
        auto fn = vec ? up_and_slot_kernel<T, RT, true> : up_and_slot_kernel<T, RT, false>;
        const unsigned slot_groups = (unsigned)p.max_items * groups;
        // the fewer workgroups first, which the others then fill the card beside (1024 requests of 4 slots: 40 us with the bank's
        // last, 37 first; 64 of 64: 31, 36)
        const bool first = slot_groups <= ups;
        fn<<<slot_groups + (unsigned)ups, 512, 0, c.st>>>(back, o, dy, lddy, v, c.dx, c.lddx, first ? slot_groups : 0u, first ? 0u : (unsigned)ups,
                                                          slot_groups, g, groups);
    };
    if (c.rank <= 16) launch(std::integral_constant<int, 1>());
    else if (c.rank <= 32) launch(std::integral_constant<int, 2>());
    else launch(std::integral_constant<int, 4>());
    RAG_HIP(hipGetLastError());
    if (c.n > p.len) {               // (else every slot is one item)
        const long long size = (long long)c.rank * (c.d_in + c.d_out);
        slot_join_kernel<<<dim3((unsigned)c.n_slots, (unsigned)std::min<long long>(64, (size + 255) / 256)), 256, 0, c.st>>>(g);
        RAG_HIP(hipGetLastError());
    }
    return RAG_OK;
}

int check_shape(const char* who, int dtype, int64_t n, int d_in, int d_out, int n_slots, int rank) {
    if (dtype != RAG_DTYPE_F32 && dtype != RAG_DTYPE_BF16)
        return fail(RAG_ERR_INVALID_ARG, "%s: dtype %d is neither fp32(0) nor bf16(1)", who, dtype);
    if (n < 0 || n > RAG_ADAPTER_MAX_N)
        return fail(RAG_ERR_INVALID_ARG, "%s: n=%lld out of range [0,%d]", who, (long long)n, RAG_ADAPTER_MAX_N);
    if (d_in < 1 || d_in > 8192 || d_out < 1 || d_out > 8192)
        return fail(RAG_ERR_INVALID_ARG, "%s: d_in=%d, d_out=%d out of range [1,8192]", who, d_in, d_out);
    if (n_slots < 1 || n_slots > RAG_ADAPTER_MAX_SLOTS)
        return fail(RAG_ERR_INVALID_ARG, "%s: n_slots=%d out of range [1,%d]", who, n_slots, RAG_ADAPTER_MAX_SLOTS);
    if (rank < 1 || rank > RAG_ADAPTER_MAX_RANK)
        return fail(RAG_ERR_INVALID_ARG, "%s: rank=%d out of range [1,%d]", who, rank, RAG_ADAPTER_MAX_RANK);
    return RAG_OK;
}

}  // namespace

extern "C" {

int rag_adapter_ws_bytes(int dtype, int64_t n, int d_in, int d_out, int n_slots, int rank, int want_grad, int64_t* bytes) {
    const int rc = check_shape("rag_adapter_ws_bytes", dtype, n, d_in, d_out, n_slots, rank);
    if (rc) return rc;
    if (!bytes) return fail(RAG_ERR_INVALID_ARG, "rag_adapter_ws_bytes: bytes is NULL");
    *bytes = (int64_t)make_plan(dtype, n, d_in, d_out, n_slots, rank, want_grad != 0).bytes;
    return RAG_OK;
}

int rag_adapter_apply_dev(int dtype, int64_t n, int d_in, int d_out, int n_slots, int rank, const void* x_dev, int64_t ldx,
                          const void* w_dev, const void* a_dev, const void* b_dev, const float* scale_dev,
                          const int64_t* slots_dev, void* y_dev, int64_t ldy, void* ws_dev, int64_t ws_bytes, void* stream) {
    const char* who = "rag_adapter_apply_dev";
    RAG_REQUIRE_INIT();
    const int rc = check_shape(who, dtype, n, d_in, d_out, n_slots, rank);
    if (rc) return rc;
    if (n == 0) return RAG_OK;
    if (!x_dev || !w_dev || !a_dev || !b_dev || !scale_dev || !slots_dev || !y_dev)
        return fail(RAG_ERR_INVALID_ARG, "%s: NULL buffer", who);
    if (ldx < d_in || ldy < d_out)
        return fail(RAG_ERR_INVALID_ARG, "%s: row strides %lld / %lld are below d_in=%d / d_out=%d", who, (long long)ldx,
                    (long long)ldy, d_in, d_out);
    const Plan p = make_plan(dtype, n, d_in, d_out, n_slots, rank, false);
    if (!ws_dev || ws_bytes < (int64_t)p.bytes || ((uintptr_t)ws_dev & 255))
        return fail(RAG_ERR_INVALID_ARG, "%s: needs a workspace of %lld bytes, aligned to 256 (rag_adapter_ws_bytes)", who,
                    (long long)p.bytes);
    Call c{};
    c.dtype = dtype; c.n = n; c.d_in = d_in; c.d_out = d_out; c.n_slots = n_slots; c.rank = rank;
    c.x = x_dev; c.ldx = ldx; c.w = w_dev; c.a = a_dev; c.b = b_dev; c.scale = scale_dev;
    c.slots = reinterpret_cast<const long long*>(slots_dev);
    c.y = y_dev; c.ldy = ldy;
    c.ws = static_cast<char*>(ws_dev);
    c.st = (hipStream_t)stream;
    DeviceScope dev;
    return dtype == RAG_DTYPE_BF16 ? run_apply<u16>(c, p) : run_apply<float>(c, p);
}

int rag_adapter_grad_dev(int dtype, int64_t n, int d_in, int d_out, int n_slots, int rank, const void* x_dev, int64_t ldx,
                         const void* w_dev, const void* a_dev, const void* b_dev, const float* scale_dev,
                         const int64_t* slots_dev, const void* dy_dev, int64_t lddy, void* dx_dev, int64_t lddx,
                         float* da_dev, float* db_dev, void* ws_dev, int64_t ws_bytes, void* stream) {
    const char* who = "rag_adapter_grad_dev";
    RAG_REQUIRE_INIT();
    const int rc = check_shape(who, dtype, n, d_in, d_out, n_slots, rank);
    if (rc) return rc;
    if (!da_dev || !db_dev) return fail(RAG_ERR_INVALID_ARG, "%s: NULL buffer", who);
    if (n > 0 && (!x_dev || !w_dev || !a_dev || !b_dev || !scale_dev || !slots_dev || !dy_dev))
        return fail(RAG_ERR_INVALID_ARG, "%s: NULL buffer", who);
    if (n > 0 && (ldx < d_in || lddy < d_out || (dx_dev && lddx < d_in)))
        return fail(RAG_ERR_INVALID_ARG, "%s: row strides %lld / %lld / %lld are below d_in=%d / d_out=%d / d_in", who,
                    (long long)ldx, (long long)lddy, (long long)lddx, d_in, d_out);
    const Plan p = make_plan(dtype, n, d_in, d_out, n_slots, rank, true);
    if (!ws_dev || ws_bytes < (int64_t)p.bytes || ((uintptr_t)ws_dev & 255))
        return fail(RAG_ERR_INVALID_ARG, "%s: needs a workspace of %lld bytes, aligned to 256 (rag_adapter_ws_bytes)", who,
                    (long long)p.bytes);
    Call c{};
    c.dtype = dtype; c.n = n; c.d_in = d_in; c.d_out = d_out; c.n_slots = n_slots; c.rank = rank;
    c.x = x_dev; c.ldx = ldx; c.w = w_dev; c.a = a_dev; c.b = b_dev; c.scale = scale_dev;
    c.slots = reinterpret_cast<const long long*>(slots_dev);
    c.dy = dy_dev; c.lddy = lddy; c.dx = dx_dev; c.lddx = lddx; c.da = da_dev; c.db = db_dev;
    c.ws = static_cast<char*>(ws_dev);
    c.st = (hipStream_t)stream;
    DeviceScope dev;
    return dtype == RAG_DTYPE_BF16 ? run_grad<u16>(c, p) : run_grad<float>(c, p);
}

}  // extern "C"
