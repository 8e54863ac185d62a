// adapter.hip -- low-rank adapters of many requests beside a shared projection (rag_adapter_apply_dev / _grad_dev).
//
// Request t has an embedding x_t and a slot s = slots[t] (-1: no adapter) of a bank A (slots x R x d_in),
// B (slots x d_out x R), scale c (slots):
//     u_t = c_s A_s x_t                 y_t = W x_t + B_s u_t
// and, with dy the gradient of y (W is frozen),
//     v_t = c_s B_s^T dy_t              dx_t = W^T dy_t + A_s^T v_t
//     dA_s = sum_t v_t x_t^T            dB_s = sum_t dy_t u_t^T      over the requests of slot s.
// u, v, dA, dB and every sum are fp32; y and dx are rounded once, to the type of x.
#include "common.h"

#include <algorithm>

namespace {

using namespace rag;

constexpr int THREADS = 256;

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const unsigned short* p) { return __uint_as_float((unsigned)*p << 16); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(unsigned short* p, float f) {
    const unsigned u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) *p = (unsigned short)((u >> 16) | 0x40);   // NaN stays NaN
    else *p = (unsigned short)((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
}
__device__ __forceinline__ float wave_sum(float v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

struct Call {
    long long n, ldx, ldy, lddy, lddx;
    int d_in, d_out, slots_n, rank;
    const void *x, *w, *a, *b, *dy;
    const float* scale;
    const long long* slots;
    void *y, *dx;
    float *da, *db;
    float *u, *v;   // n x R
};

// slot of a request: >= 0, -1 (none) or -2 (outside the bank: its results are NaN)
__device__ __forceinline__ int slot_of(const Call& c, long long t) {
    const long long s = c.slots[t];
    return s >= -1 && s < c.slots_n ? (int)s : -2;
}

template <typename T>
__global__ __launch_bounds__(THREADS) void down_kernel(Call c) {
    const long long t = blockIdx.x;
    const int s = slot_of(c, t), lane = threadIdx.x & 63;
    const T* x = static_cast<const T*>(c.x) + t * c.ldx;
    for (int r = threadIdx.x >> 6; r < c.rank; r += THREADS / 64) {
        float acc = 0.f;
        if (s >= 0) {
            const T* a = static_cast<const T*>(c.a) + ((long long)s * c.rank + r) * c.d_in;
            for (int j = lane; j < c.d_in; j += 64) acc = fmaf(load1(a + j), load1(x + j), acc);
            acc = wave_sum(acc) * c.scale[s];
        }
        if (lane == 0) c.u[t * c.rank + r] = s == -2 ? NAN : acc;
    }
}

template <typename T>
__global__ __launch_bounds__(THREADS) void apply_kernel(Call c) {
    const long long t = blockIdx.x;
    const int s = slot_of(c, t), lane = threadIdx.x & 63;
    const T* x = static_cast<const T*>(c.x) + t * c.ldx;
    for (int o = threadIdx.x >> 6; o < c.d_out; o += THREADS / 64) {
        const T* w = static_cast<const T*>(c.w) + (long long)o * c.d_in;
        float acc = 0.f;
        for (int j = lane; j < c.d_in; j += 64) acc = fmaf(load1(w + j), load1(x + j), acc);
        if (s >= 0) {
            const T* b = static_cast<const T*>(c.b) + ((long long)s * c.d_out + o) * c.rank;
            for (int r = lane; r < c.rank; r += 64) acc = fmaf(load1(b + r), c.u[t * c.rank + r], acc);
        }
        acc = wave_sum(acc);
        if (lane == 0) store1(static_cast<T*>(c.y) + t * c.ldy + o, s == -2 ? NAN : acc);
    }
}

template <typename T>
__global__ __launch_bounds__(THREADS) void up_grad_kernel(Call c) {
    const long long t = blockIdx.x;
    const int s = slot_of(c, t);
    const T* dy = static_cast<const T*>(c.dy) + t * c.lddy;
    for (int r = threadIdx.x; r < c.rank; r += THREADS) {
        float acc = 0.f;
        if (s >= 0) {
            const T* b = static_cast<const T*>(c.b) + (long long)s * c.d_out * c.rank + r;
            for (int o = 0; o < c.d_out; ++o) acc = fmaf(load1(b + (long long)o * c.rank), load1(dy + o), acc);
            acc *= c.scale[s];
        }
        c.v[t * c.rank + r] = s == -2 ? NAN : acc;
    }
}

template <typename T>
__global__ __launch_bounds__(THREADS) void input_grad_kernel(Call c) {
    const long long t = blockIdx.x;
    const int s = slot_of(c, t);
    const T* dy = static_cast<const T*>(c.dy) + t * c.lddy;
    for (int j = threadIdx.x; j < c.d_in; j += THREADS) {
        float acc = 0.f;
        for (int o = 0; o < c.d_out; ++o)
            acc = fmaf(load1(static_cast<const T*>(c.w) + (long long)o * c.d_in + j), load1(dy + o), acc);
        if (s >= 0)
            for (int r = 0; r < c.rank; ++r)
                acc = fmaf(load1(static_cast<const T*>(c.a) + ((long long)s * c.rank + r) * c.d_in + j), c.v[t * c.rank + r], acc);
        store1(static_cast<T*>(c.dx) + t * c.lddx + j, s == -2 ? NAN : acc);
    }
}

template <typename T>
__global__ __launch_bounds__(THREADS) void a_grad_kernel(Call c) {
    const int s = blockIdx.x / c.rank, r = blockIdx.x % c.rank;
    for (int j = threadIdx.x; j < c.d_in; j += THREADS) {
        float acc = 0.f;
        for (long long t = 0; t < c.n; ++t)
            if (c.slots[t] == s) acc = fmaf(c.v[t * c.rank + r], load1(static_cast<const T*>(c.x) + t * c.ldx + j), acc);
        c.da[((long long)s * c.rank + r) * c.d_in + j] = acc;
    }
}

template <typename T>
__global__ __launch_bounds__(THREADS) void b_grad_kernel(Call c) {
    const int s = blockIdx.x, o = blockIdx.y;
    for (int r = threadIdx.x; r < c.rank; r += THREADS) {
        float acc = 0.f;
        for (long long t = 0; t < c.n; ++t)
            if (c.slots[t] == s) acc = fmaf(load1(static_cast<const T*>(c.dy) + t * c.lddy + o), c.u[t * c.rank + r], acc);
        c.db[((long long)s * c.d_out + o) * c.rank + r] = acc;
    }
}

struct Plan {
    size_t u_off, v_off, bytes;
};

Plan make_plan(long long n, int rank, bool grad) {
    Plan p{};
    auto take = [&](size_t bytes) {
        const size_t at = p.bytes;
        p.bytes += (bytes + 255) & ~(size_t)255;
        return at;
    };
    p.u_off = take((size_t)n * rank * sizeof(float));
    p.v_off = take(grad ? (size_t)n * rank * sizeof(float) : 0);
    return p;
}

template <typename T>
int run_apply(const Call& c, hipStream_t st) {
    const unsigned n = (unsigned)c.n;
    down_kernel<T><<<n, THREADS, 0, st>>>(c);
    RAG_HIP(hipGetLastError());
    apply_kernel<T><<<n, THREADS, 0, st>>>(c);
    RAG_HIP(hipGetLastError());
    return RAG_OK;
}

template <typename T>
int run_grad(const Call& c, hipStream_t st) {
    const unsigned n = (unsigned)c.n;
    if (n > 0) {
        down_kernel<T><<<n, THREADS, 0, st>>>(c);
        RAG_HIP(hipGetLastError());
        up_grad_kernel<T><<<n, THREADS, 0, st>>>(c);
        RAG_HIP(hipGetLastError());
        if (c.dx) {
            input_grad_kernel<T><<<n, THREADS, 0, st>>>(c);
            RAG_HIP(hipGetLastError());
        }
    }
    a_grad_kernel<T><<<(unsigned)(c.slots_n * c.rank), THREADS, 0, st>>>(c);
    RAG_HIP(hipGetLastError());
    b_grad_kernel<T><<<dim3((unsigned)c.slots_n, (unsigned)c.d_out), THREADS, 0, st>>>(c);
    RAG_HIP(hipGetLastError());
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
    *bytes = (int64_t)make_plan(n, rank, want_grad != 0).bytes;
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
    const Plan p = make_plan(n, rank, false);
    if (!ws_dev || ws_bytes < (int64_t)p.bytes || ((uintptr_t)ws_dev & 255))
        return fail(RAG_ERR_INVALID_ARG, "%s: needs a workspace of %lld bytes, aligned to 256 (rag_adapter_ws_bytes)", who,
                    (long long)p.bytes);
    Call c{};
    c.n = n; c.d_in = d_in; c.d_out = d_out; c.slots_n = n_slots; c.rank = rank;
    c.x = x_dev; c.ldx = ldx; c.w = w_dev; c.a = a_dev; c.b = b_dev; c.scale = scale_dev;
    c.slots = reinterpret_cast<const long long*>(slots_dev);
    c.y = y_dev; c.ldy = ldy;
    c.u = reinterpret_cast<float*>(static_cast<char*>(ws_dev) + p.u_off);
    DeviceScope dev;
    return dtype == RAG_DTYPE_BF16 ? run_apply<unsigned short>(c, (hipStream_t)stream) : run_apply<float>(c, (hipStream_t)stream);
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
    const Plan p = make_plan(n, rank, true);
    if (n > 0 && (!ws_dev || ws_bytes < (int64_t)p.bytes || ((uintptr_t)ws_dev & 255)))
        return fail(RAG_ERR_INVALID_ARG, "%s: needs a workspace of %lld bytes, aligned to 256 (rag_adapter_ws_bytes)", who,
                    (long long)p.bytes);
    Call c{};
    c.n = n; c.d_in = d_in; c.d_out = d_out; c.slots_n = n_slots; c.rank = rank;
    c.x = x_dev; c.ldx = ldx; c.w = w_dev; c.a = a_dev; c.b = b_dev; c.scale = scale_dev;
    c.slots = reinterpret_cast<const long long*>(slots_dev);
    c.dy = dy_dev; c.lddy = lddy; c.dx = dx_dev; c.lddx = lddx; c.da = da_dev; c.db = db_dev;
    c.u = reinterpret_cast<float*>(static_cast<char*>(ws_dev) + p.u_off);
    c.v = reinterpret_cast<float*>(static_cast<char*>(ws_dev) + p.v_off);
    DeviceScope dev;
    return dtype == RAG_DTYPE_BF16 ? run_grad<unsigned short>(c, (hipStream_t)stream) : run_grad<float>(c, (hipStream_t)stream);
}

}  // extern "C"
