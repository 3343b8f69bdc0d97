// Layer norm over the last dimension, forward and backward, for sm_100a.
//     mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r, y = h w + b
//     c = dy w:  dx = r (c - mean(c) - h mean(c h)),   dw = sum_rows dy h,   db = sum_rows dy
// Bound by HBM: x in and y out, or x and dy in and dx out, once.  TPR threads own a row and keep
// it in registers (E elements each), so the second pass of the variance and the output need no
// second reading.  All sums are float32.
//
// Measured (32768 rows, forward and backward): 2564 float32 99 us (6.8 TB/s) and 170 (5.9); 2565 float32,
// whose rows allow no vectors, 121 (5.6) and 187 (5.4); 2560 bfloat16 70 (4.8) and 116 (4.3): half of the
// bytes in flight per row, and the warps wait for them (at 16384 x 768 the first stall, with issue at 38 to 46%).
//
// Backward: a thread owns the same columns of every row it meets, so the sums of dw and db
// stay in its registers over all rows of a CTA; each CTA leaves one partial row, and a second
// kernel adds the partial rows in a fixed order (deterministic, no floating-point atomics).
//
// Rows of more than 8192 elements do not fit the registers: they are read again for each pass
// (from L2), element by element, and dw and db get a pass of their own.  4096 rows of 16384: bfloat16 97 us
// forward (2.8 TB/s) and 238 backward (1.7), float32 117 (4.6) and 328 (2.5).
#include <atomic>

#include "common.cuh"
#include "params.h"

namespace ssm {

namespace {

// VT elements from p as raw bits, widened when used
template <typename T, int VT> struct Raw;
template <> struct Raw<float, 4> { float4 r; __device__ void load(const float* p) { r = *reinterpret_cast<const float4*>(p); }
    __device__ float get(int i) const { return i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w; } };
template <> struct Raw<float, 1> { float r; __device__ void load(const float* p) { r = *p; } __device__ float get(int) const { return r; } };
template <> struct Raw<__nv_bfloat16, 8> { uint4 r; __device__ void load(const __nv_bfloat16* p) { r = *reinterpret_cast<const uint4*>(p); }
    __device__ float get(int i) const {
        const uint32_t w = i < 2 ? r.x : i < 4 ? r.y : i < 6 ? r.z : r.w;
        return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
    } };
template <> struct Raw<__nv_bfloat16, 2> { uint32_t r; __device__ void load(const __nv_bfloat16* p) { r = *reinterpret_cast<const uint32_t*>(p); }
    __device__ float get(int i) const { return __uint_as_float((i & 1) ? (r & 0xffff0000u) : (r << 16)); } };
template <> struct Raw<__nv_bfloat16, 1> { __nv_bfloat16 r; __device__ void load(const __nv_bfloat16* p) { r = *p; }
    __device__ float get(int) const { return __bfloat162float(r); } };

template <int VT>
__device__ __forceinline__ void load_f32(const float* p, float (&v)[VT]) {
    if constexpr (VT == 1) {
        v[0] = *p;
    } else if constexpr (VT == 2) {
        const float2 x = *reinterpret_cast<const float2*>(p);
        v[0] = x.x; v[1] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < VT; i += 4) {
            const float4 x = *reinterpret_cast<const float4*>(p + i);
            v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w;
        }
    }
}

template <typename T, int VT>
__device__ __forceinline__ void store_elems(T* p, const float (&v)[VT]) {
    if constexpr (VT == 1) {
        *p = from_f<T>(v[0]);
    } else if constexpr (VT == 2) {
        store_pair<T>(p, make_float2(v[0], v[1]));
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 x = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&x);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Sums of N values over the TPR threads of a row; every thread gets them.  Rows of one warp need
// no barrier; wider rows are the CTA's only row, and `slot` alternates so that one barrier
// per sum is enough.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* slot) {
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int m = 16; m >= 1; m >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], m);
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
        for (int i = 0; i < N; i++)
            if (lane == 0) slot[i * W + warp] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < W; w++) s += slot[i * W + w];
            v[i] = s;
        }
    }
}

template <int TPR> constexpr int kRowsPerCta = TPR > 32 ? 1 : 4;

template <typename T, int VT, int E, int TPR>
__global__ void __launch_bounds__(TPR * kRowsPerCta<TPR>) layer_norm_fwd_kernel(const __grid_constant__ LnParams p) {
    constexpr int NV = E / VT, RPC = kRowsPerCta<TPR>;
    __shared__ float slots[2][TPR / 32];
    const int64_t row = (int64_t)blockIdx.x * RPC + threadIdx.x / TPR;
    const int tid = threadIdx.x % TPR;
    if (row >= p.rows) return;                    // whole warps; with TPR > 32 whole CTAs
    const T* x = static_cast<const T*>(p.x) + row * p.x_s;
    Raw<T, VT> xr[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (tid + i * TPR) * VT;
        if (c < p.dim) xr[i].load(x + c);
    }
    float v[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; i++)
        if ((tid + i * TPR) * VT < p.dim)
#pragma unroll
            for (int j = 0; j < VT; j++) v[0] += xr[i].get(j);
    row_sum<TPR>(v, slots[0]);
    const float mean = v[0] / (float)p.dim;    // a division: exact for a constant row's exact sum
    v[0] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; i++)
        if ((tid + i * TPR) * VT < p.dim)
#pragma unroll
            for (int j = 0; j < VT; j++) {
                const float d = xr[i].get(j) - mean;
                v[0] = fmaf(d, d, v[0]);
            }
    row_sum<TPR>(v, slots[1]);
    const float rstd = rsqrtf(fmaf(v[0], p.inv_dim, p.eps));
    if (tid == 0 && p.mean) {
        p.mean[row] = mean;
        p.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(p.y) + row * p.y_s;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (tid + i * TPR) * VT;
        if (c >= p.dim) continue;
        float o[VT], t[VT];
#pragma unroll
        for (int j = 0; j < VT; j++) o[j] = (xr[i].get(j) - mean) * rstd;
        if (p.weight) {
            load_f32<VT>(p.weight + c, t);
#pragma unroll
            for (int j = 0; j < VT; j++) o[j] *= t[j];
        }
        if (p.bias) {
            load_f32<VT>(p.bias + c, t);
#pragma unroll
            for (int j = 0; j < VT; j++) o[j] += t[j];
        }
        store_elems<T, VT>(y + c, o);
    }
}

// Rows on their way through shared memory, cnt elements from p to `at`, by TPR threads.  Vectors of 16
// bytes go each to the place where the same thread takes it up again.  Rows that allow none are copied
// in aligned pieces of 16 bytes and read from their first element on once all threads' pieces
// are there (32768 rows of 1601 bfloat16: 157 us with a copy per element, 111 so; 2565 float32: 235, 187).  The
// first piece begins up to 15 bytes before the row, in the aligned 16 bytes that hold its first
// element; the last one ends with the row.
template <typename T, int VT, int E, int TPR>
struct Flight {
    static constexpr bool kWhole = VT * sizeof(T) < 16;
    static constexpr int kBytes = E * TPR * (int)sizeof(T) + (kWhole ? 16 : 0);     // of a row's place
    static __device__ int head(const T* p) { return kWhole ? (int)(reinterpret_cast<uintptr_t>(p) & 15) : 0; }
    static __device__ void start(unsigned char* at, const T* p, int cnt) {
        const int tid = threadIdx.x % TPR, end = head(p) + cnt * (int)sizeof(T);
        const unsigned char* from = reinterpret_cast<const unsigned char*>(p) - head(p);
        const uint32_t to = (uint32_t)__cvta_generic_to_shared(at);
#pragma unroll
        for (int i = 0; i < (kBytes / 16 + TPR - 1) / TPR; i++) {
            const int k = (tid + i * TPR) * 16;
            if (k < end)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + k), "l"(from + k),
                             "r"(min(end - k, 16))
                             : "memory");
        }
    }
};

// Backward: rows in flight per row in work, so that an SM has the 40 KB and more under way that HBM
// needs; with one row ahead in registers 32768 float32 rows of 2565 took 255 us.
constexpr int kAhead = 2;
template <typename T, int VT, int E, int TPR>
constexpr int kBwdBytes = (kAhead + 1) * kRowsPerCta<TPR> * (2 * Flight<T, VT, E, TPR>::kBytes + TPR / 32 * 8);

template <typename T, int VT, int E, int TPR>
__global__ void __launch_bounds__(TPR * kRowsPerCta<TPR>) layer_norm_bwd_kernel(const __grid_constant__ LnParams p) {
    constexpr int NV = E / VT, RPC = kRowsPerCta<TPR>, WARPS = TPR * RPC / 32;
    using Rows = Flight<T, VT, E, TPR>;
    __shared__ float slots[2][2 * (TPR / 32)];
    __shared__ float fold[RPC > 1 ? RPC * TPR * VT : 1];
    // [stage][x, dy][row], then [stage][warp] mean and rstd
    extern __shared__ __align__(16) unsigned char flight[];
    float2* stats = reinterpret_cast<float2*>(flight + (kAhead + 1) * 2 * RPC * Rows::kBytes);
    const int tid = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    float dw[NV][VT] = {}, db[NV][VT] = {};
    auto place = [&](int stage, int which) { return flight + ((stage * 2 + which) * RPC + sub) * Rows::kBytes; };
    auto stat = [&](int stage) { return stats + stage * WARPS + threadIdx.x / 32; };
    auto x_row = [&](int64_t row) { return static_cast<const T*>(p.x) + row * p.x_s; };
    auto dy_row = [&](int64_t row) { return static_cast<const T*>(p.dy) + row * p.dy_s; };
    auto fetch = [&](int64_t row, int stage) {
        if (row < p.rows) {
            Rows::start(place(stage, 0), x_row(row), p.dim);
            Rows::start(place(stage, 1), dy_row(row), p.dim);
            if (threadIdx.x % 32 == 0) {
                const uint32_t to = (uint32_t)__cvta_generic_to_shared(stat(stage));
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(p.mean + row) : "memory");
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + 4), "l"(p.rstd + row) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // narrow vectors: the weights stay in registers too
    constexpr bool kKeep = VT < 8;
    float kept[kKeep ? NV : 1][VT];
    if (kKeep) {
#pragma unroll
        for (int i = 0; i < (kKeep ? NV : 1); i++) {
            const int c = (tid + i * TPR) * VT;
            if (p.weight && c < p.dim) load_f32<VT>(p.weight + c, kept[i]);
            else
#pragma unroll
                for (int j = 0; j < VT; j++) kept[i][j] = 1.f;
        }
    }
    auto weights = [&](int i, float (&w)[VT]) {
        const int c = (tid + i * TPR) * VT;
        if (!kKeep && p.weight) {
            load_f32<VT>(p.weight + c, w);
        } else {
#pragma unroll
            for (int j = 0; j < VT; j++) w[j] = kKeep ? kept[i][j] : 1.f;
        }
    };
    const int64_t step = (int64_t)gridDim.x * RPC, first = (int64_t)blockIdx.x * RPC + sub;
    int turn = 0, stage = 0;
#pragma unroll
    for (int i = 0; i < kAhead; i++) fetch(first + i * step, i);
    for (int64_t row = first; row < p.rows; row += step, turn ^= 1, stage = stage == kAhead ? 0 : stage + 1) {
        fetch(row + kAhead * step, stage == 0 ? kAhead : stage - 1);     // the stage of the row before
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
        if (Rows::kWhole && TPR > 32) __syncthreads();
        else __syncwarp();                        // mean and rstd come by lane 0
        const T* xs = reinterpret_cast<const T*>(place(stage, 0) + Rows::head(x_row(row)));
        const T* gs = reinterpret_cast<const T*>(place(stage, 1) + Rows::head(dy_row(row)));
        const float mean = stat(stage)->x, rstd = stat(stage)->y;
        struct {
            Raw<T, VT> x[NV], g[NV];
        } now;
        float v[2] = {0.f, 0.f};                  // sum of c, sum of c h
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (tid + i * TPR) * VT;
            if (c >= p.dim) continue;
            now.x[i].load(xs + c);
            now.g[i].load(gs + c);
            float w[VT];
            weights(i, w);
#pragma unroll
            for (int j = 0; j < VT; j++) {
                const float g = now.g[i].get(j), h = (now.x[i].get(j) - mean) * rstd, e = g * w[j];
                v[0] += e;
                v[1] = fmaf(e, h, v[1]);
                dw[i][j] = fmaf(g, h, dw[i][j]);
                db[i][j] += g;
            }
        }
        row_sum<TPR>(v, slots[turn]);
        const float m0 = v[0] * p.inv_dim, m1 = v[1] * p.inv_dim;
        T* dx = static_cast<T*>(p.dx) + row * p.dx_s;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (tid + i * TPR) * VT;
            if (c >= p.dim) continue;
            float o[VT], w[VT];
            weights(i, w);
#pragma unroll
            for (int j = 0; j < VT; j++) {
                const float h = (now.x[i].get(j) - mean) * rstd;
                o[j] = rstd * (now.g[i].get(j) * w[j] - m0 - h * m1);
            }
            store_elems<T, VT>(dx + c, o);
        }
    }
    // one partial row per CTA: [cta][0] dw, [cta][1] db
    float* out = p.part + (int64_t)blockIdx.x * 2 * p.dim;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        if (which ? !p.dbias : !p.dweight) continue;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (tid + i * TPR) * VT;
            if constexpr (RPC > 1) {
                __syncthreads();
#pragma unroll
                for (int j = 0; j < VT; j++) fold[sub * TPR * VT + j * TPR + tid] = which ? db[i][j] : dw[i][j];
                __syncthreads();
                if (sub == 0 && c < p.dim)
#pragma unroll
                    for (int j = 0; j < VT; j++) {
                        float s = 0.f;
#pragma unroll
                        for (int q = 0; q < RPC; q++) s += fold[q * TPR * VT + j * TPR + tid];
                        out[which * p.dim + c + j] = s;
                    }
            } else if (c < p.dim) {
#pragma unroll
                for (int j = 0; j < VT; j++) out[which * p.dim + c + j] = which ? db[i][j] : dw[i][j];
            }
        }
    }
}

// ---- rows too long for the registers ----------------------------------------------------------
constexpr int kWide = 512;

template <typename T>
__global__ void __launch_bounds__(kWide) layer_norm_wide_fwd_kernel(const __grid_constant__ LnParams p) {
    __shared__ float slots[2][kWide / 32];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.x_s;
    float v[1] = {0.f};
    for (int c = threadIdx.x; c < p.dim; c += kWide) v[0] += to_f(x[c]);
    row_sum<kWide>(v, slots[0]);
    const float mean = v[0] / (float)p.dim;    // a division: exact for a constant row's exact sum
    v[0] = 0.f;
    for (int c = threadIdx.x; c < p.dim; c += kWide) {
        const float d = to_f(x[c]) - mean;
        v[0] = fmaf(d, d, v[0]);
    }
    row_sum<kWide>(v, slots[1]);
    const float rstd = rsqrtf(fmaf(v[0], p.inv_dim, p.eps));
    if (threadIdx.x == 0 && p.mean) {
        p.mean[row] = mean;
        p.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(p.y) + row * p.y_s;
    for (int c = threadIdx.x; c < p.dim; c += kWide) {
        const float h = (to_f(x[c]) - mean) * rstd;
        y[c] = from_f<T>((p.weight ? h * p.weight[c] : h) + (p.bias ? p.bias[c] : 0.f));
    }
}

template <typename T>
__global__ void __launch_bounds__(kWide) layer_norm_wide_dx_kernel(const __grid_constant__ LnParams p) {
    __shared__ float slots[2 * (kWide / 32)];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.x_s;
    const T* dy = static_cast<const T*>(p.dy) + row * p.dy_s;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float v[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < p.dim; c += kWide) {
        const float e = p.weight ? to_f(dy[c]) * p.weight[c] : to_f(dy[c]);
        v[0] += e;
        v[1] = fmaf(e, (to_f(x[c]) - mean) * rstd, v[1]);
    }
    row_sum<kWide>(v, slots);
    const float m0 = v[0] * p.inv_dim, m1 = v[1] * p.inv_dim;
    T* dx = static_cast<T*>(p.dx) + row * p.dx_s;
    for (int c = threadIdx.x; c < p.dim; c += kWide) {
        const float e = p.weight ? to_f(dy[c]) * p.weight[c] : to_f(dy[c]);
        dx[c] = from_f<T>(rstd * (e - m0 - (to_f(x[c]) - mean) * rstd * m1));
    }
}

// thread = column, blockIdx.y = slice of the rows
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_wide_dw_kernel(const __grid_constant__ LnParams p) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= p.dim) return;
    float dw = 0.f, db = 0.f;
    for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
        const float g = to_f(static_cast<const T*>(p.dy)[row * p.dy_s + c]);
        dw = fmaf(g, (to_f(static_cast<const T*>(p.x)[row * p.x_s + c]) - p.mean[row]) * p.rstd[row], dw);
        db += g;
    }
    float* out = p.part + (int64_t)blockIdx.y * 2 * p.dim + c;
    out[0] = dw;
    out[p.dim] = db;
}

// dweight / dbias = sums of the nparts partial rows: 32 columns x 32 threads per CTA, each
// thread every 32nd row, then the 32 sums in order
__global__ void __launch_bounds__(1024) layer_norm_dw_kernel(const float* part, int nparts, int dim, float* dweight,
                                                             float* dbias) {
    __shared__ float s[32][33];
    const int lane = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float* out = blockIdx.y ? dbias : dweight;
    if (!out) return;
    float sum = 0.f;
    if (c < dim)
#pragma unroll 4
        for (int i = y; i < nparts; i += 32) sum += part[((int64_t)i * 2 + blockIdx.y) * dim + c];
    s[y][lane] = sum;
    __syncthreads();
    // warp y adds up column y
    sum = s[lane][y];
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    if (lane == 0 && blockIdx.x * 32 + y < dim) out[blockIdx.x * 32 + y] = sum;
}

// CTAs of the backward: as many as fit on the SMs of the current device at once.  The first call on a
// device also lets the kernel have its shared memory there.
constexpr int kDevices = 64;
template <typename K>
cudaError_t resident_ctas(K kernel, int threads, int bytes, std::atomic<int> (&known)[kDevices], int* ctas) {
    int dev = 0, sms = 0, occ = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < kDevices && (*ctas = known[dev].load(std::memory_order_acquire)) != 0) return cudaSuccess;
    if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) != cudaSuccess ||
        (e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess ||
        (e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kernel, threads, bytes)) != cudaSuccess)
        return e;
    *ctas = sms * (occ < 1 ? 1 : occ);
    if (dev < kDevices) known[dev].store(*ctas, std::memory_order_release);
    return cudaSuccess;
}

template <typename T, int VT, int E, int TPR>
cudaError_t launch_fwd(const LnParams& p, cudaStream_t stream) {
    constexpr int RPC = kRowsPerCta<TPR>;
    layer_norm_fwd_kernel<T, VT, E, TPR><<<(unsigned)((p.rows + RPC - 1) / RPC), TPR * RPC, 0, stream>>>(p);
    return cudaGetLastError();
}
template <typename T, int VT, int E, int TPR>
cudaError_t launch_bwd(LnParams& p, cudaStream_t stream) {
    constexpr int RPC = kRowsPerCta<TPR>, bytes = kBwdBytes<T, VT, E, TPR>;
    static std::atomic<int> known[kDevices];
    int resident = 0;
    cudaError_t e = resident_ctas(layer_norm_bwd_kernel<T, VT, E, TPR>, TPR * RPC, bytes, known, &resident);
    if (e != cudaSuccess) return e;
    if (p.nparts > resident) p.nparts = resident;
    // and no CTA without a row
    if (p.nparts > (p.rows + RPC - 1) / RPC) p.nparts = (int)((p.rows + RPC - 1) / RPC);
    layer_norm_bwd_kernel<T, VT, E, TPR><<<p.nparts, TPR * RPC, bytes, stream>>>(p);
    return cudaGetLastError();
}

// Forward: what a thread holds is what it has in flight, so a row gets as few threads as can hold it
// (32768 rows of 5120 bfloat16: 217 us with 512 threads of 16, 141 with 256 of 24; 700 float32: 32 with
// 128 of 8, 27 with 32 of 24).  Single elements cost more instructions than they fill the pipes
// with, and up to 4096 go to more threads (801 bfloat16: 60 us with 32 of 32, 40 with 128 of 8).
template <typename T, int VT>
cudaError_t dispatch_fwd(const LnParams& p, cudaStream_t stream) {
    if (p.dim <= 256) return launch_fwd<T, VT, 8, 32>(p, stream);
    if (p.dim <= 512) return launch_fwd<T, VT, 16, 32>(p, stream);
    if constexpr (VT == 1) {
        if (p.dim <= 1024) return launch_fwd<T, VT, 8, 128>(p, stream);
        if (p.dim <= 2048) return launch_fwd<T, VT, 8, 256>(p, stream);
        if (p.dim <= 256 * 12) return launch_fwd<T, VT, 12, 256>(p, stream);
        if (p.dim <= 256 * 16) return launch_fwd<T, VT, 16, 256>(p, stream);
    } else {
        if (p.dim <= 768) return launch_fwd<T, VT, 24, 32>(p, stream);
        if (p.dim <= 1024) return launch_fwd<T, VT, 32, 32>(p, stream);
        if (p.dim <= 64 * 24) return launch_fwd<T, VT, 24, 64>(p, stream);
        if (p.dim <= 64 * 32) return launch_fwd<T, VT, 32, 64>(p, stream);
        if (p.dim <= 128 * 24) return launch_fwd<T, VT, 24, 128>(p, stream);
        if (p.dim <= 128 * 32) return launch_fwd<T, VT, 32, 128>(p, stream);
    }
    if (p.dim <= 256 * 24) return launch_fwd<T, VT, 24, 256>(p, stream);
    return launch_fwd<T, VT, 32, 256>(p, stream);
}
// Backward: up to 32 elements per thread as vectors of 16 bytes of bfloat16, else 16: there are two sums
// per column as well.  What a row costs besides its elements favours few threads with many (2565
// float32: 263 us with 512 of 6, 235 with 256 of 12; 5120 bfloat16: 369 with 512 of 16, 236 with 256 of 24).
template <typename T, int VT>
cudaError_t dispatch_bwd(LnParams& p, cudaStream_t stream) {
    if (p.dim <= 256) return launch_bwd<T, VT, 8, 32>(p, stream);
    if (p.dim <= 512) return launch_bwd<T, VT, 16, 32>(p, stream);
    if constexpr (VT == 8) {
        if (p.dim <= 768) return launch_bwd<T, VT, 24, 32>(p, stream);
        if (p.dim <= 1024) return launch_bwd<T, VT, 16, 64>(p, stream);
        if (p.dim <= 2048) return launch_bwd<T, VT, 16, 128>(p, stream);
        if (p.dim <= 128 * 24) return launch_bwd<T, VT, 24, 128>(p, stream);
        if (p.dim <= 4096) return launch_bwd<T, VT, 32, 128>(p, stream);
        if (p.dim <= 256 * 24) return launch_bwd<T, VT, 24, 256>(p, stream);
        return launch_bwd<T, VT, 32, 256>(p, stream);
    } else {
        if (p.dim <= 1024) return launch_bwd<T, VT, 16, 64>(p, stream);
        if (p.dim <= 2048) return launch_bwd<T, VT, 16, 128>(p, stream);
        if (p.dim <= 256 * 12) return launch_bwd<T, VT, 12, 256>(p, stream);
        if (p.dim <= 4096) return launch_bwd<T, VT, VT == 4 ? 8 : 16, VT == 4 ? 512 : 256>(p, stream);
        return launch_bwd<T, VT, 16, 512>(p, stream);
    }
}
template <typename T, int VT>
cudaError_t dispatch(LnParams& p, int backward, cudaStream_t stream) {
    return backward ? dispatch_bwd<T, VT>(p, stream) : dispatch_fwd<T, VT>(p, stream);
}

template <typename T>
cudaError_t dispatch_wide(const LnParams& p, int backward, cudaStream_t stream) {
    if (!backward) {
        layer_norm_wide_fwd_kernel<T><<<(unsigned)p.rows, kWide, 0, stream>>>(p);
    } else {
        layer_norm_wide_dx_kernel<T><<<(unsigned)p.rows, kWide, 0, stream>>>(p);
        if (p.dweight || p.dbias)
            layer_norm_wide_dw_kernel<T><<<dim3((p.dim + 255) / 256, p.nparts), 256, 0, stream>>>(p);
    }
    return cudaGetLastError();
}

}  // namespace

// Partial rows of dw and db there is room for: one per CTA of the backward, at most four CTAs per SM, or eight
// of those with 64 threads (32768 rows of 801 bfloat16: 80 and 53 us); for wide rows 64 slices of the rows.
// Which kernel runs goes by the alignment too, so the launch may take fewer: bfloat16 vectors of 513 to
// 768 have four rows to a CTA.
int layer_norm_parts(int64_t rows, int dim, int sms) {
    if (dim > kLnMaxDim) return (int)(rows < 64 ? rows : 64);
    const int rpc = dim <= 512 ? 4 : 1;
    const int64_t ctas = (rows + rpc - 1) / rpc, most = (int64_t)sms * (dim <= 1024 ? 8 : 4);
    return (int)(ctas < most ? ctas : most);
}

cudaError_t launch_layer_norm(const LnParams& params, int is_bf16, int vec, int backward, cudaStream_t stream) {
    LnParams p = params;
    cudaError_t e;
    if (p.dim > kLnMaxDim) {
        e = is_bf16 ? dispatch_wide<__nv_bfloat16>(p, backward, stream) : dispatch_wide<float>(p, backward, stream);
    } else if (is_bf16) {
        e = vec == 2 ? dispatch<__nv_bfloat16, 8>(p, backward, stream)
            : vec == 1 ? dispatch<__nv_bfloat16, 2>(p, backward, stream) : dispatch<__nv_bfloat16, 1>(p, backward, stream);
    } else {
        e = vec == 2 ? dispatch<float, 4>(p, backward, stream) : dispatch<float, 1>(p, backward, stream);
    }
    if (e != cudaSuccess || !backward || (!p.dweight && !p.dbias)) return e;
    layer_norm_dw_kernel<<<dim3((p.dim + 31) / 32, 2), 1024, 0, stream>>>(p.part, p.nparts, p.dim, p.dweight, p.dbias);
    return cudaGetLastError();
}

}  // namespace ssm
