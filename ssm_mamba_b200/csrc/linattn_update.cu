// One decode step of linear attention with a decay for each head:
//     S = w S + k v^T (in place),   out = scale q^T S,   w = exp(log_decay[h])
// per (batch row, head).  Bound by HBM: the float32 state is read and written once, everything
// else is three short rows.  A CTA of 8 warps owns up to 64 columns of one (batch row, head): its part of
// a row of S is one coalesced run of float4 over LPR lanes, a warp takes 32 / LPR rows at a time and issues the
// loads of all its rows before it uses any; the column sums of q^T S are joined over the warps
// through shared memory in a fixed order.  64 x 40 heads of 128 x 128 take 61 us (5.6 TB/s, half of
// it writes).  A state whose rows do not start on 16 bytes goes element by element: 104 us (3.2 TB/s).
#include "common.cuh"
#include "linattn.h"

namespace ssm {

namespace {

constexpr int kUpdWarps = 8;

template <typename T, int VT, int LPR>
__global__ void __launch_bounds__(kUpdWarps * 32) linattn_update_kernel(const __grid_constant__ LaUpdParams p) {
    constexpr int RPW = 32 / LPR, STEP = kUpdWarps * RPW, IT = 128 / STEP;
    __shared__ float part[STEP][LPR * VT];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = warp * RPW + lane / LPR;
    const int col = blockIdx.y * (LPR * VT) + (lane % LPR) * VT;
    const int b = blockIdx.x / p.heads, h = blockIdx.x - b * p.heads;
    const bool on = col < p.dv;                  // VT divides dv, or is 1
    float* st = p.state + b * p.st_sb + h * p.st_sh + col;
    // the previous kernel in the stream may still run: nothing it wrote is read before this
    griddep_wait();
    float s[IT][VT];
#pragma unroll
    for (int i = 0; i < IT; i++) {
        const int r = sub + i * STEP;
        if (on && r < p.dk) {
            if constexpr (VT == 4) {
                const float4 x = *reinterpret_cast<const float4*>(st + r * p.st_sk);
                s[i][0] = x.x; s[i][1] = x.y; s[i][2] = x.z; s[i][3] = x.w;
            } else {
                s[i][0] = st[r * p.st_sk];
            }
        }
    }
    const T* q = static_cast<const T*>(p.q) + b * p.q_sb + (h / p.q_share) * p.q_sh;
    const T* k = static_cast<const T*>(p.k) + b * p.k_sb + (h / p.k_share) * p.k_sh;
    const T* v = static_cast<const T*>(p.v) + b * p.v_sb + (h / p.v_share) * p.v_sh + col;
    const float w = exp2f(la_log2_decay(p.log_decay[h]));
    float vv[VT], acc[VT];
#pragma unroll
    for (int j = 0; j < VT; j++) {
        vv[j] = on ? to_f(v[j]) : 0.f;
        acc[j] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < IT; i++) {
        const int r = sub + i * STEP;
        if (!on || r >= p.dk) continue;
        const float kr = to_f(k[r]), qr = to_f(q[r]);
#pragma unroll
        for (int j = 0; j < VT; j++) {
            s[i][j] = fmaf(w, s[i][j], kr * vv[j]);
            acc[j] = fmaf(qr, s[i][j], acc[j]);
        }
        if constexpr (VT == 4) *reinterpret_cast<float4*>(st + r * p.st_sk) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
        else st[r * p.st_sk] = s[i][0];
    }
    griddep_launch_dependents();
#pragma unroll
    for (int j = 0; j < VT; j++) part[sub][(lane % LPR) * VT + j] = acc[j];
    __syncthreads();
    for (int c = threadIdx.x; c < LPR * VT; c += kUpdWarps * 32) {
        const int oc = blockIdx.y * (LPR * VT) + c;
        if (oc >= p.dv) break;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < STEP; i++) sum += part[i][c];
        static_cast<T*>(p.out)[b * p.o_sb + h * p.o_sh + oc] = from_f<T>(p.scale * sum);
    }
}

template <typename T, int VT, int LPR>
cudaError_t launch_update(const LaUpdParams& p, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.batch * p.heads), (unsigned)((p.dv + LPR * VT - 1) / (LPR * VT)));
    cfg.blockDim = dim3(kUpdWarps * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, linattn_update_kernel<T, VT, LPR>, p);
}

template <typename T>
cudaError_t dispatch_update(const LaUpdParams& p, int vec, cudaStream_t stream) {
    if (!vec) return launch_update<T, 1, 32>(p, stream);
    if (p.dv <= 16) return launch_update<T, 4, 4>(p, stream);
    if (p.dv <= 32) return launch_update<T, 4, 8>(p, stream);
    // 64 columns per CTA: 4 CTAs of 64 registers share an SM, and their loads and stores overlap (64 x 40 heads of
    // 128 x 128: 66 us with 128 columns, 61 with 64, 62 with 32)
    return launch_update<T, 4, 16>(p, stream);
}

}  // namespace

// vec: dv a multiple of 4 and every state row 16-byte aligned
cudaError_t launch_linattn_update(const LaUpdParams& p, int is_bf16, int vec, cudaStream_t stream) {
    return is_bf16 ? dispatch_update<__nv_bfloat16>(p, vec, stream) : dispatch_update<float>(p, vec, stream);
}

}  // namespace ssm
