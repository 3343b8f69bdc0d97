// Linear attention with a decay for each head on the FP32 pipe (every stream type, any sizes,
// strides and head counts; the recurrence and its four uses are in linattn.h).
//
// Chunked form: a CTA owns one (batch row, head, segment) and a tile of 64 columns of c, and
// walks the segment in chunks of 64 tokens.  The state tile (db x 64) stays in registers, with
// a copy in shared memory for the product with a.  Per chunk, all in float32:
//     P   = (A B^T) o W              64 x 64, W the decays of the causal triangle
//     out = alpha P C + beta diag(w^.) A S
//     S   = w^n S + sigma (diag(w^.) B)^T C
// 256 threads as a 16 x 16 grid, each with a 4 x 4 tile of P and out and a (db / 16) x 4 tile
// of S; the operands come from shared memory as 16-byte loads.  Splitting c (not b) keeps the
// sum over b inside the CTA; the 64 x 64 scores are recomputed by each column tile.
//
// Few (batch, head) pairs leave SMs idle, so a long row is cut into segments: the STATE pass
// leaves each segment's state from a zero start, and the main pass's CTAs fold the states of
// the segments before theirs in order (the decay across n tokens is one factor w^n).
#include "common.cuh"
#include "linattn.h"

namespace ssm {

namespace {

constexpr int kC = 64;         // tokens per chunk
constexpr int kDc = 64;        // columns of c per CTA
constexpr int kThreads = 256;

template <int DB>
struct SimtSmem {
    static constexpr int LDA = DB + 4;    // row strides: 16 bytes past a multiple of 128
    static constexpr int LDC = kDc + 4;
    float a[kC * LDA], b[kC * LDA], c[kC * LDC], s[DB * LDC], p[kC * LDC];
    float w[kC + 1];                      // w^0 .. w^64
};

// rows [0, n) x channels [0, d) of a chunk into float32 rows of stride LD, zeros up to (kC, W)
template <typename T, int W, int LD>
__device__ __forceinline__ void load_tile(float* dst, const LaTensor& t, int b, int h, int64_t tok, int n, int col0,
                                          int d) {
    const T* base = static_cast<const T*>(t.p) + b * t.sb + (int64_t)(h / t.share) * t.sh + tok * t.st + col0;
    constexpr int V = 16 / sizeof(T);
    if (t.vec) {
        for (int i = threadIdx.x; i < kC * (W / V); i += kThreads) {
            const int r = i / (W / V), c = (i - r * (W / V)) * V;
            float v[V];
            if (r < n && c + V <= d) {
                const uint4 raw = *reinterpret_cast<const uint4*>(base + r * t.st + c);
                const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
                for (int j = 0; j < V; j++) v[j] = to_f(e[j]);
            } else {
#pragma unroll
                for (int j = 0; j < V; j++) v[j] = (r < n && c + j < d) ? to_f(base[r * t.st + c + j]) : 0.f;
            }
#pragma unroll
            for (int j = 0; j < V; j++) dst[r * LD + c + j] = v[j];
        }
    } else {
        for (int i = threadIdx.x; i < kC * W; i += kThreads) {
            const int r = i / W, c = i - r * W;
            dst[r * LD + c] = (r < n && c < d) ? to_f(base[r * t.st + c]) : 0.f;
        }
    }
}

template <typename T, int DB, bool STATE>
__global__ void __launch_bounds__(kThreads) linattn_simt_kernel(const __grid_constant__ LaParams p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    using Smem = SimtSmem<DB>;
    constexpr int LDA = Smem::LDA, LDC = Smem::LDC, RS = DB / 16;
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    const LaRole& r = p.role[blockIdx.z];
    const int col0 = blockIdx.y * kDc;
    if (col0 >= r.dc) return;
    // one CTA per (segment, batch row, head); heads vary fastest
    int64_t id = blockIdx.x;
    const int h = (int)(id % p.heads);
    id /= p.heads;
    const int b = (int)(id % p.batch);
    const int slot = (int)(id / p.batch);
    const int seg = r.reverse ? p.nseg - 1 - slot : slot;
    const int64_t bh = (int64_t)b * p.heads + h;
    const int cols = min(kDc, r.dc - col0);
    const int row_len = la_row_length(p, b);
    const int ntok = la_segment_tokens(p, row_len, seg);
    const int64_t tok0 = (int64_t)seg * p.seglen;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const float g2 = la_log2_decay(p.log_decay[h]);

    for (int i = tid; i <= kC; i += kThreads) sm.w[i] = exp2f(g2 * (float)i);

    // state tile: rows ty * RS .. + RS, columns tx * 4 .. + 4
    float s[RS][4];
    auto valid = [&](int i, int j) { return ty * RS + i < r.db && tx * 4 + j < cols; };
#pragma unroll
    for (int i = 0; i < RS; i++)
#pragma unroll
        for (int j = 0; j < 4; j++)
            s[i][j] = (!STATE && r.state0 && valid(i, j))
                          ? r.state0[bh * r.db * r.dc + (int64_t)(ty * RS + i) * r.s_i + (col0 + tx * 4 + j) * r.s_j]
                          : 0.f;
    if (!STATE) {
        for (int q = 0; q < slot; q++) {
            const int sg = r.reverse ? p.nseg - 1 - q : q;
            const float f = exp2f(g2 * (float)la_segment_tokens(p, row_len, sg));
            const float* e = r.seg + (bh * p.nseg + sg) * r.db * r.dc;
#pragma unroll
            for (int i = 0; i < RS; i++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (valid(i, j)) s[i][j] = fmaf(f, s[i][j], e[(ty * RS + i) * r.dc + col0 + tx * 4 + j]);
        }
    }

    const int nchunk = (ntok + kC - 1) / kC;
    for (int it = 0; it < nchunk; it++) {
        const int ch = r.reverse ? nchunk - 1 - it : it;
        const int64_t t0 = tok0 + (int64_t)ch * kC;
        const int n = min(kC, ntok - ch * kC);
        __syncthreads();                       // the previous chunk's readers are done
        if (!STATE) load_tile<T, DB, LDA>(sm.a, r.a, b, h, t0, n, 0, r.db);
        load_tile<T, DB, LDA>(sm.b, r.b, b, h, t0, n, 0, r.db);
        load_tile<T, kDc, LDC>(sm.c, r.c, b, h, t0, n, col0, cols);
        if (!STATE) {
#pragma unroll
            for (int i = 0; i < RS; i++)
                *reinterpret_cast<float4*>(&sm.s[(ty * RS + i) * LDC + tx * 4]) =
                    make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
        }
        __syncthreads();
        if (!STATE) {
            // scores: rows ty * 4.., columns tx + 16 j (so a half warp's rows of b are spread
            // over the banks)
            float acc[4][4] = {};
#pragma unroll 2
            for (int k = 0; k < DB; k += 4) {
                float4 av[4], bv[4];
#pragma unroll
                for (int i = 0; i < 4; i++) av[i] = lds128(&sm.a[(ty * 4 + i) * LDA + k]);
#pragma unroll
                for (int j = 0; j < 4; j++) bv[j] = lds128(&sm.b[(tx + 16 * j) * LDA + k]);
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        acc[i][j] = fmaf(av[i].x, bv[j].x, acc[i][j]);
                        acc[i][j] = fmaf(av[i].y, bv[j].y, acc[i][j]);
                        acc[i][j] = fmaf(av[i].z, bv[j].z, acc[i][j]);
                        acc[i][j] = fmaf(av[i].w, bv[j].w, acc[i][j]);
                    }
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int row = ty * 4 + i, col = tx + 16 * j;
                    const int dist = r.reverse ? col - row : row - col;
                    sm.p[row * LDC + col] = dist >= 0 ? r.alpha * acc[i][j] * sm.w[dist] : 0.f;
                }
            // state part of the output
            float o[4][4] = {};
#pragma unroll 2
            for (int k = 0; k < DB; k += 4) {
                float4 av[4], sv[4];
#pragma unroll
                for (int i = 0; i < 4; i++) av[i] = lds128(&sm.a[(ty * 4 + i) * LDA + k]);
#pragma unroll
                for (int j = 0; j < 4; j++) sv[j] = lds128(&sm.s[(k + j) * LDC + tx * 4]);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float a4[4] = {av[i].x, av[i].y, av[i].z, av[i].w};
#pragma unroll
                    for (int kk = 0; kk < 4; kk++) {
                        o[i][0] = fmaf(a4[kk], sv[kk].x, o[i][0]);
                        o[i][1] = fmaf(a4[kk], sv[kk].y, o[i][1]);
                        o[i][2] = fmaf(a4[kk], sv[kk].z, o[i][2]);
                        o[i][3] = fmaf(a4[kk], sv[kk].w, o[i][3]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = ty * 4 + i;
                const int pos = r.reverse ? max(n - 1 - row, 0) : row + 1;
                const float f = r.beta * sm.w[pos];
#pragma unroll
                for (int j = 0; j < 4; j++) o[i][j] *= f;
            }
            __syncthreads();                   // p is complete
            // causal part: the warp's rows are ty0 * 4 .. + 8 with ty0 = 2 * warp
            const int warp = tid >> 5;
            const int k_lo = r.reverse ? warp * 8 : 0, k_hi = r.reverse ? kC : warp * 8 + 8;
            for (int k = k_lo; k < k_hi; k += 4) {
                float4 pv[4], cv[4];
#pragma unroll
                for (int i = 0; i < 4; i++) pv[i] = lds128(&sm.p[(ty * 4 + i) * LDC + k]);
#pragma unroll
                for (int j = 0; j < 4; j++) cv[j] = lds128(&sm.c[(k + j) * LDC + tx * 4]);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p4[4] = {pv[i].x, pv[i].y, pv[i].z, pv[i].w};
#pragma unroll
                    for (int kk = 0; kk < 4; kk++) {
                        o[i][0] = fmaf(p4[kk], cv[kk].x, o[i][0]);
                        o[i][1] = fmaf(p4[kk], cv[kk].y, o[i][1]);
                        o[i][2] = fmaf(p4[kk], cv[kk].z, o[i][2]);
                        o[i][3] = fmaf(p4[kk], cv[kk].w, o[i][3]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = ty * 4 + i;
                if (row >= n) continue;
                const int64_t at = b * r.o_sb + (t0 + row) * r.o_st + h * r.o_sh + col0 + tx * 4;
                if (r.out_f32) {
                    float* op = static_cast<float*>(r.out) + at;
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (tx * 4 + j < cols) op[j] = o[i][j];
                } else {
                    T* op = static_cast<T*>(r.out) + at;
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (tx * 4 + j < cols) op[j] = from_f<T>(o[i][j]);
                }
            }
        }
        // state update
        const float fn = sm.w[n];
#pragma unroll
        for (int i = 0; i < RS; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) s[i][j] *= fn;
#pragma unroll 4
        for (int k = 0; k < n; k++) {
            const float f = r.sigma * sm.w[r.reverse ? k + 1 : n - 1 - k];
            float4 cv = lds128(&sm.c[k * LDC + tx * 4]);
            cv.x *= f; cv.y *= f; cv.z *= f; cv.w *= f;
#pragma unroll
            for (int i4 = 0; i4 < RS; i4 += 4) {
                const float4 bv = lds128(&sm.b[k * LDA + ty * RS + i4]);
                const float b4[4] = {bv.x, bv.y, bv.z, bv.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    s[i4 + i][0] = fmaf(b4[i], cv.x, s[i4 + i][0]);
                    s[i4 + i][1] = fmaf(b4[i], cv.y, s[i4 + i][1]);
                    s[i4 + i][2] = fmaf(b4[i], cv.z, s[i4 + i][2]);
                    s[i4 + i][3] = fmaf(b4[i], cv.w, s[i4 + i][3]);
                }
            }
        }
    }

    if (STATE) {
        float* e = r.seg + (bh * p.nseg + seg) * r.db * r.dc;
#pragma unroll
        for (int i = 0; i < RS; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (valid(i, j)) e[(ty * RS + i) * r.dc + col0 + tx * 4 + j] = s[i][j];
        return;
    }
    if (slot == p.nseg - 1 && r.state_out) {
#pragma unroll
        for (int i = 0; i < RS; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (valid(i, j))
                    r.state_out[bh * r.db * r.dc + (int64_t)(ty * RS + i) * r.s_i + (col0 + tx * 4 + j) * r.s_j] =
                        s[i][j];
    }
    // tokens past the row's length
    const int seg_end = (int)min((int64_t)p.seglen, (int64_t)p.seqlen - tok0);
    for (int i = tid; i < (seg_end - ntok) * kDc; i += kThreads) {
        const int t = ntok + i / kDc, c = i % kDc;
        if (c >= cols) continue;
        const int64_t at = b * r.o_sb + (tok0 + t) * r.o_st + h * r.o_sh + col0 + c;
        if (r.out_f32) static_cast<float*>(r.out)[at] = 0.f;
        else static_cast<T*>(r.out)[at] = from_f<T>(0.f);
    }
}

template <typename T, int DB>
cudaError_t launch_simt(const LaParams& p, int max_dc, cudaStream_t stream) {
    constexpr int bytes = (int)sizeof(SimtSmem<DB>);
    auto main_k = linattn_simt_kernel<T, DB, false>;
    auto state_k = linattn_simt_kernel<T, DB, true>;
    cudaError_t e = cudaFuncSetAttribute(main_k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(state_k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    const dim3 tiles(1, (max_dc + kDc - 1) / kDc, p.nroles);
    if (p.nseg > 1) {
        // the last segment (in walking order) needs no state of its own
        const dim3 g((unsigned)((int64_t)p.batch * p.heads * (p.nseg - 1)), tiles.y, tiles.z);
        state_k<<<g, kThreads, bytes, stream>>>(p);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
    const dim3 g((unsigned)((int64_t)p.batch * p.heads * p.nseg), tiles.y, tiles.z);
    main_k<<<g, kThreads, bytes, stream>>>(p);
    return cudaGetLastError();
}

// A CTA does kGroupTokens tokens; V channels (V divides d) per thread and step.
constexpr int kGroupTokens = 16;
template <typename T, int V>
__global__ void __launch_bounds__(256) linattn_group_kernel(const __grid_constant__ LaGroupParams p) {
    const int groups = p.heads / p.share, dv = p.d / V, per = groups * dv;
    const int64_t tokens = (int64_t)p.batch * p.seqlen, first = (int64_t)blockIdx.x * kGroupTokens;
    const int64_t b0 = first / p.seqlen;
    const int t0 = (int)(first - b0 * p.seqlen);
    const int n = (int)(tokens - first < kGroupTokens ? tokens - first : kGroupTokens);
    for (int i = threadIdx.x; i < n * per; i += 256) {
        const int tl = i / per, pos = i - tl * per, g = pos / dv, c = (pos - g * dv) * V;
        const float* s = p.src + ((first + tl) * p.heads + (int64_t)g * p.share) * p.d + c;
        float sum[V] = {};
        for (int k = 0; k < p.share; k++, s += p.d) {
            if constexpr (V == 4) {
                const float4 x = *reinterpret_cast<const float4*>(s);
                sum[0] += x.x; sum[1] += x.y; sum[2] += x.z; sum[3] += x.w;
            } else {
                sum[0] += s[0];
            }
        }
        int64_t b = b0;
        int t = t0 + tl;
        while (t >= p.seqlen) {
            t -= p.seqlen;
            b++;
        }
        T* out = static_cast<T*>(p.out) + b * p.o_sb + t * p.o_st + g * p.o_sh + c;
#pragma unroll
        for (int e = 0; e < V; e++) out[e] = from_f<T>(sum[e]);
    }
}

template <typename T>
cudaError_t launch_group(const LaGroupParams& p, cudaStream_t stream) {
    const int64_t tokens = (int64_t)p.batch * p.seqlen;
    const unsigned grid = (unsigned)((tokens + kGroupTokens - 1) / kGroupTokens);
    if (p.d % 4 == 0) linattn_group_kernel<T, 4><<<grid, 256, 0, stream>>>(p);
    else linattn_group_kernel<T, 1><<<grid, 256, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_linattn_simt(const LaParams& p, int is_bf16, cudaStream_t stream) {
    int db = 0, dc = 0;
    for (int i = 0; i < p.nroles; i++) {
        db = p.role[i].db > db ? p.role[i].db : db;
        dc = p.role[i].dc > dc ? p.role[i].dc : dc;
    }
    if (is_bf16) return db <= 64 ? launch_simt<__nv_bfloat16, 64>(p, dc, stream) : launch_simt<__nv_bfloat16, 128>(p, dc, stream);
    return db <= 64 ? launch_simt<float, 64>(p, dc, stream) : launch_simt<float, 128>(p, dc, stream);
}

cudaError_t launch_linattn_group(const LaGroupParams& p, int is_bf16, cudaStream_t stream) {
    return is_bf16 ? launch_group<__nv_bfloat16>(p, stream) : launch_group<float>(p, stream);
}

}  // namespace ssm
