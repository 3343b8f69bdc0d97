// Linear attention with a decay for each head on the FP32 pipe: float32 streams of any sizes,
// strides and head counts (the recurrence and its four uses are in linattn.h).
//
// A CTA owns one (batch row, head, segment) and a tile of DC columns of c, and walks the segment in
// chunks of 64 tokens.  The state tile (db x DC) stays in registers, with a copy in shared memory
// for the product with a.  Per chunk, all in float32:
//     P   = (A B^T) o W              64 x 64, W the decays of the causal triangle
//     out = alpha P C + beta diag(w^.) A S
//     S   = w^n S + sigma (diag(w^.) B)^T C
// 256 threads as a 16 x 16 grid, each with a 4 x 4 tile of P, a 4 x DC/16 tile of out and a
// DB/16 x DC/16 tile of S; the operands come from shared memory as 16-byte loads.  Splitting c (not
// b) keeps the sum over b inside the CTA; the scores are recomputed by each column tile.
//
// A chunk alone is a chain of loads, products and barriers that leaves the pipe idle, so a row is
// cut into segments until there are several CTAs per SM: a first pass leaves each segment's state
// from a zero start, a scan turns those into the states that the segments start from, and the
// main pass runs all segments at once.  S is computed twice, a quarter more products; at
// 2 x 1024 tokens of 24 heads of 64 forward and backward took 395 us with two segments.
#include "common.cuh"
#include "linattn.h"

namespace ssm {

namespace {

constexpr int kC = 64;         // tokens per chunk
constexpr int kThreads = 256;

template <int DB, int DC>
struct SimtSmem {
    static constexpr int LDA = DB + 4;    // row strides: 16 bytes past a multiple of 128
    static constexpr int LDC = DC + 4;
    static constexpr int LDP = kC + 4;
    float b[kC * LDA], c[kC * LDC], s[DB * LDC];
    float a[kC * (LDA > LDP ? LDA : LDP)];   // a, then P
    float w[kC + 1];                      // w^0 .. w^64
};

// rows [0, n) x channels [0, d) of a chunk into rows of stride LD, zeros up to (kC, W)
template <int W, int LD>
__device__ __forceinline__ void load_tile(float* dst, const LaTensor& t, int b, int h, int64_t tok, int n, int col0,
                                          int d) {
    const float* base = static_cast<const float*>(t.p) + b * t.sb + (int64_t)(h / t.share) * t.sh + tok * t.st + col0;
    for (int i = threadIdx.x; i < kC * (W / 4); i += kThreads) {
        const int r = i / (W / 4), c = (i - r * (W / 4)) * 4;
        const float* p = base + r * t.st + c;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < n) {
            if (t.vec && c + 4 <= d) {
                v = *reinterpret_cast<const float4*>(p);
            } else {
                if (c < d) v.x = p[0];
                if (c + 1 < d) v.y = p[1];
                if (c + 2 < d) v.z = p[2];
                if (c + 3 < d) v.w = p[3];
            }
        }
        *reinterpret_cast<float4*>(dst + r * LD + c) = v;
    }
}

template <int N>
__device__ __forceinline__ void load_row(const float* p, float (&v)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 x = lds128(p + i);
            v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w;
        }
    } else {
        const float2 x = *reinterpret_cast<const float2*>(p);
        v[0] = x.x; v[1] = x.y;
    }
}
template <int N>
__device__ __forceinline__ void store_row(float* p, const float (&v)[N]) {
    static_assert(N == 2 || N == 4);
    if constexpr (N == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
}

template <int DB, int DC, bool STATE>
__global__ void __launch_bounds__(kThreads) linattn_simt_kernel(const __grid_constant__ LaParams p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    using Smem = SimtSmem<DB, DC>;
    constexpr int LDA = Smem::LDA, LDC = Smem::LDC, LDP = Smem::LDP, RS = DB / 16, NC = DC / 16;
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    const LaRole& r = p.role[blockIdx.z];
    const int col0 = blockIdx.y * DC;
    if (col0 >= r.dc) return;
    // one CTA per (segment, batch row, head); heads vary fastest
    int64_t id = blockIdx.x;
    const int h = (int)(id % p.heads);
    id /= p.heads;
    const int b = (int)(id % p.batch);
    const int slot = (int)(id / p.batch);
    const int seg = r.reverse ? p.nseg - 1 - slot : slot;
    const int64_t bh = (int64_t)b * p.heads + h;
    const int cols = min(DC, r.dc - col0);
    const int row_len = la_row_length(p, b);
    const int ntok = la_segment_tokens(p, row_len, seg);
    const int64_t tok0 = (int64_t)seg * p.seglen;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const float g2 = la_log2_decay(p.log_decay[h]);

    for (int i = tid; i <= kC; i += kThreads) sm.w[i] = exp2f(g2 * (float)i);

    // state tile: rows ty * RS .. + RS, columns tx * NC .. + NC; from the segment's start state, which the
    // scan has left in its place, or from the initial state
    float s[RS][NC];
    auto valid = [&](int i, int j) { return ty * RS + i < r.db && tx * NC + j < cols; };
    const float* start = !STATE && p.nseg > 1 ? r.seg + (bh * p.nseg + seg) * r.db * r.dc
                         : !STATE && r.state0 ? r.state0 + bh * r.db * r.dc : nullptr;
    const int64_t s_i = p.nseg > 1 ? r.dc : r.s_i, s_j = p.nseg > 1 ? 1 : r.s_j;
#pragma unroll
    for (int i = 0; i < RS; i++)
#pragma unroll
        for (int j = 0; j < NC; j++)
            s[i][j] = start && valid(i, j) ? start[(ty * RS + i) * s_i + (col0 + tx * NC + j) * s_j] : 0.f;

    const int nchunk = (ntok + kC - 1) / kC;
    for (int it = 0; it < nchunk; it++) {
        const int ch = r.reverse ? nchunk - 1 - it : it;
        const int64_t t0 = tok0 + (int64_t)ch * kC;
        const int n = min(kC, ntok - ch * kC);
        __syncthreads();                       // the previous chunk's readers are done
        if (!STATE) load_tile<DB, LDA>(sm.a, r.a, b, h, t0, n, 0, r.db);
        load_tile<DB, LDA>(sm.b, r.b, b, h, t0, n, 0, r.db);
        load_tile<DC, LDC>(sm.c, r.c, b, h, t0, n, col0, cols);
        if (!STATE) {
#pragma unroll
            for (int i = 0; i < RS; i++)
                store_row<NC>(&sm.s[(ty * RS + i) * LDC + tx * NC], s[i]);
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
            // state part of the output
            float o[4][NC] = {};
#pragma unroll 2
            for (int k = 0; k < DB; k += 4) {
                float4 av[4];
                float sv[4][NC];
#pragma unroll
                for (int i = 0; i < 4; i++) av[i] = lds128(&sm.a[(ty * 4 + i) * LDA + k]);
#pragma unroll
                for (int j = 0; j < 4; j++) load_row<NC>(&sm.s[(k + j) * LDC + tx * NC], sv[j]);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float a4[4] = {av[i].x, av[i].y, av[i].z, av[i].w};
#pragma unroll
                    for (int kk = 0; kk < 4; kk++)
#pragma unroll
                        for (int j = 0; j < NC; j++) o[i][j] = fmaf(a4[kk], sv[kk][j], o[i][j]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = ty * 4 + i;
                const int pos = r.reverse ? max(n - 1 - row, 0) : row + 1;
                const float f = r.beta * sm.w[pos];
#pragma unroll
                for (int j = 0; j < NC; j++) o[i][j] *= f;
            }
            __syncthreads();                   // a has been read: P goes over it
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int row = ty * 4 + i, col = tx + 16 * j;
                    const int dist = r.reverse ? col - row : row - col;
                    sm.a[row * LDP + col] = dist >= 0 ? r.alpha * acc[i][j] * sm.w[dist] : 0.f;
                }
            __syncthreads();                   // P is complete
            // causal part: the warp's rows are 8 * warp .. + 8
            const int warp = tid >> 5;
            const int k_lo = r.reverse ? warp * 8 : 0, k_hi = r.reverse ? kC : warp * 8 + 8;
            for (int k = k_lo; k < k_hi; k += 4) {
                float4 pv[4];
                float cv[4][NC];
#pragma unroll
                for (int i = 0; i < 4; i++) pv[i] = lds128(&sm.a[(ty * 4 + i) * LDP + k]);
#pragma unroll
                for (int j = 0; j < 4; j++) load_row<NC>(&sm.c[(k + j) * LDC + tx * NC], cv[j]);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p4[4] = {pv[i].x, pv[i].y, pv[i].z, pv[i].w};
#pragma unroll
                    for (int kk = 0; kk < 4; kk++)
#pragma unroll
                        for (int j = 0; j < NC; j++) o[i][j] = fmaf(p4[kk], cv[kk][j], o[i][j]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = ty * 4 + i;
                if (row >= n) continue;
                const int64_t at = b * r.o_sb + (t0 + row) * r.o_st + h * r.o_sh + col0 + tx * NC;
                float* op = static_cast<float*>(r.out) + at;
#pragma unroll
                for (int j = 0; j < NC; j++)
                    if (tx * NC + j < cols) op[j] = o[i][j];
            }
        }
        // state update
        const float fn = sm.w[n];
#pragma unroll
        for (int i = 0; i < RS; i++)
#pragma unroll
            for (int j = 0; j < NC; j++) s[i][j] *= fn;
#pragma unroll 4
        for (int k = 0; k < n; k++) {
            const float f = r.sigma * sm.w[r.reverse ? k + 1 : n - 1 - k];
            float cv[NC], bv[RS];
            load_row<NC>(&sm.c[k * LDC + tx * NC], cv);
            load_row<RS>(&sm.b[k * LDA + ty * RS], bv);
#pragma unroll
            for (int j = 0; j < NC; j++) cv[j] *= f;
#pragma unroll
            for (int i = 0; i < RS; i++)
#pragma unroll
                for (int j = 0; j < NC; j++) s[i][j] = fmaf(bv[i], cv[j], s[i][j]);
        }
    }

    if (STATE || (slot == p.nseg - 1 && r.state_out)) {
        float* dst = STATE ? r.seg + (bh * p.nseg + seg) * r.db * r.dc : r.state_out + bh * r.db * r.dc;
        const int64_t d_i = STATE ? r.dc : r.s_i, d_j = STATE ? 1 : r.s_j;
#pragma unroll
        for (int i = 0; i < RS; i++)
#pragma unroll
            for (int j = 0; j < NC; j++)
                if (valid(i, j)) dst[(ty * RS + i) * d_i + (col0 + tx * NC + j) * d_j] = s[i][j];
    }
    if (STATE) return;
    // tokens past the row's length
    const int seg_end = (int)min((int64_t)p.seglen, (int64_t)p.seqlen - tok0);
    for (int i = tid; i < (seg_end - ntok) * DC; i += kThreads) {
        const int t = ntok + i / DC, c = i % DC;
        if (c >= cols) continue;
        static_cast<float*>(r.out)[b * r.o_sb + (tok0 + t) * r.o_st + h * r.o_sh + col0 + c] = 0.f;
    }
}

// The segments' states from a zero start become the states they start from: thread = state element,
// the segments in the order of walking, eight loads ahead of the fold.
__global__ void __launch_bounds__(256) linattn_scan_kernel(const __grid_constant__ LaParams p) {
    const LaRole& r = p.role[blockIdx.z];
    const int e = blockIdx.y * 256 + threadIdx.x, size = r.db * r.dc;
    if (e >= size) return;
    const int64_t bh = blockIdx.x;
    const int b = (int)(bh / p.heads), h = (int)(bh - (int64_t)b * p.heads);
    const int row_len = la_row_length(p, b);
    const float g2 = la_log2_decay(p.log_decay[h]);
    float x = r.state0 ? r.state0[bh * size + (int64_t)(e / r.dc) * r.s_i + (e % r.dc) * r.s_j] : 0.f;
    float* seg = r.seg + bh * p.nseg * size + e;
    auto place = [&](int slot) { return r.reverse ? p.nseg - 1 - slot : slot; };
    for (int s0 = 0; s0 < p.nseg; s0 += 8) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = s0 + i < p.nseg - 1 ? seg[(int64_t)place(s0 + i) * size] : 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (s0 + i >= p.nseg) break;
            const int s = place(s0 + i);
            seg[(int64_t)s * size] = x;
            x = fmaf(exp2f(g2 * (float)la_segment_tokens(p, row_len, s)), x, v[i]);
        }
    }
}

}  // namespace

cudaError_t launch_linattn_scan(const LaParams& p, cudaStream_t stream) {
    const int size = p.role[0].db * p.role[0].dc;         // every role's states have dk x dv elements
    linattn_scan_kernel<<<dim3((unsigned)(p.batch * p.heads), (size + 255) / 256, p.nroles), 256, 0, stream>>>(p);
    return cudaGetLastError();
}

namespace {

template <int DB, int DC>
cudaError_t launch_simt(const LaParams& p, int max_dc, cudaStream_t stream) {
    constexpr int bytes = (int)sizeof(SimtSmem<DB, DC>);
    auto main_k = linattn_simt_kernel<DB, DC, false>;
    auto state_k = linattn_simt_kernel<DB, DC, true>;
    cudaError_t e = cudaFuncSetAttribute(main_k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(state_k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    const unsigned rows = (unsigned)(p.batch * p.heads), tiles = (max_dc + DC - 1) / DC;
    if (p.nseg > 1) {
        // the last segment (in walking order) feeds nobody
        state_k<<<dim3(rows * (p.nseg - 1), tiles, p.nroles), kThreads, bytes, stream>>>(p);
        if ((e = cudaGetLastError()) != cudaSuccess || (e = launch_linattn_scan(p, stream)) != cudaSuccess) return e;
    }
    main_k<<<dim3(rows * p.nseg, tiles, p.nroles), kThreads, bytes, stream>>>(p);
    return cudaGetLastError();
}

// bfloat16 (batch, token, head, channel) of any strides into rows of whole 16-byte pieces, which a TMA
// can fetch; thread = piece.  EVEN: rows start on 4 bytes and have an even number of channels.
template <bool EVEN>
__global__ void __launch_bounds__(256) linattn_pack_kernel(const __grid_constant__ LaPackParams p) {
    const int per = (p.d + 7) / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)p.seqlen * p.heads * per) return;
    const int64_t row = i / per;
    const int c = (int)(i - row * per) * 8, t = (int)(row / p.heads), h = (int)(row - (int64_t)t * p.heads);
    const int n = p.d - c < 8 ? p.d - c : 8;
    for (int64_t b = blockIdx.y; b < p.batch; b += gridDim.y) {
        const uint16_t* src = static_cast<const uint16_t*>(p.src) + b * p.sb + t * p.st + h * p.sh + c;
        uint32_t w[4] = {};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (EVEN) {
                if (2 * e < n) w[e] = reinterpret_cast<const uint32_t*>(src)[e];
            } else {
                if (2 * e < n) w[e] = src[2 * e];
                if (2 * e + 1 < n) w[e] |= (uint32_t)src[2 * e + 1] << 16;
            }
        }
        reinterpret_cast<uint4*>(p.dst)[b * p.seqlen * p.heads * per + i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
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

cudaError_t launch_linattn_simt(const LaParams& p, cudaStream_t stream) {
    int db = 0, dc = 0;
    for (int i = 0; i < p.nroles; i++) {
        db = p.role[i].db > db ? p.role[i].db : db;
        dc = p.role[i].dc > dc ? p.role[i].dc : dc;
    }
    if (db <= 32) return dc <= 32 ? launch_simt<32, 32>(p, dc, stream) : launch_simt<32, 64>(p, dc, stream);
    if (db <= 64) return dc <= 32 ? launch_simt<64, 32>(p, dc, stream) : launch_simt<64, 64>(p, dc, stream);
    return dc <= 32 ? launch_simt<128, 32>(p, dc, stream) : launch_simt<128, 64>(p, dc, stream);
}

cudaError_t launch_linattn_pack(const LaPackParams& p, int even, cudaStream_t stream) {
    const int64_t pieces = (int64_t)p.seqlen * p.heads * ((p.d + 7) / 8);
    const dim3 grid((unsigned)((pieces + 255) / 256), p.batch < 65535 ? p.batch : 65535);
    if (even) linattn_pack_kernel<true><<<grid, 256, 0, stream>>>(p);
    else linattn_pack_kernel<false><<<grid, 256, 0, stream>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_linattn_group(const LaGroupParams& p, int is_bf16, cudaStream_t stream) {
    return is_bf16 ? launch_group<__nv_bfloat16>(p, stream) : launch_group<float>(p, stream);
}

}  // namespace ssm
