// Linear attention with a decay for each head for float32 streams of any sizes, strides and head
// counts (the recurrence and its four uses are in linattn.h).
//
// A CTA owns one (batch row, head, segment) and a tile of DC columns of c, and walks the segment in
// chunks of 64 tokens.  The state tile (DB x DC) stays in registers, with a copy in shared memory
// for the product with a.  Per chunk:
//     P   = (A B^T) o W              64 x 64, W the decays of the causal triangle
//     out = alpha P C + beta diag(w^.) A S
//     S   = w^n S + sigma (diag(w^.) B)^T C
// The products run on mma.sync (m16n8k8, tf32) in three passes: every operand is split as
// x = hi + lo with hi rounded to tf32 (11 bits), and hi hi' + lo hi' + hi lo' misses x x' by about
// 2^-22.  On B200 that has 92 TFLOP/s of float32 products against 74 on the FMA pipe, and a sixth of its
// shared-memory traffic, which bounded a version on packed FMAs (67% of the wavefronts, 35% of
// the FMAs).  On tcgen05 both halves of a, b, c and S would have to be stored in shared memory: 224 KB at 128
// channels and 64 columns (a and b 64 KB each, c 32, S 64) of the 227 that a CTA has, without room for the next
// chunk; at 64 channels 128 KB would do, which is not built.  An infinity becomes a NaN when it is split.
//
// Measured: 2 x 1024 tokens of 24 heads of 64, forward and backward, 193 us (325 us on FMAs); 11 x 94
// tokens of 40 heads, 96 and 80 channels, forward, 113 us.  What bounds it is the latency of a
// chunk's steps with 8 to 14 warps on an SM: the tensor pipe is busy 20 to 40% of the time, issue 34 to 49%
// (two tiles' products interleaved by hand: 191 us and 115 us).
//
// Shared-memory rows are strided so that a fragment's 32 elements lie on different banks: 4 (mod
// 32) for operands read along their rows, 8 for operands read across them; b, which is read both
// ways, has 4 and two elements to some banks when read across.  The next chunk is copied meanwhile.
//
// A chunk alone is a chain of loads, products and barriers that leaves the pipe idle, so a row is
// cut into segments until there are two CTAs per SM: a first pass leaves each segment's state from a
// zero start, and the main pass runs all segments at once from the states that those add up to,
// folded by each CTA or, of many segments, scanned before.  S is computed twice, a quarter more
// products.
#include "common.cuh"
#include "linattn.h"

namespace ssm {

namespace {

constexpr int kC = 64;         // tokens per chunk
// Up to so many segments each CTA folds the states of those before its own; more are scanned (six and two
// segments of the training step above: 202 us scanned, 193 folded).
constexpr int kFold = 8;

// threads of a CTA: with 128 channels it has an SM to itself
template <int DB>
constexpr int kThreads = DB > 64 ? 512 : 256;

template <int DB, int DC>
struct F32Smem {
    static constexpr int LDB = DB + 4, LDN = DC + 8, LDP = kC + 4;
    float a[kC * LDB];
    float b[2][kC * LDB], c[2][kC * LDN];
    float s[DB * LDN > kC * LDP ? DB * LDN : kC * LDP];   // S, then P
    float w[kC + 1];                                      // w^0 .. w^64
};

// Starts the copy of rows [0, n) x channels [0, d) of a chunk to rows of stride LD, zeros up to (kC, W)
template <int W, int LD, int THREADS>
__device__ __forceinline__ void load_tile(float* dst, const LaTensor& t, int b, int h, int64_t tok, int n, int col0,
                                          int d) {
    const float* base = static_cast<const float*>(t.p) + b * t.sb + (int64_t)(h / t.share) * t.sh + tok * t.st + col0;
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst);
#pragma unroll 4
    for (int i = threadIdx.x; i < kC * (W / 4); i += THREADS) {
        const int r = i / (W / 4), c = (i - r * (W / 4)) * 4;
        const int left = r < n ? min(max(d - c, 0), 4) : 0;      // elements that exist
        const float* p = left ? base + r * t.st + c : base;
        const uint32_t q = to + (r * LD + c) * 4;
        if (t.vec) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(q), "l"(p), "r"(left * 4) : "memory");
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(q + 4 * e), "l"(e < left ? p + e : p),
                             "r"(e < left ? 4 : 0)
                             : "memory");
        }
    }
}

// x = hi + lo, hi a tf32 (rounded by integers: cvt.rna.tf32 made the training step below 239 instead of 221 us);
// the unit reads the leading 11 bits of lo
struct Split {
    uint32_t hi, lo;
};
__device__ __forceinline__ Split split(float x) {
    Split s;
    s.hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    s.lo = __float_as_uint(x - __uint_as_float(s.hi));
    return s;
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two tiles of 16 x 8, split: a(row 0..15, k 0..15) reads an element
struct Rows {
    Split f[2][4];
};
template <typename A>
__device__ __forceinline__ Rows rows(A a) {
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
    Rows r;
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) r.f[i][e] = split(a(g + (e & 1) * 8, t + i * 8 + (e >> 1) * 4));
    return r;
}
// c[j] += A B_j for N tiles of 16 x 8, 16 of the summed index: b(k, column of tile j) reads an element;
// live(j) (the same for the whole warp) says whether tile j is wanted.  The unit truncates its sums
// (1.6e-6 of relative error over a layer's backward), so each one starts from zero and is added,
// rounded, on the FMA pipe (2.0e-7, and 1.9e-7 at 221 instead of 211 us if after every 8).
template <int N, typename B, typename Live>
__device__ __forceinline__ void product(float (&c)[N][4], const Rows& a, B b, Live live) {
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
#pragma unroll
    for (int j = 0; j < N; j++) {
        if (!live(j)) continue;
        float d[4] = {};
        Split s[2][2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const auto& f = a.f[i];
            const Split b0 = split(b(t + 8 * i, j * 8 + g)), b1 = split(b(t + 8 * i + 4, j * 8 + g));
            mma_tf32(d, f[0].lo, f[1].lo, f[2].lo, f[3].lo, b0.hi, b1.hi);
            mma_tf32(d, f[0].hi, f[1].hi, f[2].hi, f[3].hi, b0.lo, b1.lo);
            s[i][0] = b0;
            s[i][1] = b1;
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const auto& f = a.f[i];
            mma_tf32(d, f[0].hi, f[1].hi, f[2].hi, f[3].hi, s[i][0].hi, s[i][1].hi);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) c[j][e] += d[e];
    }
}

template <int DB, int DC, bool STATE>
__global__ void __launch_bounds__(kThreads<DB>) linattn_f32_kernel(const __grid_constant__ LaParams p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    using Smem = F32Smem<DB, DC>;
    constexpr int LDB = Smem::LDB, LDN = Smem::LDN, LDP = Smem::LDP;
    // warps over the state: DB / 16 rows of tiles, the rest along its columns; over P and out: 4 rows
    constexpr int NT = kThreads<DB>, NW = NT / 32, MT = DB / 16, CS = DC / (NW / MT), NS = CS / 8;
    constexpr int NP = kC / (NW / 4) / 8, CO = DC / (NW / 4), NO = CO / 8;
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
    const int tid = threadIdx.x, warp = tid >> 5, g = (tid & 31) >> 2, t = tid & 3;
    const int sm0 = warp % MT * 16, sn0 = warp / MT * CS;          // this warp's tiles of the state
    // of P and of out: the mask leaves the later rows more to do, and of 8 warps each scheduler has two rows
    constexpr int CW = NW / 4;
    const int mt = warp / CW, cw = warp % CW, m0 = (NW == 8 && mt >= 2 ? 5 - mt : mt) * 16, on0 = cw * CO;
    auto p_col = [&](int j) { return (j * CW + cw) * 8; };
    const float g2 = la_log2_decay(p.log_decay[h]);

    for (int i = tid; i <= kC; i += NT) sm.w[i] = exp2f(g2 * (float)i);

    const int nchunk = (ntok + kC - 1) / kC;
    // copies of chunk `it`, one group for b and c and one for a; the groups may be empty
    auto chunk_start = [&](int it) { return (int64_t)(r.reverse ? nchunk - 1 - it : it) * kC; };
    auto load_bc = [&](int it) {
        if (it < nchunk) {
            const int64_t at = chunk_start(it);
            load_tile<DB, LDB, NT>(sm.b[it & 1], r.b, b, h, tok0 + at, (int)(ntok - at), 0, r.db);
            load_tile<DC, LDN, NT>(sm.c[it & 1], r.c, b, h, tok0 + at, (int)(ntok - at), col0, cols);
        }
    };
    auto load_a = [&](int it) {
        if (!STATE && it < nchunk) {
            const int64_t at = chunk_start(it);
            load_tile<DB, LDB, NT>(sm.a, r.a, b, h, tok0 + at, (int)(ntok - at), 0, r.db);
        }
    };
    load_bc(0);
    load_a(0);

    // state fragments: element e of tile j is row sm0 + g (+ 8), column sn0 + 8 j + 2 t (+ 1); from the state that
    // the scan has left in the segment's place, or from the initial state and the segments before
    float s[NS][4];
    auto s_row = [&](int e) { return sm0 + g + (e & 2) * 4; };
    auto s_col = [&](int j, int e) { return sn0 + 8 * j + 2 * t + (e & 1); };
    auto valid = [&](int j, int e) { return s_row(e) < r.db && s_col(j, e) < cols; };
    const float* segs = r.seg + bh * p.nseg * r.db * r.dc;
    const bool scanned = p.nseg > kFold;
    const float* start = STATE ? nullptr : scanned ? segs + (int64_t)seg * r.db * r.dc
                         : r.state0 ? r.state0 + bh * r.db * r.dc : nullptr;
    const int64_t s_i = scanned ? r.dc : r.s_i, s_j = scanned ? 1 : r.s_j;
#pragma unroll
    for (int j = 0; j < NS; j++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            s[j][e] = start && valid(j, e) ? start[s_row(e) * s_i + (col0 + s_col(j, e)) * s_j] : 0.f;
    if (!STATE && !scanned) {
#pragma unroll 2
        for (int before = 0; before < slot; before++) {
            const int at = r.reverse ? p.nseg - 1 - before : before;
            const float f = exp2f(g2 * (float)la_segment_tokens(p, row_len, at));
            const float* v = segs + (int64_t)at * r.db * r.dc + col0;
#pragma unroll
            for (int j = 0; j < NS; j++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    s[j][e] = fmaf(f, s[j][e], valid(j, e) ? v[s_row(e) * r.dc + s_col(j, e)] : 0.f);
        }
    }

    const auto all = [](int) { return true; };
    for (int it = 0; it < nchunk; it++) {
        const int64_t t0 = tok0 + chunk_start(it);
        const int n = (int)min((int64_t)kC, ntok - chunk_start(it));
        const float *sb = sm.b[it & 1], *sc = sm.c[it & 1];
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();                       // this chunk is here; the last one's readers are done
        load_bc(it + 1);
        if (!STATE) {
#pragma unroll
            for (int j = 0; j < NS; j++)
#pragma unroll
                for (int e = 0; e < 4; e += 2)
                    *reinterpret_cast<float2*>(&sm.s[s_row(e) * LDN + s_col(j, e)]) = make_float2(s[j][e], s[j][e + 1]);
            __syncthreads();
            float acc[NP][4] = {}, o[NO][4] = {};
            // scores, of which the causal mask leaves a warp the tiles up to (reverse: from) its rows
            uint32_t tiles = 0;
#pragma unroll
            for (int j = 0; j < NP; j++)
                tiles |= (p_col(j) < n && (r.reverse ? p_col(j) + 7 >= m0 : p_col(j) <= m0 + 15)) << j;
            auto live = [&](int j) { return (tiles >> j & 1) != 0; };
            const int k_end = m0 < n ? DB : 0;             // rows past the last token need nothing
#pragma unroll 1
            for (int k = 0; k < k_end; k += 16) {
                const Rows a = rows([&](int m, int i) { return sm.a[(m0 + m) * LDB + k + i]; });
                product(acc, a, [&](int i, int c) { return sb[(p_col(c >> 3) + (c & 7)) * LDB + k + i]; }, live);
                product(o, a, [&](int i, int c) { return sm.s[(k + i) * LDN + on0 + c]; }, all);   // the state's part
            }
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const int row = m0 + g + e * 4;
                const float f = r.beta * sm.w[r.reverse ? max(n - 1 - row, 0) : row + 1];
#pragma unroll
                for (int j = 0; j < NO; j++) {
                    o[j][e] *= f;
                    o[j][e + 1] *= f;
                }
            }
            __syncthreads();                   // a and S have been read: P goes over S
            load_a(it + 1);
#pragma unroll
            for (int j = 0; j < NP; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int row = m0 + g + (e & 2) * 4, col = p_col(j) + 2 * t + (e & 1);
                    const int dist = r.reverse ? col - row : row - col;
                    sm.s[row * LDP + col] = dist >= 0 ? r.alpha * acc[j][e] * sm.w[dist] : 0.f;
                }
            __syncthreads();                   // P is complete
            // causal part
            const int k_lo = r.reverse ? m0 : 0, k_hi = k_end == 0 ? 0 : r.reverse ? n : m0 + 16;
#pragma unroll 1
            for (int k = k_lo; k < k_hi; k += 16)
                product(o, rows([&](int m, int i) { return sm.s[(m0 + m) * LDP + k + i]; }),
                        [&](int i, int c) { return sc[(k + i) * LDN + on0 + c]; }, all);
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const int row = m0 + g + e * 4;
                if (row >= n) continue;
                float* op = static_cast<float*>(r.out) + b * r.o_sb + (t0 + row) * r.o_st + h * r.o_sh + col0;
#pragma unroll
                for (int j = 0; j < NO; j++) {
                    const int col = on0 + 8 * j + 2 * t;
                    if (r.out_vec && col + 1 < cols) {
                        *reinterpret_cast<float2*>(op + col) = make_float2(o[j][e], o[j][e + 1]);
                    } else {
                        if (col < cols) op[col] = o[j][e];
                        if (col + 1 < cols) op[col + 1] = o[j][e + 1];
                    }
                }
            }
        }
        // state update
        const float fn = sm.w[n];
#pragma unroll
        for (int j = 0; j < NS; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[j][e] *= fn;
#pragma unroll 1
        for (int k = 0; k < n; k += 16) {
            // weights of the tokens of this thread's elements; rows past n are zero
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int at = k + t + 4 * i;
                f[i] = r.sigma * sm.w[r.reverse ? at + 1 : max(n - 1 - at, 0)];
            }
            product(s, rows([&](int m, int i) { return sb[(k + i) * LDB + sm0 + m] * f[i >> 2]; }),
                    [&](int i, int c) { return sc[(k + i) * LDN + sn0 + c]; }, all);
        }
    }

    if (STATE || (slot == p.nseg - 1 && r.state_out)) {
        float* dst = STATE ? r.seg + (bh * p.nseg + seg) * r.db * r.dc : r.state_out + bh * r.db * r.dc;
        const int64_t d_i = STATE ? r.dc : r.s_i, d_j = STATE ? 1 : r.s_j;
#pragma unroll
        for (int j = 0; j < NS; j++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (valid(j, e)) dst[s_row(e) * d_i + (col0 + s_col(j, e)) * d_j] = s[j][e];
    }
    if (STATE) return;
    // tokens past the row's length
    const int seg_end = (int)min((int64_t)p.seglen, (int64_t)p.seqlen - tok0);
    const int64_t total = (int64_t)(seg_end - ntok) * DC;
    for (int64_t i = tid; i < total; i += NT) {
        const int tk = ntok + (int)(i / DC), c = (int)(i % DC);
        if (c >= cols) continue;
        static_cast<float*>(r.out)[b * r.o_sb + (tok0 + tk) * r.o_st + h * r.o_sh + col0 + c] = 0.f;
    }
}

// The segments' states from a zero start become the states they start from: thread = state element,
// the segments in the order of walking, eight loads ahead of the fold.  Bound by HBM or, as in most
// calls, by the latency of one pass (14 rows x 15 segments of 37 x 100: 8 us).
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
cudaError_t launch_f32(const LaParams& p, int max_dc, cudaStream_t stream) {
    constexpr int bytes = (int)sizeof(F32Smem<DB, DC>);
    auto main_k = linattn_f32_kernel<DB, DC, false>;
    auto state_k = linattn_f32_kernel<DB, DC, true>;
    cudaError_t e = cudaFuncSetAttribute(main_k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(state_k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    const unsigned rows = (unsigned)(p.batch * p.heads), tiles = (max_dc + DC - 1) / DC;
    if (p.nseg > 1) {
        // the last segment (in walking order) feeds nobody
        state_k<<<dim3(rows * (p.nseg - 1), tiles, p.nroles), kThreads<DB>, bytes, stream>>>(p);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
        if (p.nseg > kFold && (e = launch_linattn_scan(p, stream)) != cudaSuccess) return e;
    }
    main_k<<<dim3(rows * p.nseg, tiles, p.nroles), kThreads<DB>, bytes, stream>>>(p);
    return cudaGetLastError();
}

// bfloat16 (batch, token, head, channel) of any strides into rows of whole 16-byte pieces, which a TMA
// can fetch; thread = piece.  EVEN: rows start on 4 bytes and have an even number of channels.
// Bound by its loads of 2 and 4 bytes: 22560 tokens of 14 heads of 37 in 14 us (3.5 TB/s), of 100
// in 33 us (3.9 TB/s).
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

// A CTA does p.tokens tokens; V channels (V divides d) per thread and step.  Bound by HBM: 22560
// tokens of 14 float32 heads of 100 into 7 of bfloat16 in 40 us (3.9 TB/s).
template <typename T, int V>
__global__ void __launch_bounds__(256) linattn_group_kernel(const __grid_constant__ LaGroupParams p) {
    const int groups = p.heads / p.share, dv = p.d / V, per = groups * dv;
    const int64_t tokens = (int64_t)p.batch * p.seqlen, first = (int64_t)blockIdx.x * p.tokens;
    const int64_t b0 = first / p.seqlen;
    const int t0 = (int)(first - b0 * p.seqlen);
    const int n = (int)(tokens - first < p.tokens ? tokens - first : p.tokens);
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
cudaError_t launch_group(LaGroupParams p, cudaStream_t stream) {
    const int64_t tokens = (int64_t)p.batch * p.seqlen;
    // so many that a CTA's elements count in 32 bits (one token has at most 2^23 heads of 128)
    p.tokens = (int64_t)p.heads / p.share * p.d < (1 << 26) ? 16 : 1;
    const unsigned grid = (unsigned)((tokens + p.tokens - 1) / p.tokens);
    if (p.d % 4 == 0) linattn_group_kernel<T, 4><<<grid, 256, 0, stream>>>(p);
    else linattn_group_kernel<T, 1><<<grid, 256, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_linattn_f32(const LaParams& p, cudaStream_t stream) {
    int db = 0, dc = 0;
    for (int i = 0; i < p.nroles; i++) {
        db = p.role[i].db > db ? p.role[i].db : db;
        dc = p.role[i].dc > dc ? p.role[i].dc : dc;
    }
    if (db <= 32) return dc <= 32 ? launch_f32<32, 32>(p, dc, stream) : launch_f32<32, 64>(p, dc, stream);
    if (db <= 64) return dc <= 32 ? launch_f32<64, 32>(p, dc, stream) : launch_f32<64, 64>(p, dc, stream);
    return dc <= 32 ? launch_f32<128, 32>(p, dc, stream) : launch_f32<128, 64>(p, dc, stream);
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
