// Linear attention with a decay for each head on the fifth-generation tensor cores: bfloat16
// streams whose rows a TMA can fetch (the recurrence and its four uses are in linattn.h).
//
// A CTA walks one (batch row, head, segment) in chunks of 128 tokens.  Per chunk, with
// w = exp(log_decay[h]) and the float32 state S^T (row = channel of c) in registers:
//     scores = A B^T                         128 x 128, then P = alpha scores o W as bfloat16
//     O      = P C + beta diag(w^.) (A S)    two products; the second is taken out of TMEM and
//                                            scaled per row before the first uses its columns
//     U      = (C'^T) B,  S^T = w^n S^T + U      C' = sigma diag(w^.) C
// Operands: A, B, C arrive by TMA in 128-byte-swizzled tiles (two stages); B serves as the K-major
// operand of the scores and as the N-major operand of U, C as the N-major operand of P C; P and
// C'^T are written by the threads into TMEM as A operands; bfloat16(S) goes to shared memory.
//
// Roundings below float32: P and the copy of S that A multiplies are bfloat16, each on its own
// part of O, whose result is rounded to bfloat16 anyway.  The state itself is float32: C' is
// carried as a sum of three bfloat16 planes (24 bits) with the smallest terms added first where the
// TMEM has room, and U is added to the decayed state in float32.
//
// Warps 0-7 (two warpgroups, each with half of the columns) do the work between products;
// warp 8 issues the products, warp 9 the copies.  The order of the phases lets each run beside a
// product:  C'(c) | scores, A S;   P(c) | U;   S(c + 1) | P C;   O(c) | scores(c + 1).
// Every wait is bounded: the first that runs out sets the device error word and a flag that
// ends all others.
#include "common.cuh"
#include "linattn.h"
#include "tcgen05.cuh"

namespace ssm {

namespace {

constexpr int kT = 128;                    // tokens per chunk
constexpr int kPanel = kT * 128;           // bytes of 128 rows x 64 channels
constexpr int kCompute = 256;
constexpr int kThreads = kCompute + 128;   // the third warpgroup issues copies and products
// Registers: launched with 168 each (384 * 168 = 64512 = 256 * 224 + 128 * 56)
constexpr int kRegsCompute = 224, kRegsControl = 56;
constexpr uint32_t kTmemCols = 512;
// TMEM columns
constexpr uint32_t kColScores = 0;         // 128: scores, then P in [0, 32) and [64, 96), the
                                           //      third plane of C' in [32, 64) and [96, 128)
constexpr uint32_t kColO = 128;            // 128: A S, then P C
constexpr uint32_t kColU = 256;            // 128: U
constexpr uint32_t kColC = 384;            // 64 + 64: second and first plane of C'^T

// Decay tables in shared memory, filled once per CTA.
struct Decays {
    float pow[kT + 1];                     // w^0 .. w^128
    float score[kT];                       // alpha w^d: weights of P by distance
    alignas(16) float full[kT];            // weights of C' for a chunk of 128 tokens
    alignas(16) float part[kT];            // and for the row's one shorter chunk, zero past its end
};

__device__ __forceinline__ void fill_decays(Decays& d, float g2, float alpha, float sigma, int reverse, int n_part) {
    for (int i = threadIdx.x; i <= kT; i += kThreads) {
        d.pow[i] = exp2f(g2 * (float)i);
        if (i < kT) {
            d.score[i] = alpha * exp2f(g2 * (float)i);
            d.full[i] = sigma * exp2f(g2 * (float)(reverse ? i + 1 : kT - 1 - i));
            d.part[i] = i < n_part ? sigma * exp2f(g2 * (float)(reverse ? i + 1 : n_part - 1 - i)) : 0.f;
        }
    }
}

// KB: channels of a and b, KC: channels of c and out, padded to 64 or 128
template <int KB, int KC>
struct TcSmem {
    static constexpr int A = KB / 64 * kPanel, C = KC / 64 * kPanel;
    static constexpr int STAGE = 2 * A + C;
    static constexpr int S = KB / 64 * KC * 128;       // [i panel][j row][64 i]
    static constexpr int OFF_S = 2 * STAGE;
    static constexpr int OFF_W = OFF_S + S;
    static constexpr int OFF_BAR = OFF_W + (int)sizeof(Decays);
    static constexpr int NBAR = 16;
    static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
    static constexpr int USED = OFF_MISC + 16;
    // more than half an SM, so that two CTAs never share one SM's TMEM
    static constexpr int BYTES = USED > 120 * 1024 ? USED : 120 * 1024;
};

enum Bar { kFull = 0, kStaged = 2, kScores = 4, kAS, kUpd, kPC, kSReady, kCReady, kPReady, kFixed, kDrain };

struct Waiter {
    uint64_t* bars;
    volatile int* abort;
    int* err;
    // false once any wait of the CTA has run out
    __device__ __forceinline__ bool operator()(int bar, uint32_t parity) const {
        if (mbar_try_wait(bars + bar, parity)) return true;
        return slow(bar, parity);
    }
    __device__ __forceinline__ bool slow(int bar, uint32_t parity) const {
        const long long start = clock64();
        while (!mbar_try_wait(bars + bar, parity)) {
            if (*abort) return false;
            if (clock64() - start > 2000000000LL) {
                *abort = 1;
                *err = kDevErrTmaTimeout;
                return false;
            }
        }
        return true;
    }
};

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// The three bfloat16 planes of the decayed, transposed C' for the 32 channels j0 .. of the warp and
// the 64 tokens s0 .., as TMEM fragments: plane[lanes 0-15, 16-31][two registers per 8 tokens].
// weights points at the weight of token s0.
struct Planes {
    uint32_t p[3][2][16];
};
__device__ __forceinline__ void decayed_planes(uint32_t tile, int j0, int s0, const float* weights, float factor,
                                               Planes& o) {
    const int lane = threadIdx.x & 31, rr = lane & 7;
    const uint32_t addr = tile + (j0 >> 6) * kPanel + (s0 + rr) * 128 +
                          (((((j0 & 63) >> 3) + (lane >> 3)) ^ rr) << 4);
    const float* wp = weights + 2 * (lane & 3);
#pragma unroll
    for (int blk = 0; blk < 8; blk++) {
        uint32_t m[4];
        ldmatrix_x4_trans(addr + blk * 1024, m[0], m[1], m[2], m[3]);
        float2 wt = *reinterpret_cast<const float2*>(wp + blk * 8);
        wt.x *= factor;
        wt.y *= factor;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float x = bf16_lo(m[i]) * wt.x, y = bf16_hi(m[i]) * wt.y;
            const int at = 2 * blk + (i & 1);
            const uint32_t h = pack_bf16(x, y);
            o.p[0][i >> 1][at] = h;
            x -= bf16_lo(h);
            y -= bf16_hi(h);
            const uint32_t l = pack_bf16(x, y);
            o.p[1][i >> 1][at] = l;
            o.p[2][i >> 1][at] = pack_bf16(x - bf16_lo(l), y - bf16_hi(l));
        }
    }
}
__device__ __forceinline__ void store_plane(uint32_t addr, const uint32_t (&p)[2][16]) {
    tmem_st_16x128b_x8(addr, p[0]);
    tmem_st_16x128b_x8(addr + (16u << 16), p[1]);
}

// zeros into rows [n, 128) of `panels` panels of a stage
__device__ __forceinline__ void zero_rows(unsigned char* st, int panels, int n, int tid) {
    for (int i = tid; i < panels * (kT - n) * 8; i += kCompute) {
        const int piece = i % 8, rw = n + (i / 8) % (kT - n), pn = i / 8 / (kT - n);
        *reinterpret_cast<uint4*>(st + pn * kPanel + rw * 128 + piece * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();
}

// What a CTA works on.
struct Work {
    int ri, h, b, slot, seg, row_len, ntok, tok0, nchunk;
    int64_t bh;
};
__device__ __forceinline__ Work locate(const LaParams& p) {
    Work k;
    // the roles of one (batch row, head) run side by side: they read the same tensors
    int64_t id = blockIdx.x;
    k.ri = (int)(id % p.nroles);
    id /= p.nroles;
    k.h = (int)(id % p.heads);
    id /= p.heads;
    k.b = (int)(id % p.batch);
    k.slot = (int)(id / p.batch);
    k.seg = p.role[k.ri].reverse ? p.nseg - 1 - k.slot : k.slot;
    k.bh = (int64_t)k.b * p.heads + k.h;
    k.row_len = la_row_length(p, k.b);
    k.ntok = la_segment_tokens(p, k.row_len, k.seg);
    k.tok0 = k.seg * p.seglen;
    k.nchunk = (k.ntok + kT - 1) / kT;
    return k;
}

template <int KB, int KC>
__global__ void __launch_bounds__(kThreads, 1) linattn_tc_kernel(const __grid_constant__ LaParams p,
                                                                 const __grid_constant__ LaMaps maps) {
    extern __shared__ __align__(1024) unsigned char smem[];
    using L = TcSmem<KB, KC>;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
    Decays& dec = *reinterpret_cast<Decays*>(smem + L::OFF_W);
    volatile int* abort = reinterpret_cast<volatile int*>(smem + L::OFF_MISC);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC + 4);
    const Waiter wait{bars, abort, p.err};

    const Work k = locate(p);
    const LaRole& r = p.role[k.ri];
    const int reverse = r.reverse, nchunk = k.nchunk;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float g2 = la_log2_decay(p.log_decay[k.h]);
    const bool tma_out = !r.out_f32 && r.out_vec;
    // chunk of step c, its first token and its tokens
    auto first = [&](int c) { return k.tok0 + (reverse ? nchunk - 1 - c : c) * kT; };
    auto count = [&](int c) { return min(kT, k.tok0 + k.ntok - first(c)); };

    if ((smem_u32(smem) & 1023u) != 0) {
        if (tid == 0) *p.err = kDevErrSmemAlign;
        return;
    }
    if (warp == 8) tmem_alloc(tmem_slot, kTmemCols);
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(bars + kFull + i, 1);
            mbar_init(bars + kStaged + i, 8);
        }
        for (int i : {kScores, kAS, kUpd, kPC, kDrain}) mbar_init(bars + i, 1);
        for (int i : {kSReady, kCReady, kPReady, kFixed}) mbar_init(bars + i, 8);
        *abort = 0;
        fence_mbar_init();
    }
    fill_decays(dec, g2, r.alpha, r.sigma, reverse, nchunk > 0 ? k.ntok - (nchunk - 1) * kT : 0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp >= 8) {
        regs_release<kRegsControl>();
        if (warp == 9 && lane == 0) {
            // ---- copies -------------------------------------------------------------------------
            auto load = [&](int c) {
                unsigned char* st = smem + (c & 1) * L::STAGE;
                uint64_t* bar = bars + kFull + (c & 1);
                const int t = first(c);
                mbar_arrive_expect_tx(bar, L::STAGE);
#pragma unroll
                for (int i = 0; i < KB / 64; i++) {
                    tma_load_4d(st + i * kPanel, &maps.a[k.ri], bar, i * 64, t, k.h / r.a.share, k.b);
                    tma_load_4d(st + L::A + i * kPanel, &maps.b[k.ri], bar, i * 64, t, k.h / r.b.share, k.b);
                }
#pragma unroll
                for (int i = 0; i < KC / 64; i++)
                    tma_load_4d(st + 2 * L::A + i * kPanel, &maps.c[k.ri], bar, i * 64, t, k.h / r.c.share, k.b);
            };
            int issued = 0;
            for (; issued < 2 && issued < nchunk; issued++) load(issued);
            for (int c = 0; c < nchunk; c++) {
                // the chunk's output is staged over its a (and b) tile, and nobody uses its stage any more
                if (!wait(kStaged + (c & 1), (c >> 1) & 1)) break;
                if (tma_out) {
#pragma unroll
                    for (int i = 0; i < KC / 64; i++)
                        if (i * 64 < r.dc)
                            tma_store_4d(&maps.o[k.ri], smem + (c & 1) * L::STAGE + i * kPanel, i * 64, first(c), k.h, k.b);
                    tma_store_commit();
                    tma_store_wait_read_all();
                }
                if (issued < nchunk) load(issued++);
            }
            tma_store_wait_all();
            if (*abort)      // copies in flight still write to this CTA's shared memory
                for (int c = max(0, issued - 2); c < issued; c++) mbar_wait_bounded(bars + kFull + (c & 1), (c >> 1) & 1);
        } else if (warp == 8 && elect_one()) {
            // ---- products -----------------------------------------------------------------------
            constexpr uint32_t id_scores = umma_idesc(128, 128, false), id_as = umma_idesc(128, KC, false),
                               id_pc = umma_idesc(128, KC, true), id_upd = umma_idesc(128, KB, true);
            const uint32_t s_desc = umma_desc_lo(smem_u32(smem + L::OFF_S), 16);
            for (int c = 0; c < nchunk; c++) {
                const uint32_t st = smem_u32(smem + (c & 1) * L::STAGE), par = c & 1;
                if (!wait(kFull + (c & 1), (c >> 1) & 1)) break;
                if (count(c) < kT && !wait(kFixed, 0)) break;
                // P and the third plane of the previous chunk are still read until these two
                if (c > 0 && !(wait(kPC, par ^ 1) && wait(kUpd, par ^ 1))) break;
                tc_fence_after();
                // K-major panels of 64 channels: 16 channels are 32 bytes
                const uint32_t a_desc = umma_desc_lo(st, 16), b_desc = umma_desc_lo(st + L::A, 16);
#pragma unroll
                for (int i = 0; i < KB / 16; i++) {
                    const uint32_t off = ((i >> 2) * kPanel + (i & 3) * 32) >> 4;
                    umma_ss(tmem + kColScores, a_desc + off, b_desc + off, id_scores, i > 0);
                }
                umma_commit(bars + kScores);
                if (!wait(kSReady, par)) break;
                if (c > 0 && !wait(kStaged + (par ^ 1), ((c - 1) >> 1) & 1)) break;   // O has been read
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < KB / 16; i++)
                    umma_ss(tmem + kColO, a_desc + (((i >> 2) * kPanel + (i & 3) * 32) >> 4),
                            s_desc + (((i >> 2) * (KC * 128) + (i & 3) * 32) >> 4), id_as, i > 0);
                umma_commit(bars + kAS);
                if (!wait(kCReady, par)) break;
                tc_fence_after();
                // N-major panels of 64 channels: 16 tokens are 2048 bytes
                const uint32_t bn_desc = umma_desc_lo(st + L::A, kPanel), cn_desc = umma_desc_lo(st + 2 * L::A, kPanel);
#pragma unroll
                for (int i = 0; i < 2 * kT / 16; i++)      // second plane, then first
                    umma_ts(tmem + kColU, tmem + kColC + i * 8, bn_desc + (i & 7) * (2048 >> 4), id_upd, i > 0);
                if (!wait(kPReady, par)) break;
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < kT / 16; i++)
                    umma_ts(tmem + kColU, tmem + kColScores + (i >> 2) * 64 + 32 + (i & 3) * 8,
                            bn_desc + i * (2048 >> 4), id_upd, 1);
                umma_commit(bars + kUpd);
#pragma unroll
                for (int i = 0; i < kT / 16; i++)
                    umma_ts(tmem + kColO, tmem + kColScores + (i >> 2) * 64 + (i & 3) * 8, cn_desc + i * (2048 >> 4),
                            id_pc, i > 0);
                umma_commit(bars + kPC);
            }
            if (*abort) {
                umma_commit(bars + kDrain);
                mbar_wait_bounded(bars + kDrain, 0);
            }
        }
        __syncwarp();
    } else {
        // ---- the work between products ----------------------------------------------------------
        regs_claim<kRegsCompute>();
        const int q = warp & 3, half = warp >> 2;     // TMEM lanes 32 q .. + 32; half of the columns
        const uint32_t tm = tmem + ((uint32_t)(q * 32) << 16);
        const int row = q * 32 + lane;                // token of P and O, channel of c (row j of S^T)
        constexpr int NS = KB / 2;                    // columns of S^T per thread
        constexpr int NO = KC / 2;                    // columns of O per thread
        const bool s_on = q * 32 < KC;                // S^T has KC rows
        const int i0 = half * NS, o0 = half * NO;
        auto arrive = [&](int bar) {
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + bar);
        };
        auto ok = [&](bool v) { return __all_sync(0xffffffffu, v); };

        // S^T of the first chunk: the initial state, then the segments before this one.  Through TMEM,
        // so that the loop over columns stays a loop (registers have no index).
        float s[NS];
        if (s_on) {
            const float* src0 = r.state0 && row < r.dc ? r.state0 + k.bh * r.db * r.dc + row * r.s_j : nullptr;
            const float* src = r.seg + k.bh * p.nseg * r.db * r.dc + row;
#pragma unroll 1
            for (int i = 0; i < NS; i += 8) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = src0 && i0 + i + e < r.db ? src0[(i0 + i + e) * r.s_i] : 0.f;
#pragma unroll 1
                for (int g = 0; g < k.slot; g++) {
                    const int sg = reverse ? p.nseg - 1 - g : g;
                    const float f = exp2f(g2 * (float)la_segment_tokens(p, k.row_len, sg));
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        x[e] = fmaf(f, x[e], row < r.dc && i0 + i + e < r.db ? src[(sg * r.db + i0 + i + e) * r.dc] : 0.f);
                }
                uint32_t v[8];
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = __float_as_uint(x[e]);
                tmem_st8(tm + kColU + i0 + i, v);
            }
            tmem_wait_st();
#pragma unroll
            for (int i = 0; i < NS; i++) s[i] = 0.f;
        }
        // bfloat16(S^T) to shared memory for A S
        auto put_state = [&]() {
            if (s_on) {
#pragma unroll
                for (int i = 0; i < NS; i += 8) {
                    const uint4 v = make_uint4(pack_bf16(s[i], s[i + 1]), pack_bf16(s[i + 2], s[i + 3]),
                                               pack_bf16(s[i + 4], s[i + 5]), pack_bf16(s[i + 6], s[i + 7]));
                    const int ii = i0 + i;
                    *reinterpret_cast<uint4*>(smem + L::OFF_S + (ii >> 6) * (KC * 128) + swz128(row, (ii & 63) * 2)) = v;
                }
            }
            fence_proxy_async_smem();
            arrive(kSReady);
        };
        auto add_update = [&](int n) {
            if (!s_on) return;
            const float fn = dec.pow[n];
#pragma unroll
            for (int i = 0; i < NS; i += 32) {
                uint32_t v[32];
                tmem_ld32(tm + kColU + i0 + i, v);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; e++) s[i + e] = fmaf(fn, s[i + e], __uint_as_float(v[e]));
            }
        };
        add_update(0);
        if (nchunk > 0) {
            tc_fence_before();
            put_state();
        }

        bool fine = true;
        for (int c = 0; c < nchunk; c++) {
            const uint32_t par = c & 1;
            const int n = count(c);
            unsigned char* st = smem + (c & 1) * L::STAGE;
            if (!(fine = ok(wait(kFull + (c & 1), (c >> 1) & 1)))) break;
            if (n < kT) {
                // rows past the length hold whatever the caller's padding holds
                zero_rows(st, L::STAGE / kPanel, n, tid);
                arrive(kFixed);
                if (!(fine = ok(wait(kFixed, 0)))) break;
            }
            // planes of C'^T for this half's 64 tokens; the third waits for its columns
            Planes pl;
            if (s_on) {
                decayed_planes(smem_u32(st + 2 * L::A), q * 32, half * 64, (n < kT ? dec.part : dec.full) + half * 64,
                               1.f, pl);
                store_plane(tm + kColC + half * 32, pl.p[1]);
                store_plane(tm + kColC + 64 + half * 32, pl.p[0]);
                tmem_wait_st();
            }
            tc_fence_before();
            arrive(kCReady);

            // P in blocks of 32 x 32, which the mask empties, halves or leaves whole
            if (!(fine = ok(wait(kScores, par)))) break;
            tc_fence_after();
#pragma unroll 1
            for (int blk = 0; blk < 2; blk++) {
                const int sb = half * 2 + blk;
                uint32_t o[16];
                if (reverse ? sb >= q : sb <= q) {
                    uint32_t v[32];
                    tmem_ld32(tm + kColScores + sb * 32, v);
                    tmem_wait_ld();
                    const int d0 = reverse ? sb * 32 - row : row - sb * 32;   // distance to the block's first column
                    const float* wt = dec.score + d0;
                    if (reverse) {
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            o[e] = pack_bf16(d0 + 2 * e >= 0 ? __uint_as_float(v[2 * e]) * wt[2 * e] : 0.f,
                                             d0 + 2 * e + 1 >= 0 ? __uint_as_float(v[2 * e + 1]) * wt[2 * e + 1] : 0.f);
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            o[e] = pack_bf16(d0 >= 2 * e ? __uint_as_float(v[2 * e]) * wt[-2 * e] : 0.f,
                                             d0 >= 2 * e + 1 ? __uint_as_float(v[2 * e + 1]) * wt[-2 * e - 1] : 0.f);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 16; e++) o[e] = 0;
                }
                // over scores that this thread has read: 16 of the half's first 32 columns per block
                tmem_st16(tm + kColScores + half * 64 + blk * 16, o);
            }
            // every warp of this half that shares the lanes is this warp: its scores are read
            if (s_on) store_plane(tm + kColScores + half * 64 + 32, pl.p[2]);
            // A S leaves TMEM, scaled per row
            if (!(fine = ok(wait(kAS, par)))) break;
            tc_fence_after();
            float acc[NO];
            {
                const float f = r.beta * dec.pow[reverse ? max(n - 1 - row, 0) : row + 1];
#pragma unroll
                for (int i = 0; i < NO; i += 32) {
                    uint32_t v[32];
                    tmem_ld32(tm + kColO + o0 + i, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; e++) acc[i + e] = __uint_as_float(v[e]) * f;
                }
            }
            tmem_wait_st();
            tc_fence_before();
            arrive(kPReady);

            // the state after this chunk; the stage's b is also free after the update
            if (!(fine = ok(wait(kUpd, par)))) break;
            tc_fence_after();
            add_update(n);
            if (c + 1 < nchunk) {
                tc_fence_before();
                put_state();
            }

            // O
            if (!(fine = ok(wait(kPC, par)))) break;
            tc_fence_after();
#pragma unroll
            for (int i = 0; i < NO; i += 32) {
                uint32_t v[32];
                tmem_ld32(tm + kColO + o0 + i, v);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; e++) acc[i + e] = row < n ? acc[i + e] + __uint_as_float(v[e]) : 0.f;
            }
            if (tma_out) {
#pragma unroll
                for (int i = 0; i < NO; i += 8) {
                    const uint4 v = make_uint4(pack_bf16(acc[i], acc[i + 1]), pack_bf16(acc[i + 2], acc[i + 3]),
                                               pack_bf16(acc[i + 4], acc[i + 5]), pack_bf16(acc[i + 6], acc[i + 7]));
                    const int oc = o0 + i;
                    *reinterpret_cast<uint4*>(st + (oc >> 6) * kPanel + swz128(row, (oc & 63) * 2)) = v;
                }
                fence_proxy_async_smem();
            } else {
                // float32 partials and rows a TMA cannot store: through the warp's own piece of the stage,
                // 16-byte pieces swizzled by the row, then row by row
                float* own = reinterpret_cast<float*>(st) + warp * 32 * NO;
#pragma unroll
                for (int i = 0; i < NO; i += 4)
                    *reinterpret_cast<float4*>(own + lane * NO + (((i >> 2) ^ (lane & 7)) << 2)) =
                        make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
                __syncwarp();
                const int64_t at = k.b * r.o_sb + (int64_t)(first(c) + q * 32) * r.o_st + k.h * r.o_sh + o0;
                const int cols = min(NO, r.dc - o0), rows = min(32, n - q * 32);
#pragma unroll 1
                for (int i = lane; i < rows * NO; i += 32) {
                    const int rw = i / NO, col = i % NO;
                    const float x = own[rw * NO + (((col >> 2) ^ (rw & 7)) << 2) + (col & 3)];
                    if (col >= cols) continue;
                    if (r.out_f32) static_cast<float*>(r.out)[at + rw * r.o_st + col] = x;
                    else static_cast<__nv_bfloat16*>(r.out)[at + rw * r.o_st + col] = __float2bfloat16_rn(x);
                }
                fence_proxy_async_smem();
            }
            tc_fence_before();
            arrive(kStaged + (c & 1));
        }

        if (fine) {
            if (k.slot == p.nseg - 1 && r.state_out && s_on) {
#pragma unroll
                for (int i = 0; i < NS; i += 32) {
                    uint32_t v[32];
#pragma unroll
                    for (int e = 0; e < 32; e++) v[e] = __float_as_uint(s[i + e]);
                    tmem_st32(tm + kColU + i0 + i, v);
                }
                tmem_wait_st();
                float* dst = r.state_out + k.bh * r.db * r.dc + row * r.s_j;
#pragma unroll 1
                for (int i = 0; i < NS; i += 8) {
                    uint32_t v[8];
                    tmem_ld8(tm + kColU + i0 + i, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (row < r.dc && i0 + i + e < r.db) dst[(i0 + i + e) * r.s_i] = __uint_as_float(v[e]);
                }
            }
            // tokens past the row's length
            const int total = (min(p.seglen, p.seqlen - k.tok0) - k.ntok) * KC;
            for (int i = tid; i < total; i += kCompute) {
                const int t = k.ntok + i / KC, cc = i % KC;
                if (cc >= r.dc) continue;
                const int64_t at = k.b * r.o_sb + (int64_t)(k.tok0 + t) * r.o_st + k.h * r.o_sh + cc;
                if (r.out_f32) static_cast<float*>(r.out)[at] = 0.f;
                else static_cast<__nv_bfloat16*>(r.out)[at] = __float2bfloat16_rn(0.f);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 8) tmem_dealloc(tmem, kTmemCols);
}

// The state a segment reaches from a zero start: only U, with every token weighted towards the
// segment's end, so that the sum needs no rescaling between chunks.  C'^T has two buffers of
// three planes; the threads fill one while the product reads the other.
constexpr int kStages = 3;
template <int KB, int KC>
struct StateSmem {
    static constexpr int B = KB / 64 * kPanel, C = KC / 64 * kPanel;
    static constexpr int STAGE = B + C;
    static constexpr int OFF_W = kStages * STAGE;
    static constexpr int OFF_BAR = OFF_W + (int)sizeof(Decays);
    static constexpr int OFF_MISC = OFF_BAR + 16 * 8;
    static constexpr int USED = OFF_MISC + 16;
    static constexpr int BYTES = USED > 120 * 1024 ? USED : 120 * 1024;
};
enum StateBar { kSbFull = 0, kSbFree = 3, kSbReady = 6, kSbDone = 8, kSbFixed = 10, kSbDrain = 11 };

template <int KB, int KC>
__global__ void __launch_bounds__(kThreads, 1) linattn_tc_state_kernel(const __grid_constant__ LaParams p,
                                                                       const __grid_constant__ LaMaps maps) {
    extern __shared__ __align__(1024) unsigned char smem[];
    using L = StateSmem<KB, KC>;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
    Decays& dec = *reinterpret_cast<Decays*>(smem + L::OFF_W);
    volatile int* abort = reinterpret_cast<volatile int*>(smem + L::OFF_MISC);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC + 4);
    const Waiter wait{bars, abort, p.err};

    const Work k = locate(p);
    const LaRole& r = p.role[k.ri];
    const int reverse = r.reverse, nchunk = k.nchunk;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float g2 = la_log2_decay(p.log_decay[k.h]);
    auto first = [&](int c) { return k.tok0 + c * kT; };
    auto count = [&](int c) { return min(kT, k.tok0 + k.ntok - first(c)); };

    if ((smem_u32(smem) & 1023u) != 0) {
        if (tid == 0) *p.err = kDevErrSmemAlign;
        return;
    }
    if (warp == 8) tmem_alloc(tmem_slot, kTmemCols);
    if (tid == 0) {
        for (int i = 0; i < kStages; i++) {
            mbar_init(bars + kSbFull + i, 1);
            mbar_init(bars + kSbFree + i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(bars + kSbReady + i, 8);
            mbar_init(bars + kSbDone + i, 1);
        }
        mbar_init(bars + kSbFixed, 8);
        mbar_init(bars + kSbDrain, 1);
        *abort = 0;
        fence_mbar_init();
    }
    fill_decays(dec, g2, r.alpha, r.sigma, reverse, nchunk > 0 ? k.ntok - (nchunk - 1) * kT : 0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 9) {
        if (lane == 0) {
            auto load = [&](int c) {
                unsigned char* st = smem + (c % kStages) * L::STAGE;
                uint64_t* bar = bars + kSbFull + c % kStages;
                mbar_arrive_expect_tx(bar, L::STAGE);
#pragma unroll
                for (int i = 0; i < KB / 64; i++)
                    tma_load_4d(st + i * kPanel, &maps.b[k.ri], bar, i * 64, first(c), k.h / r.b.share, k.b);
#pragma unroll
                for (int i = 0; i < KC / 64; i++)
                    tma_load_4d(st + L::B + i * kPanel, &maps.c[k.ri], bar, i * 64, first(c), k.h / r.c.share, k.b);
            };
            int issued = 0;
            for (; issued < kStages && issued < nchunk; issued++) load(issued);
            for (int c = 0; issued < nchunk; c++) {
                if (!wait(kSbFree + c % kStages, (c / kStages) & 1)) break;
                load(issued++);
            }
            if (*abort)
                for (int c = max(0, issued - kStages); c < issued; c++)
                    mbar_wait_bounded(bars + kSbFull + c % kStages, (c / kStages) & 1);
        }
        __syncwarp();
    } else if (warp == 8) {
        if (elect_one()) {
            constexpr uint32_t id_upd = umma_idesc(128, KB, true);
            for (int c = 0; c < nchunk; c++) {
                if (!wait(kSbFull + c % kStages, (c / kStages) & 1)) break;
                if (!wait(kSbReady + (c & 1), (c >> 1) & 1)) break;
                tc_fence_after();
                const uint32_t bn_desc = umma_desc_lo(smem_u32(smem + (c % kStages) * L::STAGE), kPanel);
                const uint32_t cp = tmem + 128 + (c & 1) * 192;
#pragma unroll
                for (int i = 0; i < 3 * kT / 16; i++)
                    umma_ts(tmem, cp + i * 8, bn_desc + (i & 7) * (2048 >> 4), id_upd, c > 0 || i > 0);
                umma_commit(bars + kSbFree + c % kStages);
                umma_commit(bars + kSbDone + (c & 1));
            }
            if (*abort) {
                umma_commit(bars + kSbDrain);
                mbar_wait_bounded(bars + kSbDrain, 0);
            }
        }
        __syncwarp();
    } else if (warp < 8) {
        const int q = warp & 3, half = warp >> 2;
        const uint32_t tm = tmem + ((uint32_t)(q * 32) << 16);
        const int row = q * 32 + lane;
        const bool s_on = q * 32 < KC;
        auto arrive = [&](int bar) {
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + bar);
        };
        auto ok = [&](bool v) { return __all_sync(0xffffffffu, v); };
        bool fine = true;
        for (int c = 0; c < nchunk; c++) {
            const int n = count(c);
            unsigned char* st = smem + (c % kStages) * L::STAGE;
            if (!(fine = ok(wait(kSbFull + c % kStages, (c / kStages) & 1)))) break;
            if (c >= 2 && !(fine = ok(wait(kSbDone + (c & 1), ((c - 2) >> 1) & 1)))) break;   // the buffer is free
            if (n < kT) {
                zero_rows(st, L::STAGE / kPanel, n, tid);
                arrive(kSbFixed);
                if (!(fine = ok(wait(kSbFixed, 0)))) break;
            }
            if (s_on) {
                // tokens after this chunk (forward) or before it (reverse)
                const int far = reverse ? c * kT : k.ntok - c * kT - n;
                Planes pl;
                decayed_planes(smem_u32(st + L::B), q * 32, half * 64, (n < kT ? dec.part : dec.full) + half * 64,
                               exp2f(g2 * (float)far), pl);
                const uint32_t cp = tm + 128 + (c & 1) * 192 + half * 32;
#pragma unroll
                for (int i = 0; i < 3; i++) store_plane(cp + i * 64, pl.p[2 - i]);   // smallest first
                tmem_wait_st();
            }
            tc_fence_before();
            arrive(kSbReady + (c & 1));
        }
        if (fine && nchunk > 0) fine = ok(wait(kSbDone + ((nchunk - 1) & 1), ((nchunk - 1) >> 1) & 1));
        tc_fence_after();
        if (fine && s_on) {
            constexpr int NS = KB / 2;
            float* e = r.seg + (k.bh * p.nseg + k.seg) * r.db * r.dc;
#pragma unroll 1
            for (int i = half * NS; i < half * NS + NS; i += 8) {
                uint32_t v[8] = {};
                if (nchunk > 0) {
                    tmem_ld8(tm + i, v);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int u = 0; u < 8; u++)
                    if (row < r.dc && i + u < r.db) e[(i + u) * r.dc + row] = __uint_as_float(v[u]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 8) tmem_dealloc(tmem, kTmemCols);
}

template <int KB, int KC>
cudaError_t launch_tc(const LaParams& p, const LaMaps& maps, cudaStream_t stream) {
    cudaError_t e = cudaFuncSetAttribute(linattn_tc_kernel<KB, KC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         TcSmem<KB, KC>::BYTES);
    if (e != cudaSuccess) return e;
    const int64_t rows = (int64_t)p.batch * p.heads * p.nroles;
    if (p.nseg > 1) {
        e = cudaFuncSetAttribute(linattn_tc_state_kernel<KB, KC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 StateSmem<KB, KC>::BYTES);
        if (e != cudaSuccess) return e;
        linattn_tc_state_kernel<KB, KC><<<(unsigned)(rows * (p.nseg - 1)), kThreads, StateSmem<KB, KC>::BYTES, stream>>>(p, maps);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
    linattn_tc_kernel<KB, KC><<<(unsigned)(rows * p.nseg), kThreads, TcSmem<KB, KC>::BYTES, stream>>>(p, maps);
    return cudaGetLastError();
}

}  // namespace

// Every role of p has db <= kb and dc <= kc (64 or 128).
cudaError_t launch_linattn_tc(const LaParams& p, const LaMaps& maps, int kb, int kc, cudaStream_t stream) {
    if (kb == 64) return kc == 64 ? launch_tc<64, 64>(p, maps, stream) : launch_tc<64, 128>(p, maps, stream);
    return kc == 64 ? launch_tc<128, 64>(p, maps, stream) : launch_tc<128, 128>(p, maps, stream);
}

}  // namespace ssm
