// Linear attention with a decay for each head on the fifth-generation tensor cores: bfloat16
// streams whose rows a TMA can fetch (the recurrence and its four uses are in linattn.h).
//
// A row is one (batch row, head, role, segment); it is walked in chunks of 128 tokens.  Per chunk,
// with w = exp(log_decay[h]) and the float32 state S^T (row = channel of c) in registers:
//     scores = A B^T                         128 x 128, then P = alpha scores o W
//     O      = P C + beta diag(w^.) (A S)    two products; the second is taken out of TMEM and
//                                            scaled per row before the first uses its columns
//     U      = (C'^T) B,  S^T = w^n S^T + U      C' = sigma diag(w^.) C
// Operands: A, B, C arrive by TMA in 128-byte-swizzled tiles (in two or four stages); B serves as the K-major
// operand of the scores and as the N-major operand of U, C as the N-major operand of P C; P and
// C'^T are written by the threads into TMEM as A operands; S goes to shared memory.
//
// Roundings below float32: P and the copy of S that A multiplies are each the sum of two bfloat16, an upper
// and a lower half (2^-16; with the upper half alone an output was 2.35e-3 off, of which its own rounding to
// bfloat16 makes 1.66e-3).  The state itself is float32: C' is carried as a sum of four bfloat16 planes
// (24 bits of the weight) and U is added to the decayed state in float32.
//
// One CTA per SM.  Warps 0-7 do the work between products, two for each quarter of the TMEM
// lanes, each with half of the columns; warp 8 issues the products, warp 9 the loads, warp 10
// the stores.  The order of the phases lets each run beside a product:
//     C'(c), first 64 tokens | scores, A S;   P(c) | U, first half;   C'(c), last 64 | P C;
//     O(c) | U, last half;   S(c + 1) | scores(c + 1).
// At 128 x 128 channels shared memory has room for one half of S: the lower one takes the place of the upper
// between C'(c) and P(c).
// Heads of up to 64 channels would leave half of the lanes of C'^T idle.  For them lanes 0-63 take a
// chunk's first 64 tokens and lanes 64-127 the last 64, all warps at once, and the state is kept in two
// parts, each decayed alike and with the U of its half; A S sums over both, and they are joined
// where the state leaves the CTA.  Their smaller tiles have four stages.  1280 tokens of 148 heads:
// 35.0 us without parts and with two stages, 33.0 so (before the lower halves; 44 with them).
//
// With more rows than SMs the CTAs share the chunks of all rows evenly: each takes a contiguous
// range, so its first row may have been begun by the CTA before it and its last may be finished
// by the next.  It does the beginning of its last row first and publishes the state it reaches, and
// the end of its first row last: with rows of one length the state it needs is there by then, since the two
// parts of a row together are no longer than a CTA's range.  With ragged lengths a row can be longer than several
// ranges: its CTAs then run one after the other, each waiting for the one before.
//
// Measured: 4 x 2048 tokens of 40 heads of 128, forward, 100 us (3.5 TB/s of its 346 MB): 4.8 us a chunk, where
// HBM would allow 3.0 (four tiles of 32 KB on 148 SMs); heads of 64 3.2 us against 1.5.  What bounds
// it is the chain of a chunk: six times (seven at 128 x 128) the compute warps wait for a product and hand one
// on, 150 to 250 cycles each, between 500 and 1800 cycles of conversions.  Without the lower halves
// of P and S a chunk took 3.9 and 2.5 us (their products, conversions and code; see above for what they are for).
// Measured against those: groups of warps with one step each took twice as long (their code together misses the
// instruction cache), 16 compute warps 4.5 us a chunk (104 registers: spills), three planes of C' 3.7 us, but
// 1.6e-6 of error in the state.
//
// Every wait is bounded: the first that runs out sets the device error word and a flag that
// ends all others.
#include "common.cuh"
#include "linattn.h"
#include "tcgen05.cuh"

namespace ssm {

cudaError_t launch_linattn_scan(const LaParams& p, cudaStream_t stream);

namespace {

constexpr int kT = 128;                    // tokens per chunk
constexpr int kPanel = kT * 128;           // bytes of 128 rows x 64 channels
constexpr int kWarps = 8;                  // compute warps
constexpr int kCompute = kWarps * 32;
constexpr int kThreads = kCompute + 128;   // the last warpgroup issues copies and products
// Registers: launched with 168 each (384 * 168 = 256 * 216 + 128 * 72; with 56 the warp of the products spills)
constexpr int kRegsCompute = 216, kRegsControl = 72;
constexpr uint32_t kTmemCols = 512;
// TMEM columns
constexpr uint32_t kColScores = 0;         // 128: scores, then P: of each 32 columns 16 for the upper halves, 16 for the lower
constexpr uint32_t kColO = 128;            // 128: A S, then P C
constexpr uint32_t kColU = 256;            // 128: U
constexpr uint32_t kColC = 384;            // 4 x 32: planes of C'^T for 64 tokens
// Tries before a wait has run out: one that fails takes some 200 cycles among many waiters and 7800 alone
// (measured), so 0.1 to 4 s, against the microseconds of the longest wait for a product or a copy.  Tries made
// while the CTA waits for another one's state do not count: that wait has clocks of its own, 1 s and 20 us
// for every chunk that the row has before (one takes 3 to 5)
constexpr int kTries = 1 << 20;
constexpr long long kStateClocks = 2000000000LL, kChunkClocks = 40000;
constexpr float kZeroLog2 = -151.f;        // exp2 of anything below is zero in float32

// A weight as a sum of three bfloat16 of 8 bits each.
__device__ __forceinline__ void split_weight(float x, __nv_bfloat16& u, __nv_bfloat16& v, __nv_bfloat16& z) {
    u = __float2bfloat16_rn(x);
    x -= __bfloat162float(u);
    v = __float2bfloat16_rn(x);
    z = __float2bfloat16_rn(x - __bfloat162float(v));
}

// Decay tables in shared memory, filled once per row.
struct Decays {
    float pow[kT + 1];                     // w^0 .. w^128
    float score[kT];                       // weights of P: alpha w^d at d, or at 127 - d (forward); up to 31
                                           // entries before and after it are read for masked columns, unused
    alignas(16) float block[32];           // within a whole block of P: w^(31 - column), reverse w^column
    // weights of C' by token, split: [0] for a chunk of 128 tokens, [1] for the row's one shorter chunk
    // (zero past its end)
    alignas(16) __nv_bfloat16 plane[2][3][kT];
};

__device__ __forceinline__ float plane_weight(float g2, float sigma, int reverse, int i, int n) {
    return i < n ? sigma * exp2f(g2 * (float)(reverse ? i + 1 : n - 1 - i)) : 0.f;
}
__device__ __forceinline__ void fill_decays(Decays& d, float g2, float alpha, float sigma, int reverse, int n_part) {
    const int i = threadIdx.x;
    if (i <= kT) d.pow[i] = exp2f(g2 * (float)i);
    if (i < 32) d.block[i] = exp2f(g2 * (float)(reverse ? i : 31 - i));
    if (i < kT) {
        d.score[i] = alpha * exp2f(g2 * (float)(reverse ? i : kT - 1 - i));
#pragma unroll
        for (int e = 0; e < 2; e++)
            split_weight(plane_weight(g2, sigma, reverse, i, e ? n_part : kT), d.plane[e][0][i], d.plane[e][1][i],
                         d.plane[e][2][i]);
    }
}

// The chunks [c0, c1) that a CTA does of rows [row0, row1]: from chunk c0 of the first row up to
// chunk c1 of the last.
struct Range {
    int row0, row1, c0, c1;
};

// KB: channels of a and b, KC: channels of c and out, padded to 64 or 128
template <int KB, int KC>
struct TcSmem {
    static constexpr int A = KB / 64 * kPanel, C = KC / 64 * kPanel;
    static constexpr int STAGE = 2 * A + C;
    static constexpr bool TWO = KB == 64 && KC == 64;  // the state in two parts
    static constexpr int S1 = (TWO ? 2 : KB / 64) * KC * 128;  // a half of S: [i panel or part][j row][64 i]
    // both halves of S at once; at 128 x 128 channels there is room for one, and the second follows the first
    static constexpr bool BOTH = KB * KC < 128 * 128;
    static constexpr int S = (BOTH ? 2 : 1) * S1;
    static constexpr int STAGES = TWO ? 4 : 2;
    static constexpr int OFF_S = STAGES * STAGE;
    static constexpr int OFF_W = OFF_S + S;
    static constexpr int OFF_BAR = OFF_W + (int)sizeof(Decays);
    static constexpr int NBAR = 26;
    static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
    static constexpr int USED = OFF_MISC + 16 + (int)sizeof(Range);
    // more than half an SM, so that two CTAs never share one SM's TMEM
    static constexpr int BYTES = USED > 120 * 1024 ? USED : 120 * 1024;
};

// mbarriers.  Those of an array belong to one stage, whose next use nobody can reach before everybody
// has seen this one: a waiter never falls two phases behind.
enum Bar {
    kFull = 0,       // [stages] a stage's tiles are there
    kStaged = 4,     // O is staged over them
    kFree = 8,       // and stored, and every product has read them
    kUpd = 12,       // U is complete
    kScores = 16, kAS, kPC, kCFree,      // products complete; kCFree: those of the first 64 tokens' planes
    kSReady, kCReady, kPReady, kFixed, kItem, kDrain
};

struct Waiter {
    uint64_t* bars;
    volatile int* abort;         // and behind it: does the CTA wait for another one's state?
    int* err;
    // false once any wait of the CTA has run out
    __device__ __forceinline__ bool operator()(int bar, uint32_t parity) const {
        int tries = 0;
        while (!mbar_try_wait(bars + bar, parity)) {
            if (abort[1]) tries = 0;
            if (*abort || ++tries == kTries) {
                *abort = 1;
                *err = kDevErrTmaTimeout;
                return false;
            }
        }
        return true;
    }
    // has any wait run out, or this one, of a flag in global memory, begun at `start`?
    __device__ __forceinline__ bool gone(long long start, int chunks_before) const {
        if (*abort) return true;
        if (clock64() - start <= kStateClocks + chunks_before * kChunkClocks) return false;
        *abort = 1;
        *err = kDevErrTmaTimeout;
        return true;
    }
};

// Two floats as two pairs of bfloat16: their upper 16 bits, cut off, and what these leave, rounded (exact to 2^-16)
__device__ __forceinline__ uint32_t upper_bf16(float x, float y) {
    return __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
}
__device__ __forceinline__ uint32_t lower_bf16(float x, float y) {
    auto minus_upper = [](float v) { return __uint_as_float((__float_as_uint(v) & 0xffff0000u) ^ 0x80000000u); };
    const float2 d = __fadd2_rn(make_float2(x, y), make_float2(minus_upper(x), minus_upper(y)));
    const __nv_bfloat162 v = __floats2bfloat162_rn(d.x, d.y);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// The four bfloat16 planes of the decayed, transposed C' for the 32 channels j0 .. of the warp and
// the 32 tokens s0 .., as TMEM fragments: plane[lanes 0-15, 16-31][two registers per 8 tokens].
// weights(i) gives the split weights of the lane's token pair of the 8 tokens s0 + 8 i ...
//
// In packed bfloat16 arithmetic: the weight is u + v + z, 8 bits each, and c has 8 bits, so the
// rounding error of a product is itself a bfloat16, which one fused multiply-add yields:
//     c u = p0 + p1,   c v = p2 + d      both exactly,     p3 = rn(c z + d), 2^-16 of the whole
// Five operations for two elements.  Three planes (p1 + p2 joined by a two-sum, the rest in the
// third) took twelve and 1500 cycles of a chunk more, three planes cut from float32 products took
// as many on the half-rate ALU pipe, and two planes leave a state error of 2.7e-6 instead of 4e-7.
struct Planes {
    uint32_t p[4][2][8];
};
__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t v) { return *reinterpret_cast<const __nv_bfloat162*>(&v); }
__device__ __forceinline__ uint32_t as_u32(__nv_bfloat162 v) { return *reinterpret_cast<const uint32_t*>(&v); }

struct SplitPair {
    __nv_bfloat162 u, v, z;
};
template <typename W>
__device__ __forceinline__ void decayed_planes(uint32_t tile, int j0, int s0, W weights, Planes& o) {
    const int lane = threadIdx.x & 31, rr = lane & 7;
    const uint32_t addr = tile + (j0 >> 6) * kPanel + (s0 + rr) * 128 +
                          (((((j0 & 63) >> 3) + (lane >> 3)) ^ rr) << 4);
#pragma unroll
    for (int blk = 0; blk < 4; blk++) {
        uint32_t m[4];
        ldmatrix_x4_trans(addr + blk * 1024, m[0], m[1], m[2], m[3]);
        const SplitPair w = weights(blk);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 c = as_bf162(m[i]);
            const __nv_bfloat162 p0 = __hmul2_rn(c, w.u), p2 = __hmul2_rn(c, w.v);
            const int at = 2 * blk + (i & 1);
            o.p[0][i >> 1][at] = as_u32(p0);
            o.p[1][i >> 1][at] = as_u32(__hfma2(c, w.u, __hneg2(p0)));
            o.p[2][i >> 1][at] = as_u32(p2);
            o.p[3][i >> 1][at] = as_u32(__hfma2(c, w.z, __hfma2(c, w.v, __hneg2(p2))));
        }
    }
}
__device__ __forceinline__ void store_plane(uint32_t addr, const uint32_t (&p)[2][8]) {
    tmem_st_16x128b_x4(addr, p[0]);
    tmem_st_16x128b_x4(addr + (16u << 16), p[1]);
}

// zeros into rows [n, 128) of `panels` panels of a stage
__device__ __forceinline__ void zero_rows(unsigned char* st, int panels, int n, int tid) {
#pragma unroll 1
    for (int i = tid; i < panels * (kT - n) * 8; i += kCompute) {
        const int piece = i % 8, rw = n + (i / 8) % (kT - n), pn = i / 8 / (kT - n);
        *reinterpret_cast<uint4*>(st + pn * kPanel + rw * 128 + piece * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();
}

// A row: role fastest (the roles of one head read the same tensors), then head, batch row and
// segment; `slot` is the segment's place in the order of walking.
struct Row {
    int ri, h, b, seg, slot, row_len, ntok, tok0, nchunk;
    int64_t bh;
};
__device__ __forceinline__ Row locate(const LaParams& p, int id) {
    Row k;
    k.ri = id % p.nroles;
    id /= p.nroles;
    k.h = id % p.heads;
    id /= p.heads;
    k.b = id % p.batch;
    k.seg = id / p.batch;
    k.slot = p.role[k.ri].reverse ? p.nseg - 1 - k.seg : k.seg;
    k.bh = (int64_t)k.b * p.heads + k.h;
    k.row_len = la_row_length(p, k.b);
    k.ntok = la_segment_tokens(p, k.row_len, k.seg);
    k.tok0 = k.seg * p.seglen;
    k.nchunk = (k.ntok + kT - 1) / kT;
    return k;
}

// One warp finds the range of this CTA: every row counts its chunks, at least one.
__device__ __forceinline__ Range find_range(const LaParams& p) {
    if (!p.split) {
        const int id = blockIdx.x;
        return Range{id, id, 0, 1 << 30};
    }
    const int lane = threadIdx.x & 31;
    const int pairs = p.nseg * p.batch, per = p.heads * p.nroles;   // rows of one (segment, batch row)
    auto units = [&](int i) {
        const int n = la_segment_tokens(p, la_row_length(p, i % p.batch), i / p.batch);
        return max(1, (n + kT - 1) / kT);
    };
    int64_t total = 0;
    for (int i = lane; i < pairs; i += 32) total += (int64_t)units(i) * per;
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) total += __shfl_xor_sync(0xffffffffu, total, m);
    const int64_t u0 = total * blockIdx.x / gridDim.x, u1 = total * (blockIdx.x + 1) / gridDim.x - 1;
    Range r{0, 0, 0, 0};
    int64_t base = 0;
    for (int i0 = 0; i0 < pairs; i0 += 32) {
        const int i = i0 + lane;
        const int u = i < pairs ? units(i) : 1;
        const int64_t mine = i < pairs ? (int64_t)u * per : 0;
        int64_t end = mine;
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
            const int64_t o = __shfl_up_sync(0xffffffffu, end, m);
            if (lane >= m) end += o;
        }
        const int64_t at = base + end - mine;
        const bool a = u0 >= at && u0 < at + mine, z = u1 >= at && u1 < at + mine;
        const unsigned ma = __ballot_sync(0xffffffffu, a), mz = __ballot_sync(0xffffffffu, z);
        const int ra = i * per + (int)((u0 - at) / u), ca = (int)((u0 - at) % u);
        const int rz = i * per + (int)((u1 - at) / u), cz = (int)((u1 - at) % u) + 1;
        if (ma) {
            r.row0 = __shfl_sync(0xffffffffu, ra, __ffs(ma) - 1);
            r.c0 = __shfl_sync(0xffffffffu, ca, __ffs(ma) - 1);
        }
        if (mz) {
            r.row1 = __shfl_sync(0xffffffffu, rz, __ffs(mz) - 1);
            r.c1 = __shfl_sync(0xffffffffu, cz, __ffs(mz) - 1);
        }
        base += __shfl_sync(0xffffffffu, end, 31);
    }
    return r;
}

// The rows of a range in the order of work: the last (which the next CTA may wait for), those
// between, the first.
struct Items {
    const LaParams& p;
    Range r;
    __device__ __forceinline__ int count() const { return r.row1 - r.row0 + 1; }
    __device__ __forceinline__ Row row(int i, int& c0, int& c1) const {
        const int n = count();
        const int id = i == 0 ? r.row1 : i == n - 1 ? r.row0 : r.row0 + i;
        const Row k = locate(p, id);
        c0 = id == r.row0 ? min(r.c0, k.nchunk) : 0;
        c1 = id == r.row1 ? min(r.c1, k.nchunk) : k.nchunk;
        return k;
    }
};

// first token of the chunk of step c, and its tokens
__device__ __forceinline__ int chunk_first(const Row& k, int reverse, int c) {
    return k.tok0 + (reverse ? k.nchunk - 1 - c : c) * kT;
}
__device__ __forceinline__ int chunk_count(const Row& k, int reverse, int c) {
    return min(kT, k.tok0 + k.ntok - chunk_first(k, reverse, c));
}

template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&v)[N]) {
    static_assert(N == 32 || N == 64);
    tmem_ld32(addr, reinterpret_cast<uint32_t(&)[32]>(v[0]));
    if constexpr (N == 64) tmem_ld32(addr + 32, reinterpret_cast<uint32_t(&)[32]>(v[32]));
    tmem_wait_ld();
}
template <int KB, int KC>
__global__ void __launch_bounds__(kThreads, 1) linattn_tc_kernel(const __grid_constant__ LaParams p,
                                                                 const __grid_constant__ LaMaps maps) {
    extern __shared__ __align__(1024) unsigned char smem[];
    using L = TcSmem<KB, KC>;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
    Decays& dec = *reinterpret_cast<Decays*>(smem + L::OFF_W);
    volatile int* abort = reinterpret_cast<volatile int*>(smem + L::OFF_MISC);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC + 8);
    Range* range_slot = reinterpret_cast<Range*>(smem + L::OFF_MISC + 16);
    const Waiter wait{bars, abort, p.err};
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    if ((smem_u32(smem) & 1023u) != 0) {
        if (tid == 0) *p.err = kDevErrSmemAlign;
        return;
    }
    if (warp == kWarps) tmem_alloc(tmem_slot, kTmemCols);
    if (warp == 0) {
        const Range r = find_range(p);
        if (lane == 0) *range_slot = r;
    }
    if (tid == 32) {
        for (int i = 0; i < L::STAGES; i++) {
            mbar_init(bars + kFull + i, 1);
            mbar_init(bars + kStaged + i, kWarps);
            mbar_init(bars + kFree + i, 1);
            mbar_init(bars + kUpd + i, 1);
        }
        for (int i : {kScores, kAS, kPC, kCFree, kDrain}) mbar_init(bars + i, 1);
        for (int i : {kSReady, kCReady, kPReady, kFixed, kItem}) mbar_init(bars + i, kWarps);
        abort[0] = abort[1] = 0;
        fence_mbar_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const Items items{p, *range_slot};
    const int nitems = items.count();

    if (warp >= kWarps) {
        regs_release<kRegsControl>();
        if (warp == kWarps + 1 && elect_one()) {
            // ---- loads --------------------------------------------------------------------------
            int it = 0, begun = 0;
            uint32_t was_over_a = 0;                  // by stage
            bool fine = !p.test_withhold;
            for (int n = 0; n < nitems && fine; n++) {
                int c0, c1;
                const Row k = items.row(n, c0, c1);
                const LaRole& r = p.role[k.ri];
                const int ha = k.h / r.a.share, hb = k.h / r.b.share, hc = k.h / r.c.share;
                // an output tile over a alone leaves b and c free once the products have read them
                const uint32_t over_a = !L::TWO && KC <= KB && r.out_vec && !r.out_f32;
                for (int c = c0; c < c1; c++, it++) {
                    const int sg = it % L::STAGES;
                    const uint32_t last = (it / L::STAGES - 1) & 1, early = (was_over_a >> sg) & 1;
                    if (it >= L::STAGES && !(fine = wait((early ? kUpd : kFree) + sg, last))) break;
                    was_over_a = (was_over_a & ~(1u << sg)) | over_a << sg;
                    unsigned char* st = smem + sg * L::STAGE;
                    uint64_t* bar = bars + kFull + sg;
                    const int t = chunk_first(k, r.reverse, c);
                    mbar_arrive_expect_tx(bar, L::STAGE);
#pragma unroll
                    for (int i = 0; i < KB / 64; i++)
                        tma_load_4d(st + L::A + i * kPanel, &maps.b[k.ri], bar, i * 64, t, hb, k.b);
#pragma unroll
                    for (int i = 0; i < KC / 64; i++)
                        tma_load_4d(st + 2 * L::A + i * kPanel, &maps.c[k.ri], bar, i * 64, t, hc, k.b);
                    begun = it + 1;
                    if (early && !(fine = wait(kFree + sg, last))) break;
#pragma unroll
                    for (int i = 0; i < KB / 64; i++)
                        tma_load_4d(st + i * kPanel, &maps.a[k.ri], bar, i * 64, t, ha, k.b);
                }
            }
            if (!fine)       // copies in flight still write to this CTA's shared memory
                for (int i = max(0, begun - L::STAGES); i < begun; i++)
                    mbar_wait_bounded(bars + kFull + i % L::STAGES, (i / L::STAGES) & 1);
        } else if (warp == kWarps + 2 && elect_one()) {
            // ---- stores -------------------------------------------------------------------------
            int it = 0;
            bool fine = true;
            for (int n = 0; n < nitems && fine; n++) {
                int c0, c1;
                const Row k = items.row(n, c0, c1);
                const LaRole& r = p.role[k.ri];
                for (int c = c0; c < c1; c++, it++) {
                    const int sg = it % L::STAGES;
                    const uint32_t turn = (it / L::STAGES) & 1;
                    if (!(fine = wait(kStaged + sg, turn))) break;
                    if (r.out_vec) {
                        const int t = chunk_first(k, r.reverse, c), width = r.out_f32 ? 32 : 64;   // channels of a panel
                        const unsigned char* src = smem + sg * L::STAGE;
                        for (int x = 0; x < r.dc; x += width, src += kPanel)
                            tma_store_4d(&maps.o[k.ri], src, x, t, k.h, k.b);
                        tma_store_commit();
                        tma_store_wait_read_all();
                    }
                    if (!(fine = wait(kUpd + sg, turn))) break;    // the last product to read the stage
                    mbar_arrive(bars + kFree + sg);
                }
            }
            tma_store_wait_all();
        } else if (warp == kWarps && elect_one()) {
            // ---- products -----------------------------------------------------------------------
            constexpr uint32_t id_scores = umma_idesc(128, 128, false), id_as = umma_idesc(128, KC, false),
                               id_pc = umma_idesc(128, KC, true), id_upd = umma_idesc(128, KB, true);
            const uint32_t s_desc = umma_desc_lo(smem_u32(smem + L::OFF_S), 16);
            int it = 0, fixed = 0;
            bool fine = true;
            for (int n = 0; n < nitems && fine; n++) {
                int c0, c1;
                const Row k = items.row(n, c0, c1);
                const int reverse = p.role[k.ri].reverse;
                for (int c = c0; c < c1; c++, it++) {
                    const int sg = it % L::STAGES;
                    const uint32_t st = smem_u32(smem + sg * L::STAGE), par = it & 1;
                    if (!(fine = wait(kFull + sg, (it / L::STAGES) & 1))) break;
                    if (chunk_count(k, reverse, c) < kT && !(fine = wait(kFixed, fixed++ & 1))) break;
                    if (it > 0 && !(fine = wait(kPC, par ^ 1))) break;       // the last P has been read
                    tc_fence_after();
                    // K-major panels of 64 channels: 16 channels are 32 bytes
                    const uint32_t a_desc = umma_desc_lo(st, 16), b_desc = umma_desc_lo(st + L::A, 16);
#pragma unroll
                    for (int i = 0; i < KB / 16; i++) {
                        const uint32_t off = ((i >> 2) * kPanel + (i & 3) * 32) >> 4;
                        umma_ss(tmem + kColScores, a_desc + off, b_desc + off, id_scores, i > 0);
                    }
                    umma_commit(bars + kScores);
                    if (!(fine = wait(kSReady, L::BOTH ? par : 0))) break;
                    if (it > 0 && !(fine = wait(kStaged + (it - 1) % L::STAGES, ((it - 1) / L::STAGES) & 1))) break;   // O has been read
                    tc_fence_after();
                    auto a_s = [&](uint32_t half_desc, bool first) {
#pragma unroll
                        for (int i = 0; i < (L::TWO ? 2 : 1) * KB / 16; i++)
                            umma_ss(tmem + kColO, a_desc + (((L::TWO ? 0 : i >> 2) * kPanel + (i & 3) * 32) >> 4),
                                    half_desc + (((i >> 2) * (KC * 128) + (i & 3) * 32) >> 4), id_as, !first || i > 0);
                    };
                    if constexpr (L::BOTH) {
#pragma unroll 1
                        for (int e = 0; e < 2; e++) a_s(s_desc + e * (L::S1 >> 4), e == 0);
                    } else {
                        a_s(s_desc, true);
                        umma_commit(bars + kAS);
                        if (!(fine = wait(kSReady, 1))) break;
                        tc_fence_after();
                        a_s(s_desc, false);
                    }
                    umma_commit(bars + kAS);
                    // N-major panels of 64 channels: 16 tokens are 2048 bytes
                    const uint32_t bn_desc = umma_desc_lo(st + L::A, kPanel), cn_desc = umma_desc_lo(st + 2 * L::A, kPanel);
                    if (!(fine = wait(kCReady, L::TWO ? par : 0))) break;
                    tc_fence_after();
#pragma unroll
                    for (int i = 0; i < 16; i++)               // the smallest plane first
                        umma_ts(tmem + kColU, tmem + kColC + i * 8, bn_desc + (i & 3) * (2048 >> 4), id_upd, i > 0);
                    if constexpr (L::TWO) {
                        // lanes 0-63 and 64-127 each hold the channels for one half of the tokens; what the
                        // other half's columns get of them is not read
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            umma_ts(tmem + kColU + 64, tmem + kColC + i * 8, bn_desc + (4 + (i & 3)) * (2048 >> 4), id_upd,
                                    i > 0);
                        umma_commit(bars + kUpd + sg);
                    } else {
                        umma_commit(bars + kCFree);
                    }
                    if (!(fine = wait(kPReady, par))) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int e = 0; e < 2; e++)                // the lower half first
#pragma unroll
                        for (int i = 0; i < kT / 16; i++)
                            umma_ts(tmem + kColO, tmem + kColScores + (16 - e * 16) + (i >> 1) * 32 + (i & 1) * 8,
                                    cn_desc + i * (2048 >> 4), id_pc, e > 0 || i > 0);
                    umma_commit(bars + kPC);
                    if constexpr (!L::TWO) {
                        if (!(fine = wait(kCReady, 1))) break;
                        tc_fence_after();
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            umma_ts(tmem + kColU, tmem + kColC + i * 8, bn_desc + (4 + (i & 3)) * (2048 >> 4), id_upd, true);
                        umma_commit(bars + kUpd + sg);
                    }
                }
            }
            if (!fine) {
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
        const int row = q * 32 + lane;                // token of P and O
        constexpr int NS = KB / 2;                    // columns of S^T per thread
        constexpr int NO = KC / 2;                    // columns of O per thread
        const int part = L::TWO ? q >> 1 : 0;         // of the state
        const int sq = L::TWO ? q & 1 : q, srow = sq * 32 + lane;     // rows of S^T: channels of c
        const bool s_on = sq * 32 < KC;               // S^T has KC rows
        const int i0 = half * NS, o0 = half * NO;
        const uint32_t ucol = kColU + part * 64 + i0;
        auto arrive = [&](int bar) {
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + bar);
        };
        auto await = [&](int bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
        int it = 0, fixed = 0, meets = 0;
        // every compute warp has come this far
        auto meet = [&]() {
            arrive(kItem);
            return await(kItem, meets++ & 1);
        };
        bool fine = true;

        for (int item = 0; item < nitems; item++) {
            int c0, c1;
            const Row k = items.row(item, c0, c1);
            const LaRole& r = p.role[k.ri];
            const int reverse = r.reverse;
            const float g2 = la_log2_decay(p.log_decay[k.h]);
            if (!(fine = meet())) break;              // nobody reads the last row's tables any more
            fill_decays(dec, g2, r.alpha, r.sigma, reverse, k.nchunk > 0 ? k.ntok - (k.nchunk - 1) * kT : 0);

            // S^T before chunk c0: the state that the CTA before this one has published, or the one that the
            // scan has left for the segment, or the initial state.  Through TMEM, so that the loop over columns
            // stays a loop (registers have no index).
            if (c0 > 0) {
                const int* flag = p.flags + blockIdx.x;
                int there = 0;
                const long long start = clock64();
                if (tid == 0) abort[1] = 1;
                while (true) {
                    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(there) : "l"(flag) : "memory");
                    if (there || wait.gone(start, c0)) break;
                }
                if (tid == 0) abort[1] = 0;
                if (!(fine = __all_sync(0xffffffffu, there != 0))) break;
            }
            float s[NS];
            if (s_on) {
                const float* src = nullptr;
                int64_t step = r.s_i;
                if (part == 1) {
                    // the second part starts from zero
                } else if (c0 > 0) {
                    src = p.handoff + (int64_t)blockIdx.x * KB * KC + srow;
                    step = KC;
                } else if (srow < r.dc && p.nseg > 1) {
                    src = r.seg + (k.bh * p.nseg + k.seg) * r.db * r.dc + srow;
                    step = r.dc;
                } else if (srow < r.dc && r.state0) {
                    src = r.state0 + k.bh * r.db * r.dc + srow * r.s_j;
                }
                const int cols = c0 > 0 ? KB : r.db;
                // 32 loads at a time: they are what a row's start waits for
#pragma unroll 1
                for (int i = 0; i < NS; i += 32) {
                    uint32_t v[32];
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        v[e] = src && i0 + i + e < cols ? __float_as_uint(__ldcg(src + (i0 + i + e) * step)) : 0u;
                    tmem_st32(tm + ucol + i, v);
                }
                tmem_wait_st();
                uint32_t v[NS];
                tmem_ld<NS>(tm + ucol, v);
#pragma unroll
                for (int e = 0; e < NS; e++) s[e] = __uint_as_float(v[e]);
            }
            // a half of S^T to shared memory for A S
            auto put_half = [&](bool upper, int at) {
                if (s_on) {
#pragma unroll
                    for (int i = 0; i < NS; i += 8) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            w[e] = upper ? upper_bf16(s[i + 2 * e], s[i + 2 * e + 1]) : lower_bf16(s[i + 2 * e], s[i + 2 * e + 1]);
                        const int ii = i0 + i;
                        *reinterpret_cast<uint4*>(smem + L::OFF_S + at + ((ii >> 6) + part) * (KC * 128) +
                                                  swz128(srow, (ii & 63) * 2)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            };
            auto hand_state = [&]() {
                fence_proxy_async_smem();
                tc_fence_before();
                arrive(kSReady);
            };
            auto put_state = [&]() {
                put_half(true, 0);
                if constexpr (L::BOTH) put_half(false, L::S1);
                hand_state();
            };
            if (c0 < c1) put_state();
            if (!(fine = meet())) break;              // the tables are there

            for (int c = c0; c < c1; c++, it++) {
                const uint32_t par = it & 1, turn = (it / L::STAGES) & 1;
                const int sg = it % L::STAGES;
                const int n = chunk_count(k, reverse, c);
                unsigned char* st = smem + sg * L::STAGE;
                if (!(fine = await(kFull + sg, turn))) break;
                if (n < kT) {
                    // rows past the length hold whatever the caller's padding holds
                    zero_rows(st, L::STAGE / kPanel, n, tid);
                    arrive(kFixed);
                    if (!(fine = await(kFixed, fixed++ & 1))) break;
                }
                // planes of C'^T, 64 tokens at a time (of two parts: all at once), of which this warp does 32
                auto put_planes = [&](int sub) {
                    if (s_on) {
                        const __nv_bfloat16(*wt)[kT] = dec.plane[n < kT];
                        const int s0 = sub * 64 + half * 32;
                        Planes pl;
                        decayed_planes(smem_u32(st + 2 * L::A), sq * 32, s0, [&](int e) {
                            const int at = s0 + 8 * e + 2 * (lane & 3);
                            return SplitPair{*reinterpret_cast<const __nv_bfloat162*>(&wt[0][at]),
                                             *reinterpret_cast<const __nv_bfloat162*>(&wt[1][at]),
                                             *reinterpret_cast<const __nv_bfloat162*>(&wt[2][at])};
                        }, pl);
#pragma unroll
                        for (int e = 0; e < 4; e++) store_plane(tm + kColC + e * 32 + half * 16, pl.p[3 - e]);
                        tmem_wait_st();
                    }
                    tc_fence_before();
                    arrive(kCReady);
                };
                put_planes(part);
                if constexpr (!L::BOTH) {
                    if (!(fine = await(kAS, 0))) break;        // the product with the upper half has read it
                    put_half(false, 0);
                    hand_state();
                }

                // P in blocks of 32 x 32, which the mask empties, halves or leaves whole; rolled, since with the lower
                // halves a second copy of it misses the instruction cache (prompts below: 124 us instead of 117)
                if (!(fine = await(kScores, par))) break;
                tc_fence_after();
#pragma unroll 1
                for (int i = 0; i < 2; i++) {
                    const int sb = half * 2 + i;
                    uint32_t o[32];                            // upper halves, lower halves
                    auto put = [&](int e, float x, float y) {
                        o[e / 2] = upper_bf16(x, y);
                        o[16 + e / 2] = lower_bf16(x, y);
                    };
                    if (reverse ? sb >= q : sb <= q) {
                        uint32_t v[32];
                        tmem_ld<32>(tm + kColScores + sb * 32, v);
                        if (sb != q) {
                            // w^|t - s| as two factors, neither above one: up to the block's edge and inside it
                            const float f = dec.score[reverse ? sb * 32 - row : kT - 1 - row + sb * 32 + 31];
                            const float2 f2 = make_float2(f, f);
#pragma unroll
                            for (int e = 0; e < 32; e += 4) {
                                const float4 wb = lds128(dec.block + e);
                                const float2 x = __fmul2_rn(make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])),
                                                            __fmul2_rn(f2, make_float2(wb.x, wb.y)));
                                const float2 y = __fmul2_rn(make_float2(__uint_as_float(v[e + 2]), __uint_as_float(v[e + 3])),
                                                            __fmul2_rn(f2, make_float2(wb.z, wb.w)));
                                put(e, x.x, x.y);
                                put(e + 2, y.x, y.y);
                            }
                        } else {
                            // the table runs with the columns: its entry for column e of the block is wt[e]
                            const float* wt = dec.score + (reverse ? sb * 32 - row : kT - 1 - row + sb * 32);
                            const uint32_t live = reverse ? ~0u << lane : ~0u >> (31 - lane);
#pragma unroll
                            for (int e = 0; e < 32; e += 2) {
                                const float x = __uint_as_float(v[e]) * wt[e], y = __uint_as_float(v[e + 1]) * wt[e + 1];
                                put(e, live & (1u << e) ? x : 0.f, live & (2u << e) ? y : 0.f);
                            }
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = 0;
                    }
                    // over scores that this thread alone reads, and has read
                    tmem_st32(tm + kColScores + sb * 32, o);
                }
                // A S leaves TMEM
                if (!(fine = await(kAS, L::BOTH ? par : 1))) break;
                tc_fence_after();
                uint32_t as[NO];
                tmem_ld<NO>(tm + kColO + o0, as);
                tmem_wait_st();
                tc_fence_before();
                arrive(kPReady);

                if constexpr (!L::TWO) {
                    if (!(fine = await(kCFree, par))) break;
                    tc_fence_after();
                    put_planes(1);
                }

                // O
                if (!(fine = await(kPC, par))) break;
                tc_fence_after();
                float acc[NO];
                {
                    const float f = r.beta * dec.pow[reverse ? max(n - 1 - row, 0) : row + 1];
                    uint32_t v[NO];
                    tmem_ld<NO>(tm + kColO + o0, v);
#pragma unroll
                    for (int e = 0; e < NO; e += 2) {
                        const float2 x = __ffma2_rn(make_float2(f, f), make_float2(__uint_as_float(as[e]), __uint_as_float(as[e + 1])),
                                                    make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])));
                        acc[e] = x.x;
                        acc[e + 1] = x.y;
                    }
                    if (n < kT && row >= n)
#pragma unroll
                        for (int e = 0; e < NO; e++) acc[e] = 0.f;
                }
                // the tile is staged over a, and where that is not enough over b and c, which the update reads
                const bool bf16 = r.out_vec && !r.out_f32;
                if ((!bf16 || KC > KB) && !(fine = await(kUpd + sg, turn))) break;
                if (bf16) {
#pragma unroll
                    for (int i = 0; i < NO; i += 8) {
                        const uint4 v = make_uint4(pack_bf16(acc[i], acc[i + 1]), pack_bf16(acc[i + 2], acc[i + 3]),
                                                   pack_bf16(acc[i + 4], acc[i + 5]), pack_bf16(acc[i + 6], acc[i + 7]));
                        const int oc = o0 + i;
                        *reinterpret_cast<uint4*>(st + (oc >> 6) * kPanel + swz128(row, (oc & 63) * 2)) = v;
                    }
                } else {
                    // float32: panels of 32 channels, for a TMA or for the loop below
#pragma unroll
                    for (int i = 0; i < NO; i += 4) {
                        const int oc = o0 + i;
                        *reinterpret_cast<float4*>(st + (oc >> 5) * kPanel + swz128(row, (oc & 31) * 4)) =
                            make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
                    }
                }
                if (!r.out_vec) {
                    // rows that a TMA cannot store: a warp's 32 rows, one after the other
                    __syncwarp();
                    const int64_t at = k.b * r.o_sb + (int64_t)(chunk_first(k, reverse, c) + q * 32) * r.o_st +
                                       k.h * r.o_sh + o0;
                    const int cols = min(NO, r.dc - o0), rows = min(32, n - q * 32);
#pragma unroll 1
                    for (int rw = 0; rw < rows; rw++) {
#pragma unroll
                        for (int e = 0; e < NO; e += 32) {
                            const int oc = o0 + e + lane;
                            const float x = *reinterpret_cast<const float*>(st + (oc >> 5) * kPanel +
                                                                            swz128(q * 32 + rw, (oc & 31) * 4));
                            if (e + lane >= cols) continue;
                            if (r.out_f32) static_cast<float*>(r.out)[at + rw * r.o_st + e + lane] = x;
                            else static_cast<__nv_bfloat16*>(r.out)[at + rw * r.o_st + e + lane] = __float2bfloat16_rn(x);
                        }
                    }
                }
                fence_proxy_async_smem();
                tc_fence_before();
                arrive(kStaged + sg);

                // the state after this chunk
                if (!(fine = await(kUpd + sg, turn))) break;
                tc_fence_after();
                if (s_on) {
                    const float fn = dec.pow[n];
                    uint32_t v[NS];
                    tmem_ld<NS>(tm + ucol, v);
#pragma unroll
                    for (int e = 0; e < NS; e += 2) {
                        const float2 x = __ffma2_rn(make_float2(fn, fn), make_float2(s[e], s[e + 1]),
                                                    make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])));
                        s[e] = x.x;
                        s[e + 1] = x.y;
                    }
                }
                if (c + 1 < c1) put_state();
            }
            if (!fine) break;

            // the state goes to the CTA that continues the row, or out
            const bool ends = c1 == k.nchunk;
            const bool out = ends && k.slot == p.nseg - 1 && r.state_out;
            if (!ends || out) {
                if constexpr (L::TWO) {
                    // the parts are joined through the place of their copies, which no product reads any more
                    float* other = reinterpret_cast<float*>(smem + L::OFF_S) + srow;
                    if (part == 1)
#pragma unroll
                        for (int e = 0; e < NS; e++) other[(i0 + e) * KC] = s[e];
                    if (!(fine = meet())) break;
                    if (part == 0)
#pragma unroll
                        for (int e = 0; e < NS; e++) s[e] += other[(i0 + e) * KC];
                }
                if (s_on && part == 0) {
#pragma unroll
                    for (int i = 0; i < NS; i += 32) {
                        uint32_t v[32];
#pragma unroll
                        for (int e = 0; e < 32; e++) v[e] = __float_as_uint(s[i + e]);
                        tmem_st32(tm + ucol + i, v);
                    }
                    tmem_wait_st();
                    float* dst = ends ? r.state_out + k.bh * r.db * r.dc + srow * r.s_j
                                      : p.handoff + (int64_t)(blockIdx.x + 1) * KB * KC + srow;
                    const int64_t step = ends ? r.s_i : KC;
                    const int rows = ends ? r.dc : KC, cols = ends ? r.db : KB;
#pragma unroll 1
                    for (int i = 0; i < NS; i += 8) {
                        uint32_t u[8];
                        tmem_ld8(tm + ucol + i, u);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            if (srow < rows && i0 + i + e < cols) dst[(i0 + i + e) * step] = __uint_as_float(u[e]);
                    }
                }
                if (!ends) {
                    __threadfence();
                    if (!(fine = meet())) break;
                    if (tid == 0)
                        asm volatile("st.release.gpu.global.s32 [%0], %1;" ::"l"(p.flags + blockIdx.x + 1), "r"(1)
                                     : "memory");
                }
            }
            if (ends) {
                // zeros for the tokens past the row's length, 16 bytes at a time where the rows allow it
                const int es = r.out_f32 ? 4 : 2;
                const int piece = r.out_vec && r.dc * es % 16 == 0 ? 16 : es, per = r.dc * es / piece;
                const int end = min(p.seglen, p.seqlen - k.tok0);
                // so many tokens at a time that their pieces count in 32 bits
                constexpr int kFill = 1 << 20;
#pragma unroll 1
                for (int t = k.ntok; t < end; t += kFill) {
                    const int total = min(kFill, end - t) * per;
                    char* dst = static_cast<char*>(r.out) + (k.b * r.o_sb + (int64_t)(k.tok0 + t) * r.o_st + k.h * r.o_sh) * es;
#pragma unroll 1
                    for (int i = tid; i < total; i += kCompute) {
                        char* at = dst + (int64_t)(i / per) * r.o_st * es + i % per * piece;
                        if (piece == 16) *reinterpret_cast<uint4*>(at) = make_uint4(0, 0, 0, 0);
                        else if (piece == 4) *reinterpret_cast<float*>(at) = 0.f;
                        else *reinterpret_cast<__nv_bfloat16*>(at) = __float2bfloat16_rn(0.f);
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kWarps) tmem_dealloc(tmem, kTmemCols);
}

// The state a segment reaches from a zero start: only U, with every token weighted towards the
// segment's end, so that the sum needs no rescaling between chunks, and chunks whose every weight
// is zero in float32 are not read.  The tensor core cuts its sums off, so U starts from zero for each chunk,
// in one of two places by turns, and is added to the sum in registers, rounded, while the next one is formed
// (summed in the unit over 128 chunks of k and v with means of one, the state was 4.9e-5 off).  C'^T has two
// buffers of 64 tokens; the threads fill one while the product reads the other, and bound it (42 rows of 8
// segments of 20 chunks, 128 channels: 95 us, 65 at HBM's rate).
constexpr int kStages = 3;
constexpr int kStateThreads = (kWarps + 2) * 32;
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
// TMEM columns: U of even and of odd chunks, and from 128 on the planes of two buffers
constexpr uint32_t kColEven = 0, kColOdd = 384;
enum StateBar { kSbFull = 0, kSbFree = 3, kSbReady = 6, kSbDone = 8, kSbFixed = 10, kSbDrain = 11 };

template <int KB, int KC>
__global__ void __launch_bounds__(kStateThreads, 1) linattn_tc_state_kernel(const __grid_constant__ LaParams p,
                                                                            const __grid_constant__ LaMaps maps) {
    extern __shared__ __align__(1024) unsigned char smem[];
    using L = StateSmem<KB, KC>;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
    Decays& dec = *reinterpret_cast<Decays*>(smem + L::OFF_W);
    volatile int* abort = reinterpret_cast<volatile int*>(smem + L::OFF_MISC);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC + 8);
    const Waiter wait{bars, abort, p.err};

    // the last segment in the order of walking feeds nobody: segments 0 .. nseg - 2, or 1 .. reversed
    Row k = locate(p, blockIdx.x);
    const LaRole& r = p.role[k.ri];
    const int reverse = r.reverse;
    if (reverse) k = locate(p, blockIdx.x + p.nroles * p.heads * p.batch);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float g2 = la_log2_decay(p.log_decay[k.h]);
    auto first = [&](int c) { return k.tok0 + c * kT; };
    auto count = [&](int c) { return min(kT, k.ntok - c * kT); };
    // tokens between a chunk and the end of the walk: later ones, or earlier ones in reverse
    auto far = [&](int c) { return reverse ? c * kT : k.ntok - c * kT - count(c); };
    int cb = 0, ce = k.nchunk;                // chunks with a weight that is not zero
    while (cb < ce && !reverse && g2 * (float)far(cb) < kZeroLog2) cb++;
    while (cb < ce && reverse && g2 * (float)far(ce - 1) < kZeroLog2) ce--;
    const int nchunk = ce - cb;

    if ((smem_u32(smem) & 1023u) != 0) {
        if (tid == 0) *p.err = kDevErrSmemAlign;
        return;
    }
    if (warp == kWarps) tmem_alloc(tmem_slot, kTmemCols);
    if (tid == 0) {
        for (int i = 0; i < kStages; i++) {
            mbar_init(bars + kSbFull + i, 1);
            mbar_init(bars + kSbFree + i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(bars + kSbReady + i, kWarps);
            mbar_init(bars + kSbDone + i, 1);
        }
        mbar_init(bars + kSbFixed, kWarps);
        mbar_init(bars + kSbDrain, 1);
        abort[0] = abort[1] = 0;
        fence_mbar_init();
    }
    fill_decays(dec, g2, r.alpha, r.sigma, reverse, k.nchunk > 0 ? k.ntok - (k.nchunk - 1) * kT : 0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == kWarps + 1) {
        if (elect_one()) {
            const int hb = k.h / r.b.share, hc = k.h / r.c.share;
            bool fine = true;
            int i = 0;
            for (; i < nchunk; i++) {
                if (i >= kStages && !(fine = wait(kSbFree + i % kStages, (i / kStages - 1) & 1))) break;
                unsigned char* st = smem + (i % kStages) * L::STAGE;
                uint64_t* bar = bars + kSbFull + i % kStages;
                mbar_arrive_expect_tx(bar, L::STAGE);
#pragma unroll
                for (int n = 0; n < KB / 64; n++)
                    tma_load_4d(st + n * kPanel, &maps.b[k.ri], bar, n * 64, first(cb + i), hb, k.b);
#pragma unroll
                for (int n = 0; n < KC / 64; n++)
                    tma_load_4d(st + L::B + n * kPanel, &maps.c[k.ri], bar, n * 64, first(cb + i), hc, k.b);
            }
            if (!fine)
                for (int n = max(0, i - kStages); n < i; n++)
                    mbar_wait_bounded(bars + kSbFull + n % kStages, (n / kStages) & 1);
        }
        __syncwarp();
    } else if (warp == kWarps) {
        if (elect_one()) {
            constexpr uint32_t id_upd = umma_idesc(128, KB, true);
            bool fine = true;
            for (int i = 0; i < nchunk; i++) {
                if (!(fine = wait(kSbFull + i % kStages, (i / kStages) & 1))) break;
                const uint32_t bn_desc = umma_desc_lo(smem_u32(smem + (i % kStages) * L::STAGE), kPanel);
#pragma unroll 1
                for (int e = 0; e < 2; e++) {
                    if (!(fine = wait(kSbReady + e, i & 1))) break;
                    tc_fence_after();
#pragma unroll
                    for (int m = 0; m < 16; m++)               // the smallest plane first
                        umma_ts(tmem + (i & 1 ? kColOdd : kColEven), tmem + 128 + e * 128 + m * 8,
                                bn_desc + (e * 4 + (m & 3)) * (2048 >> 4), id_upd, e > 0 || m > 0);
                    umma_commit(bars + kSbDone + e);
                }
                if (!fine) break;
                umma_commit(bars + kSbFree + i % kStages);
            }
            if (!fine) {
                umma_commit(bars + kSbDrain);
                mbar_wait_bounded(bars + kSbDrain, 0);
            }
        }
        __syncwarp();
    } else {
        const int q = warp & 3, half = warp >> 2;
        const uint32_t tm = tmem + ((uint32_t)(q * 32) << 16);
        const int row = q * 32 + lane;
        const bool s_on = q * 32 < KC;
        auto arrive = [&](int bar) {
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + bar);
        };
        auto await = [&](int bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
        bool fine = true;
        constexpr int NS = KB / 2;
        float s[NS] = {};
        auto add = [&](int i) {               // U of chunk i
            if (!s_on) return;
            uint32_t v[NS];
            tmem_ld<NS>(tm + (i & 1 ? kColOdd : kColEven) + half * NS, v);
#pragma unroll
            for (int u = 0; u < NS; u++) s[u] += __uint_as_float(v[u]);
        };
        for (int i = 0; i < nchunk; i++) {
            const int c = cb + i, n = count(c);
            unsigned char* st = smem + (i % kStages) * L::STAGE;
            if (!(fine = await(kSbFull + i % kStages, (i / kStages) & 1))) break;
            if (n < kT) {
                zero_rows(st, L::STAGE / kPanel, n, tid);
                arrive(kSbFixed);
                if (!(fine = await(kSbFixed, 0))) break;
            }
            const float f = r.sigma * exp2f(g2 * (float)far(c));
#pragma unroll 1
            for (int e = 0; e < 2; e++) {
                const int s0 = e * 64 + half * 32;
                Planes pl;
                if (s_on)
                    decayed_planes(smem_u32(st + L::B), q * 32, s0, [&](int b) {
                        const int at = s0 + 8 * b + 2 * (lane & 3);
                        float x = f * dec.pow[reverse ? at + 1 : max(n - 1 - at, 0)];
                        float y = f * dec.pow[reverse ? at + 2 : max(n - 2 - at, 0)];
                        x = at < n ? x : 0.f;
                        y = at + 1 < n ? y : 0.f;
                        SplitPair w;
                        w.u = __floats2bfloat162_rn(x, y);
                        x -= __low2float(w.u);
                        y -= __high2float(w.u);
                        w.v = __floats2bfloat162_rn(x, y);
                        w.z = __floats2bfloat162_rn(x - __low2float(w.v), y - __high2float(w.v));
                        return w;
                    }, pl);
                if (i > 0 && !(fine = await(kSbDone + e, (i - 1) & 1))) break;   // the buffer is free
                tc_fence_after();
                if (s_on) {
#pragma unroll
                    for (int u = 0; u < 4; u++) store_plane(tm + 128 + e * 128 + u * 32 + half * 16, pl.p[3 - u]);
                    tmem_wait_st();
                }
                tc_fence_before();
                arrive(kSbReady + e);
            }
            if (!fine) break;
            if (i > 0) add(i - 1);            // complete: the second buffer's last use has ended
        }
        if (fine && nchunk > 0) fine = await(kSbDone + 1, (nchunk - 1) & 1);
        tc_fence_after();
        if (fine && s_on) {
            if (nchunk > 0) add(nchunk - 1);
            float* e = r.seg + (k.bh * p.nseg + k.seg) * r.db * r.dc + row;
#pragma unroll
            for (int u = 0; u < NS; u++)
                if (row < r.dc && half * NS + u < r.db) e[(half * NS + u) * r.dc] = s[u];
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kWarps) tmem_dealloc(tmem, kTmemCols);
}

template <int KB, int KC>
cudaError_t launch_tc(const LaParams& p, const LaMaps& maps, int sms, cudaStream_t stream) {
    const int64_t rows = (int64_t)p.batch * p.heads * p.nroles;
    cudaError_t e;
    if (p.nseg > 1) {
        e = cudaFuncSetAttribute(linattn_tc_state_kernel<KB, KC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 StateSmem<KB, KC>::BYTES);
        if (e != cudaSuccess) return e;
        linattn_tc_state_kernel<KB, KC><<<(unsigned)(rows * (p.nseg - 1)), kStateThreads, StateSmem<KB, KC>::BYTES, stream>>>(p, maps);
        if ((e = cudaGetLastError()) != cudaSuccess || (e = launch_linattn_scan(p, stream)) != cudaSuccess) return e;
    }
    e = cudaFuncSetAttribute(linattn_tc_kernel<KB, KC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             TcSmem<KB, KC>::BYTES);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.split ? sms : rows * p.nseg));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = TcSmem<KB, KC>::BYTES;
    cfg.stream = stream;
    // a CTA may wait for the one before it: all of them are resident at once
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeCooperative;
    attr.val.cooperative = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = p.split ? 1 : 0;
    if (p.split && (e = cudaMemsetAsync(p.flags, 0, (size_t)(sms + 1) * sizeof(int), stream)) != cudaSuccess) return e;
    return cudaLaunchKernelEx(&cfg, linattn_tc_kernel<KB, KC>, p, maps);
}

}  // namespace

// Every role of p has db <= kb and dc <= kc (64 or 128).
cudaError_t launch_linattn_tc(const LaParams& p, const LaMaps& maps, int kb, int kc, int sms, cudaStream_t stream) {
    if (kb == 64) return kc == 64 ? launch_tc<64, 64>(p, maps, sms, stream) : launch_tc<64, 128>(p, maps, sms, stream);
    return kc == 64 ? launch_tc<128, 64>(p, maps, sms, stream) : launch_tc<128, 128>(p, maps, sms, stream);
}

}  // namespace ssm
