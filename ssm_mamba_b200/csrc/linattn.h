// Kernel parameter blocks of linear attention with a decay for each head (linattn_*.cu).
// Built by capi.cu from the C-ABI argument struct after validation; strides are in elements.
#pragma once

#include <cuda.h>
#include <stdint.h>

namespace ssm {

// A (batch, token, head, channel) tensor with unit channel stride.  Head h of the operator
// reads head h / share of the tensor.
struct LaTensor {
    const void* p;
    int64_t sb, st, sh;
    int share;
    int vec;             // 1: base and strides are multiples of 16 bytes
};

// The forward and the three products of the backward are one recurrence with its operands in
// other places.  With w = exp(log_decay[h]), one role computes for every token t
//     out_t = alpha sum_{s <= t} w^(t-s) (a_t . b_s) c_s  +  beta w^(t+1) a_t^T S
//     S'    = w^n S + sigma sum_s w^(n-1-s) b_s c_s^T             (n tokens from state S)
// or, with `reverse`, the same over s >= t from the last token to the first, the state being
// kept already decayed across the next step:
//     out_t = alpha sum_{s >= t} w^(s-t) (a_t . b_s) c_s  +  beta w^(n-1-t) a_t^T S
//     S'    = w^n S + sigma sum_s w^(s+1) b_s c_s^T
//   forward  a, b, c = q, k, v       S = state                 out
//   dq       a, b, c = dout, v, k    S = state^T
//   dv       a, b, c = k, q, dout    S = state gradient        (reverse)
//   dk       a, b, c = v, dout, q    S = state gradient^T      (reverse)
struct LaRole {
    LaTensor a, b, c;
    void* out; int64_t o_sb, o_st, o_sh;
    int out_f32;          // out is float32 (float32 streams, per-head partials)
    int out_vec;          // out's rows start on 16 bytes and its strides fit a TMA
    int db, dc;           // channels of a and b; channels of c and out
    int reverse;
    float alpha, beta, sigma;
    const float* state0;  // may be null (zero); element (i, j) of head (b, h) at
    float* state_out;     //   (b * heads + h) * db * dc + i * s_i + j * s_j; may be null
    int s_i, s_j;
    float* seg;           // per-segment states (batch * heads, nseg, db, dc), null when nseg == 1
};

struct LaParams {
    int batch, seqlen, heads;
    int nroles;
    int nseg, seglen;     // tokens [s * seglen, (s + 1) * seglen) form segment s
    const float* log_decay;
    const int64_t* length;  // may be null
    int* err;             // device error word
    int test_withhold;    // test hook: no loads are issued, so that the waits for them run out
    // tensor-core kernel: the CTAs share the chunks of all rows evenly (more rows than CTAs), and a row
    // that two CTAs share passes its state through handoff, one state and one flag per CTA
    int split;
    int* flags;
    float* handoff;
    LaRole role[3];
};

// TMA maps of every role's tensors: (channel, token, head, batch), boxes of 128 bytes x 128 tokens
struct LaMaps {
    CUtensorMap a[3], b[3], c[3], o[3];
};

// out[b, t, g, :] = sum of the share heads of src (batch, seqlen, heads, d) float32
struct LaGroupParams {
    const float* src;
    void* out; int64_t o_sb, o_st, o_sh;
    int batch, seqlen, heads, d, share;
    int tokens;          // of a CTA; set by the launch
};

// A bfloat16 tensor copied to rows of 8 ceil(d / 8) channels, contiguous
struct LaPackParams {
    const void* src; int64_t sb, st, sh;
    void* dst;
    int batch, seqlen, heads, d;
};

// One token: state = w state + k v^T in place, out = scale q^T state.
struct LaUpdParams {
    int batch, heads, dk, dv;
    float scale;
    const void* q; int64_t q_sb, q_sh; int q_share;
    const void* k; int64_t k_sb, k_sh; int k_share;
    const void* v; int64_t v_sb, v_sh; int v_share;
    const float* log_decay;
    float* state; int64_t st_sb, st_sh, st_sk;
    void* out; int64_t o_sb, o_sh;
};

// log2 of a head's decay for one token.  A decay of exactly zero (log_decay = -inf) and any
// below 2^-160 become 2^-160, which exp2 flushes to zero from the first step on while
// 0 * (-160) stays 0: a distance of zero keeps its weight of one.  NaN passes through.
__device__ __forceinline__ float la_log2_decay(float log_decay) {
    const float g = log_decay * 1.4426950408889634f;
    return g < -160.f ? -160.f : g;
}

// tokens of segment s of row b that lie before the row's length
__device__ __forceinline__ int la_row_length(const LaParams& p, int b) {
    if (!p.length) return p.seqlen;
    const int64_t n = p.length[b];
    return n < 0 ? 0 : (n > p.seqlen ? p.seqlen : (int)n);
}
__device__ __forceinline__ int la_segment_tokens(const LaParams& p, int row_len, int s) {
    const int64_t n = (int64_t)row_len - (int64_t)s * p.seglen;
    return n < 0 ? 0 : (n > p.seglen ? p.seglen : (int)n);
}

}  // namespace ssm
