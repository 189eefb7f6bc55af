// Attention over time with a decay per head: linear attention whose memory of a token fades by lambda = exp(log_decay[head])
// per step.  Per head, with S [d x d] float32:
//     S_t = lambda S_(t-1) + k_t v_t^T,      o_t = m q_t S_t
// over a sequence in tiles of 32 tokens, tokens i, j of a tile, S the state before it:
//     o_i  = m ( sum_(j <= i) lambda^(i-j) (q_i . k_j) v_j  +  lambda^(i+1) q_i S )
//     S'   = lambda^32 S + sum_j lambda^(31-j) k_j v_j^T
// The gradients are the same scan with the operands in other roles:
//     dq : forward in time over (q, k, v) := (do, v, k), with S^T
//     dv : backward in time over (k, q, do) with R = dS / m, where R collects lambda^(i+1) q_i do_i^T
//     dk : backward in time over (v, do, q), with R^T;   the gradient of the first state is m R at the sequence's start
//
// What bounds it: memory.  A tile of one head takes 2 d (d + 32) products per token and tensor element moved - an order
// under what the matrix cores do in the time the rows take - so the kernels are built to keep loads in flight: a wave
// works alone on (sequence, head, segment, 32 columns of v), no barriers, its next tile's rows on their way while the
// current tile is multiplied.  Layouts (v_mfma_f32_32x32x16: lane = row of A / column of B, 8 contraction values):
//   * S^T[key x query] = K Q^T takes both rows as they lie; times the decays (a select: what a later token holds never
//     reaches an earlier one's pairs) it is the B operand of O^T = V^T P^T without leaving the registers;
//   * products that contract over tokens (V^T, K^T) read their transposed operand with ds_read_b64_tr_b16 from the tile's
//     LDS image.  The four-column pieces of that read are taken in an order that swaps bits 2 and 3 of the column index,
//     so that the accumulator registers 8s .. 8s+7 of S and O^T are the eight consecutive features 16s + 8 half ..:
//     the state's registers are then the A operand of q S, whose B operand is a q row as it lies;
//   * the state stays in float32 registers (16 (d / 32) per lane).  Its update has to be as good as float32 (it is handed
//     on): lambda^(31-j) v_j is the sum of three bfloat16 operands or two halfs (under 2^-22 of it is lost).
// Few sequences, long: the time axis is cut into segments.  A first launch computes every segment's own contribution to
// the state (reading k and v only), a second one runs along the segments, a third computes all outputs.
#include "block_common.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int DW = 4;                   // waves per workgroup, each on its own
constexpr int VP = 80;                  // bytes per row of a 32-column LDS image (64 + 16: rows spread over the banks)

struct Strides { long long b, i, n, h; };      // in elements: outer batch, inner batch, token, head

struct ScanArgs {
    const void* q; const void* k; const void* v; void* o;      // by role
    Strides qs, ks, vs, os;
    const float* log_decay;
    const int* lengths;                 // [seq] or null
    const float* s_in; float* s_out;    // [seq][head][d][d] or null
    float s_in_mul, s_out_mul;
    float* seg;                         // [seq][head][nseg][d][d]: a segment's own sum, then the state at its start
    int rs, cs;                         // strides of (row, column) of S in those three
    int inner, n, heads, nseg, seg_len, reverse, e_out, e_u;
    float m;
    long long tasks;
};

__device__ __forceinline__ int swap23(int l) { return (l & 0x13) | ((l & 4) << 1) | ((l & 8) >> 1); }

// log2 lambda, bounded so that exponents of zero tokens stay zero (lambda^1 has underflowed long before -1e4)
__device__ __forceinline__ float log2_decay(const float* log_decay, int head) {
    return fmaxf(log_decay[head] * LOG2E, -1e4f);
}

// lambda^(..) v as a sum of 16-bit operands: three of bfloat16 (8 bits each), two halfs (11 bits each).
// The matrix cores take subnormal half operands as zeros: the low halfs (2^-11 of the values at most) are multiplied up
// by 2^11, and a value that is itself below the normal range goes into the low operand as a whole.  bfloat16 has float's range.
template <typename T> struct Low { static constexpr float SCALE = 1.f; static constexpr bool THREE = true; };
template <> struct Low<_Float16> { static constexpr float SCALE = 2048.f; static constexpr bool THREE = false; };
template <typename T>
__device__ __forceinline__ T high_part(float x) { return (T)x; }
template <>
__device__ __forceinline__ _Float16 high_part<_Float16>(float x) { return (_Float16)(fabsf(x) < 0x1p-14f ? 0.f : x); }

template <typename T, int D, bool STATE_ONLY>
__global__ __launch_bounds__(DW * 64, 2) void decay_scan_kernel(const ScanArgs a) {
    typedef x8_t<T> x8;
    constexpr int KS = D / 16, KT = D / 32, KP = 2 * D + 16;
    constexpr float LOW = Low<T>::SCALE;
    constexpr bool THREE = Low<T>::THREE;
    __shared__ __attribute__((aligned(16))) char kimg_all[DW][32 * KP];
    __shared__ __attribute__((aligned(16))) char vimg_all[DW][32 * VP];
    const int lane = threadIdx.x & 63, half = lane >> 5, l31 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    char* kimg = kimg_all[wave];
    char* vimg = vimg_all[wave];
    long long w = (long long)blockIdx.x * DW + wave;
    if (w >= a.tasks) return;
    const int slice = (int)(w % KT); w /= KT;
    const int head = (int)(w % a.heads); w /= a.heads;
    const int nseg_run = STATE_ONLY && !a.s_out ? a.nseg - 1 : a.nseg;      // nobody reads the last segment's sum
    const int seg = (int)(w % nseg_run);
    const long long seq = w / nseg_run;
    const long long bb = seq / a.inner, ii = seq - bb * a.inner;
    int len = a.n;
    if (a.lengths) len = min(max(a.lengths[seq], 0), a.n);
    const int t_begin = seg * a.seg_len, t_stop = min(a.n, t_begin + a.seg_len), t_end = min(len, t_stop);
    const T* qp = static_cast<const T*>(a.q) + bb * a.qs.b + ii * a.qs.i + head * a.qs.h;
    const T* kp = static_cast<const T*>(a.k) + bb * a.ks.b + ii * a.ks.i + head * a.ks.h;
    const T* vp = static_cast<const T*>(a.v) + bb * a.vs.b + ii * a.vs.i + head * a.vs.h + slice * 32;
    T* op = static_cast<T*>(a.o) + bb * a.os.b + ii * a.os.i + head * a.os.h + slice * 32;
    x8 zero8;
#pragma unroll
    for (int j = 0; j < 8; ++j) zero8[j] = (T)0.f;

    if (!STATE_ONLY) {                      // rows behind the sequence's end
        for (int t = max(len, t_begin) + (lane >> 2); t < t_stop; t += 16)
            *reinterpret_cast<x8*>(op + (long long)t * a.os.n + 8 * (lane & 3)) = zero8;
    }

    const float l2 = log2_decay(a.log_decay, head);
    const long long state0 = (seq * a.heads + head) * (long long)(D * D);
    // this lane's elements of S: row 32 kt + 16 (r >> 3) + 8 half + (r & 7), column 32 slice + swap23(l31)
    const int s_col = (32 * slice + swap23(l31)) * a.cs;
    f32x16 S[KT];
    {
        const float* src = nullptr;
        float mul = 1.f;
        if (!STATE_ONLY) {
            if (a.nseg > 1) src = a.seg + (state0 * a.nseg + (long long)seg * (D * D));
            else if (a.s_in) { src = a.s_in + state0; mul = a.s_in_mul; }
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                S[kt][r] = src ? src[(32 * kt + 16 * (r >> 3) + 8 * half + (r & 7)) * a.rs + s_col] * mul : 0.f;
    }
    // decays: of a pair (register = key, lane = query), of the state towards a query, of a token towards the tile's end
    float dw[16], uw[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int key = (r & 3) + 8 * (r >> 2) + 4 * half;
        dw[r] = a.m * __builtin_amdgcn_exp2f(l2 * (float)max(l31 - key, 0));
    }
    const float ow = a.m * __builtin_amdgcn_exp2f(l2 * (float)(l31 + a.e_out));
    auto token_decays = [&](int cnt) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
            uw[r] = __builtin_amdgcn_exp2f(l2 * (float)(max(cnt - 1 - ((r & 3) + 8 * (r >> 2) + 4 * half), 0) + a.e_u));
    };
    token_decays(32);
    float whole = __builtin_amdgcn_exp2f(l2 * 32.f);

    x8 kreg[KS], vreg[2], qreg[KS];
    auto row_at = [&](int t) { return (long long)(a.reverse ? len - 1 - t : t); };
    auto load = [&](int t0) {
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            const int p = lane + 64 * i, t = t0 + p / (D / 8);
            kreg[i] = t < t_end ? *reinterpret_cast<const x8*>(kp + row_at(t) * a.ks.n + 8 * (p % (D / 8))) : zero8;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int t = t0 + 16 * i + (lane >> 2);
            vreg[i] = t < t_end ? *reinterpret_cast<const x8*>(vp + row_at(t) * a.vs.n + 8 * (lane & 3)) : zero8;
        }
        if (!STATE_ONLY) {
            const int t = t0 + l31;
            const T* p = qp + row_at(t) * a.qs.n + 8 * half;
#pragma unroll
            for (int i = 0; i < KS; ++i) qreg[i] = t < t_end ? *reinterpret_cast<const x8*>(p + 16 * i) : zero8;
        }
    };
    // transposed reads: lane 4 q + p of a 16-lane group supplies row q, four columns; its half's contraction values are
    // rows 4 half + 0..3 and + 8 (accumulator-row order), the column pieces in swapped order (see above)
    const int g16 = lane >> 4, tq = (lane >> 2) & 3, tp = lane & 3;
    const int tr_row = 4 * (g16 >> 1) + tq, tr_col = (16 * (g16 & 1) + 4 * (((tp & 1) << 1) | (tp >> 1))) * 2;
    const char* ktr = kimg + tr_row * KP + tr_col;
    const char* vtr = vimg + tr_row * VP + tr_col;

    if (t_begin < t_end) load(t_begin);
    for (int t0 = t_begin; t0 < t_end; t0 += 32) {
        const int cnt = min(32, t_end - t0);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            const int p = lane + 64 * i;
            *reinterpret_cast<x8*>(kimg + (p / (D / 8)) * KP + 16 * (p % (D / 8))) = kreg[i];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) *reinterpret_cast<x8*>(vimg + (16 * i + (lane >> 2)) * VP + 16 * (lane & 3)) = vreg[i];
        x8 q[KS];
#pragma unroll
        for (int i = 0; i < KS; ++i) q[i] = qreg[i];
        if (t0 + 32 < t_end) load(t0 + 32);
        const x8 v0 = tr_operand<T>(vtr, 8 * VP), v1 = tr_operand<T>(vtr + 16 * VP, 8 * VP);
        if (!STATE_ONLY) {
            f32x16 st = zero16(), o = zero16();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const x8 kf = *reinterpret_cast<const x8*>(kimg + l31 * KP + 32 * ks + 16 * half);
                st = mfma16(kf, q[ks], st);
                o = mfma16(acc_operand<T>(S[ks >> 1], ks & 1), q[ks], o);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                st[r] = (r & 3) + 8 * (r >> 2) + 4 * half <= l31 ? st[r] * dw[r] : 0.f;
                o[r] *= ow;
            }
            o = mfma16(v0, acc_operand<T>(st, 0), o);
            o = mfma16(v1, acc_operand<T>(st, 1), o);
            // through LDS (the tile's v image is in registers by now) to 16-byte stores, four lanes on a row's 64 bytes
            *reinterpret_cast<x8*>(vimg + l31 * VP + 16 * half) = acc_operand<T>(o, 0);
            *reinterpret_cast<x8*>(vimg + l31 * VP + 32 + 16 * half) = acc_operand<T>(o, 1);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = 16 * i + (lane >> 2);
                const x8 piece = *reinterpret_cast<const x8*>(vimg + row * VP + 16 * (lane & 3));
                if (row < cnt) *reinterpret_cast<x8*>(op + row_at(t0 + row) * a.os.n + 8 * (lane & 3)) = piece;
            }
        }
        if (cnt < 32) {
            token_decays(cnt);
            whole = __builtin_amdgcn_exp2f(l2 * (float)cnt);
        }
        x8 h0, h1, e0, e1, f0, f1;          // lambda^(..) v as a sum of operands
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x0 = (float)v0[j] * uw[j], x1 = (float)v1[j] * uw[8 + j];
            h0[j] = high_part<T>(x0);
            h1[j] = high_part<T>(x1);
            const float y0 = (x0 - (float)h0[j]) * LOW, y1 = (x1 - (float)h1[j]) * LOW;
            e0[j] = (T)y0;
            e1[j] = (T)y1;
            if (THREE) {
                f0[j] = (T)(y0 - (float)e0[j]);
                f1[j] = (T)(y1 - (float)e1[j]);
            }
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            const x8 k0 = tr_operand<T>(ktr + 64 * kt, 8 * KP), k1 = tr_operand<T>(ktr + 64 * kt + 16 * KP, 8 * KP);
            f32x16 add = mfma16(k0, e0, zero16());
#pragma unroll
            for (int r = 0; r < 16; ++r) S[kt][r] *= whole;
            S[kt] = mfma16(k0, h0, S[kt]);
            add = mfma16(k1, e1, add);
            S[kt] = mfma16(k1, h1, S[kt]);
            if (THREE) {
                f32x16 last = mfma16(k0, f0, zero16());
                last = mfma16(k1, f1, last);
#pragma unroll
                for (int r = 0; r < 16; ++r) add[r] += last[r];
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) S[kt][r] += add[r] * (1.f / LOW);
        }
    }
    float* dst = nullptr;
    float mul = 1.f;
    if (STATE_ONLY) dst = a.seg + (state0 * a.nseg + (long long)seg * (D * D));
    else if (a.s_out && a.nseg == 1) { dst = a.s_out + state0; mul = a.s_out_mul; }
    if (dst) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int r = 0; r < 16; ++r) dst[(32 * kt + 16 * (r >> 3) + 8 * half + (r & 7)) * a.rs + s_col] = S[kt][r] * mul;
    }
}

// Along the segments of a sequence: sums of single segments -> states at their starts, and the state after the last one.
// One thread per element of S; bound by reading and writing the segment states once.
__global__ __launch_bounds__(256) void decay_segments_kernel(const ScanArgs a, int dd) {
    const long long sh = blockIdx.x;                    // (sequence, head)
    const int e = blockIdx.y * 256 + threadIdx.x;
    const long long seq = sh / a.heads;
    const float l2 = log2_decay(a.log_decay, (int)(sh - seq * a.heads));
    int len = a.n;
    if (a.lengths) len = min(max(a.lengths[seq], 0), a.n);
    float* p = a.seg + sh * a.nseg * (long long)dd + e;
    float cur = a.s_in ? a.s_in[sh * dd + e] * a.s_in_mul : 0.f;
    const int have = a.s_out ? a.nseg : a.nseg - 1;     // segments whose sum was computed
    constexpr int AHEAD = 8;
    float next[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) next[i] = i < have ? p[(long long)i * dd] : 0.f;
    for (int s0 = 0; s0 < a.nseg; s0 += AHEAD) {
        float sum[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            sum[i] = next[i];
            const int s = s0 + AHEAD + i;
            next[i] = s < have ? p[(long long)s * dd] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int s = s0 + i;
            if (s < a.nseg) {
                p[(long long)s * dd] = cur;
                const int cnt = min(max(len - s * a.seg_len, 0), a.seg_len);
                cur = cur * __builtin_amdgcn_exp2f(l2 * (float)cnt) + sum[i];
            }
        }
    }
    if (a.s_out) a.s_out[sh * dd + e] = cur * a.s_out_mul;
}

// ------------------------------------------------------------------------------------------------------------------
// Sequences of up to 32 tokens without states (the frames of a site): g = 32 / n whole sequences share a tile of 32
// rows, pairs of different sequences are masked, and the backward pass does all three gradients from one read of q, k,
// v and do (dP^T = V dO^T with lane = query for dq; P = Q K^T and dP = dO V^T with lane = key for dv and dk).  A wave
// takes (tile, head) units one after the other, always of the same head, the next unit's rows in flight.
// A row that is not finite must not reach the other sequences of its tile (zero times infinity): such a tile is
// computed once per sequence with the others' rows as zeros.
// ------------------------------------------------------------------------------------------------------------------
struct ShortArgs {
    const void* q; const void* k; const void* v; const void* g;        // g: gradient of o
    void* o; void* dq; void* dk; void* dv;
    Strides qs, ks, vs, gs, os, dqs, dks, dvs;
    const float* log_decay;
    const int* lengths;
    int inner, n, heads, per_tile;
    float m;
    long long nseq, units;
};

template <typename T>
__device__ __forceinline__ bool not_finite(const x8_t<T>& x) {
    const uint4 w = __builtin_bit_cast(uint4, x);
    const unsigned lo = Pack<T>::EXP, hi = lo << 16;
    bool bad = false;
    for (unsigned u : {w.x, w.y, w.z, w.w}) bad |= (u & lo) == lo || (u & hi) == hi;
    return bad;
}

template <typename T, int D, bool BWD>
__global__ __launch_bounds__(DW * 64, D == 128 ? 1 : 2) void decay_short_kernel(const ShortArgs a) {
    typedef x8_t<T> x8;
    constexpr int KS = D / 16, DT = D / 32, P = 2 * D + 16, NI = BWD ? 3 : 1;
    __shared__ __attribute__((aligned(16))) char img_all[DW][NI][32 * P];       // forward: v; backward: k, q, do
    __shared__ __attribute__((aligned(16))) char out_all[DW][32 * VP];
    const int lane = threadIdx.x & 63, half = lane >> 5, l31 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    char* oimg = out_all[wave];
    const long long gid = (long long)blockIdx.x * DW + wave, stride = (long long)gridDim.x * DW;   // stride % heads == 0
    const int head = (int)(gid % a.heads), n = a.n;
    const int slot = l31 / n, ti = l31 - slot * n;
    const bool in_tile = slot < a.per_tile;
    const float l2 = log2_decay(a.log_decay, head);
    // decays of (register = key, lane = query) and, for the backward, (register = query, lane = key); zero bits of the
    // masks: later keys, other sequences
    float dw[16], dwt[16];
    unsigned mask = 0, maskt = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int t = (r & 3) + 8 * (r >> 2) + 4 * half;
        const bool same = in_tile && t / n == slot;
        if (same && t <= l31) mask |= 1u << r;
        if (same && t >= l31) maskt |= 1u << r;
        dw[r] = a.m * __builtin_amdgcn_exp2f(l2 * (float)max(l31 - t, 0));
        dwt[r] = a.m * __builtin_amdgcn_exp2f(l2 * (float)max(t - l31, 0));
    }
    x8 zero8;
#pragma unroll
    for (int j = 0; j < 8; ++j) zero8[j] = (T)0.f;
    const int g16 = lane >> 4, tq = (lane >> 2) & 3, tp = lane & 3;
    const int tr_off = (4 * (g16 >> 1) + tq) * P + (16 * (g16 & 1) + 4 * (((tp & 1) << 1) | (tp >> 1))) * 2;

    // the sequence of a unit's row, as (outer, inner) batch indexes
    auto seq_of = [&](long long u, int sl, long long& bb, long long& ii) {
        const long long seq = (u / a.heads) * a.per_tile + sl;
        if (sl >= a.per_tile || seq >= a.nseq) return false;
        bb = seq / a.inner;
        ii = seq - bb * a.inner;
        return true;
    };
    struct Unit { x8 q[KS], k[KS], v[KS], g[BWD ? KS : 1]; };
    auto fetch = [&](long long u, Unit& x) {
        long long bb = 0, ii = 0;
        bool ok = u < a.units && seq_of(u, slot, bb, ii);
        if (ok && a.lengths) ok = ti < a.lengths[bb * a.inner + ii];
        const T* qp = static_cast<const T*>(a.q) + bb * a.qs.b + ii * a.qs.i + ti * a.qs.n + head * a.qs.h + 8 * half;
        const T* kp = static_cast<const T*>(a.k) + bb * a.ks.b + ii * a.ks.i + ti * a.ks.n + head * a.ks.h + 8 * half;
        const T* vp = static_cast<const T*>(a.v) + bb * a.vs.b + ii * a.vs.i + ti * a.vs.n + head * a.vs.h + 8 * half;
        const T* gp = static_cast<const T*>(a.g) + bb * a.gs.b + ii * a.gs.i + ti * a.gs.n + head * a.gs.h + 8 * half;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            x.q[s] = ok ? *reinterpret_cast<const x8*>(qp + 16 * s) : zero8;
            x.k[s] = ok ? *reinterpret_cast<const x8*>(kp + 16 * s) : zero8;
            x.v[s] = ok ? *reinterpret_cast<const x8*>(vp + 16 * s) : zero8;
            if constexpr (BWD) x.g[s] = ok ? *reinterpret_cast<const x8*>(gp + 16 * s) : zero8;
        }
    };
    auto to_image = [&](char* im, const x8 (&x)[KS]) {
#pragma unroll
        for (int s = 0; s < KS; ++s) *reinterpret_cast<x8*>(im + l31 * P + 32 * s + 16 * half) = x[s];
    };
    // [features x features] contraction of two row sets, in two accumulators (no chain of dependent products)
    auto pairs = [&](const x8 (&x)[KS], const x8 (&y)[KS]) {
        f32x16 p = zero16(), p2 = zero16();
#pragma unroll
        for (int s = 0; s < KS; s += 2) {
            p = mfma16(x[s], y[s], p);
            p2 = mfma16(x[s + 1], y[s + 1], p2);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] += p2[r];
        return p;
    };
    auto weigh = [&](f32x16& p, const float (&d)[16], unsigned m) {
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] = ((m >> r) & 1u) ? p[r] * d[r] : 0.f;
    };
    // rows of 32 tokens x D: (transposed image)^T x pairs, stored for the sequences [s_lo, s_hi) of the tile
    auto product = [&](const char* im, const f32x16& p, void* dst, const Strides& ds, long long u, int s_lo, int s_hi) {
        const x8 p0 = acc_operand<T>(p, 0), p1 = acc_operand<T>(p, 1);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            f32x16 o = mfma16(tr_operand<T>(im + tr_off + 64 * dt, 8 * P), p0, zero16());
            o = mfma16(tr_operand<T>(im + tr_off + 64 * dt + 16 * P, 8 * P), p1, o);
            *reinterpret_cast<x8*>(oimg + l31 * VP + 16 * half) = acc_operand<T>(o, 0);
            *reinterpret_cast<x8*>(oimg + l31 * VP + 32 + 16 * half) = acc_operand<T>(o, 1);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = 16 * i + (lane >> 2), sl = row / n;
                const x8 piece = *reinterpret_cast<const x8*>(oimg + row * VP + 16 * (lane & 3));
                long long bb, ii;
                if (sl >= s_lo && sl < s_hi && seq_of(u, sl, bb, ii))
                    *reinterpret_cast<x8*>(static_cast<T*>(dst) + bb * ds.b + ii * ds.i + (row - sl * n) * ds.n + head * ds.h +
                                           32 * dt + 8 * (lane & 3)) = piece;
            }
        }
    };

    Unit nx;
    fetch(gid, nx);
    for (long long u = gid; u < a.units; u += stride) {
        const Unit c = nx;
        fetch(u + stride, nx);
        bool bad = false;
        if (a.per_tile > 1) {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                bad |= not_finite<T>(c.v[s]);
                if constexpr (BWD) bad |= not_finite<T>(c.k[s]) || not_finite<T>(c.q[s]) || not_finite<T>(c.g[s]);
            }
        }
        const bool apart = __builtin_amdgcn_ballot_w64(bad) != 0;
        const int passes = apart ? a.per_tile : 1;
        for (int pass = 0; pass < passes; ++pass) {
            const int s_lo = apart ? pass : 0, s_hi = apart ? pass + 1 : a.per_tile;
            const bool on = !apart || slot == pass;
            Unit x;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                x.q[s] = on ? c.q[s] : zero8;
                x.k[s] = on ? c.k[s] : zero8;
                x.v[s] = on ? c.v[s] : zero8;
                if constexpr (BWD) x.g[s] = on ? c.g[s] : zero8;
            }
            if constexpr (!BWD) {
                to_image(img_all[wave][0], x.v);
                f32x16 st = pairs(x.k, x.q);
                weigh(st, dw, mask);
                product(img_all[wave][0], st, a.o, a.os, u, s_lo, s_hi);
            } else {
                to_image(img_all[wave][0], x.k);
                to_image(img_all[wave][1], x.q);
                to_image(img_all[wave][2], x.g);
                f32x16 p = pairs(x.v, x.g);                 // [key x query]
                weigh(p, dw, mask);
                product(img_all[wave][0], p, a.dq, a.dqs, u, s_lo, s_hi);
                p = pairs(x.q, x.k);                        // [query x key]
                weigh(p, dwt, maskt);
                product(img_all[wave][2], p, a.dv, a.dvs, u, s_lo, s_hi);
                p = pairs(x.g, x.v);
                weigh(p, dwt, maskt);
                product(img_all[wave][1], p, a.dk, a.dks, u, s_lo, s_hi);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------
// One more token of every sequence: S <- lambda S + k v^T in place, o = m q S.  Bound by reading and writing S once.  A
// wave takes 32 columns of one (sequence, head): 8 rows x 128 contiguous bytes per load, all its loads in flight.
// ------------------------------------------------------------------------------------------------------------------
struct StepArgs {
    const void* q; const void* k; const void* v; void* o;
    long long qb, qh, kb, kh, vb, vh, ob, oh;           // strides: sequence, head
    const float* log_decay;
    float* state;
    int heads;
    float m;
    long long tasks;
};

template <typename T, int D>
__global__ __launch_bounds__(256) void decay_step_kernel(const StepArgs a) {
    constexpr int IT = D / 8;
    long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (w >= a.tasks) return;
    const int lane = threadIdx.x & 63, row = lane >> 3, c4 = 4 * (lane & 7);
    const int slice = (int)(w % (D / 32)); w /= D / 32;
    const int head = (int)(w % a.heads);
    const long long seq = w / a.heads;
    float* s = a.state + w * (long long)(D * D) + row * D + 32 * slice + c4;
    f32x4 x[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) x[i] = *reinterpret_cast<const f32x4*>(s + i * 8 * D);
    const T* qp = static_cast<const T*>(a.q) + seq * a.qb + head * a.qh;
    const T* kp = static_cast<const T*>(a.k) + seq * a.kb + head * a.kh;
    const T* vp = static_cast<const T*>(a.v) + seq * a.vb + head * a.vh + 32 * slice + c4;
    float v[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)vp[j];
    const float lam = __builtin_amdgcn_exp2f(log2_decay(a.log_decay, head));
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const float kk = (float)kp[8 * i + row], qq = (float)qp[8 * i + row];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[i][j] = lam * x[i][j] + kk * v[j];
            o[j] += qq * x[i][j];
        }
        *reinterpret_cast<f32x4*>(s + i * 8 * D) = x[i];
    }
    // rows 8 i + lane / 8: add the eight lanes of a column
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        o[j] += __shfl_xor(o[j], 8);
        o[j] += __shfl_xor(o[j], 16);
        o[j] = xhalf_add(o[j]) * a.m;
    }
    if (row == 0) {
        T* op = static_cast<T*>(a.o) + seq * a.ob + head * a.oh + 32 * slice + c4;
#pragma unroll
        for (int j = 0; j < 4; ++j) op[j] = (T)o[j];
    }
}

// ------------------------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------------------------
struct Plan { bool is_short; int nseg, seg_len; long long nseq; size_t bytes; };

bool rows_ok(const vdmi_rows4& r) {
    return r.p && aligned16(r.p) && r.b % 8 == 0 && r.i % 8 == 0 && r.n % 8 == 0 && r.h % 8 == 0;
}

int check_args(const vdmi_decay_args* a) {
    if (!a || !a->log_decay) return VDMI_E_ARG;
    if (a->dtype != VDMI_DT_BF16 && a->dtype != VDMI_DT_F16) return VDMI_E_ARG;
    if (!(a->scale != 0.f) || !(a->scale - a->scale == 0.f)) return VDMI_E_ARG;       // zero, infinite, NaN
    if (a->b <= 0 || a->inner <= 0 || a->n <= 0 || a->heads <= 0 || a->heads > 65535) return VDMI_E_SHAPE;
    if (a->d != 32 && a->d != 64 && a->d != 128) return VDMI_E_SHAPE;
    if ((long long)a->b * a->inner > 0x7fffffffLL / a->heads || a->n > (1 << 30)) return VDMI_E_SHAPE;
    if (!a->q.p || !a->k.p || !a->v.p) return VDMI_E_ARG;
    if (!rows_ok(a->q) || !rows_ok(a->k) || !rows_ok(a->v)) return VDMI_E_ALIGN;
    return VDMI_OK;
}

// How the time axis is cut: waves = sequences x heads x d / 32 column slices x segments.  The card holds 256 x 8 waves of
// these kernels; a segment costs its state (4 d d bytes written and read twice) and a second read of k and v, so segments
// are only cut until the card is filled and never shorter than 4 d tokens (state traffic under half of its rows').
Plan plan(const vdmi_decay_args* a, bool states) {
    Plan p;
    p.nseq = (long long)a->b * a->inner;
    p.is_short = a->n <= 32 && !states;
    p.nseg = 1;
    p.seg_len = a->n;
    p.bytes = 0;
    if (p.is_short) return p;
    const long long waves = p.nseq * a->heads * (a->d / 32);
    long long want = 2048 / waves;
    const long long most = a->n / (4 * a->d);
    if (want > most) want = most;
    if (want > 1) {
        p.seg_len = (int)(((a->n + want - 1) / want + 31) / 32 * 32);
        p.nseg = (a->n + p.seg_len - 1) / p.seg_len;
    }
    if (p.nseg > 1) p.bytes = (size_t)p.nseq * a->heads * p.nseg * a->d * a->d * sizeof(float);
    return p;
}

bool wants_states(const vdmi_decay_args* a) { return a->state_in || a->state_out || a->dstate_in || a->dstate_out; }

Strides strides_of(const vdmi_rows4& r) { return Strides{r.b, r.i, r.n, r.h}; }

template <bool STATE_ONLY>
int launch_scan(const ScanArgs& s, const vdmi_decay_args* a, const Plan& p, hipStream_t st) {
    ScanArgs x = s;
    const long long segs = STATE_ONLY && !x.s_out ? p.nseg - 1 : p.nseg;
    x.tasks = p.nseq * a->heads * segs * (a->d / 32);
    const long long wgs = (x.tasks + DW - 1) / DW;
    if (wgs > 0x7fffffffLL) return VDMI_E_SHAPE;
    const dim3 grid((unsigned)wgs), block(DW * 64);
#define SCAN(T, D) hipLaunchKernelGGL((decay_scan_kernel<T, D, STATE_ONLY>), grid, block, 0, st, x)
#define SCAN_D(T) do { if (a->d == 32) SCAN(T, 32); else if (a->d == 64) SCAN(T, 64); else SCAN(T, 128); } while (0)
    if (a->dtype == VDMI_DT_BF16) SCAN_D(__bf16); else SCAN_D(_Float16);
#undef SCAN_D
#undef SCAN
    VDMI_LAUNCH_CHECK();
    return VDMI_OK;
}

// sums of the segments and the states at their starts (nothing to do for one segment)
int segment_states(ScanArgs s, const vdmi_decay_args* a, const Plan& p, hipStream_t st) {
    if (p.nseg == 1) return VDMI_OK;
    s.rs = a->d;
    s.cs = 1;
    const int r = launch_scan<true>(s, a, p, st);
    if (r != VDMI_OK) return r;
    hipLaunchKernelGGL(decay_segments_kernel, dim3((unsigned)(p.nseq * a->heads), (unsigned)(a->d * a->d / 256)), dim3(256), 0, st,
                       s, a->d * a->d);
    VDMI_LAUNCH_CHECK();
    return VDMI_OK;
}

void role(ScanArgs& s, const vdmi_rows4& q, const vdmi_rows4& k, const vdmi_rows4& v, const vdmi_rows4& o) {
    s.q = q.p; s.k = k.p; s.v = v.p; s.o = o.p;
    s.qs = strides_of(q); s.ks = strides_of(k); s.vs = strides_of(v); s.os = strides_of(o);
}

ScanArgs scan_args(const vdmi_decay_args* a, const Plan& p) {
    ScanArgs s = {};
    s.log_decay = a->log_decay;
    s.lengths = a->lengths;
    s.s_in_mul = s.s_out_mul = 1.f;
    s.seg = static_cast<float*>(a->workspace);
    s.rs = a->d; s.cs = 1;
    s.inner = a->inner; s.n = a->n; s.heads = a->heads;
    s.nseg = p.nseg; s.seg_len = p.seg_len;
    s.m = a->scale;
    return s;
}

int launch_short(const vdmi_decay_args* a, const Plan& p, bool bwd, hipStream_t st) {
    ShortArgs s = {};
    s.q = a->q.p; s.k = a->k.p; s.v = a->v.p; s.g = a->dout.p;
    s.o = a->o.p; s.dq = a->dq.p; s.dk = a->dk.p; s.dv = a->dv.p;
    s.qs = strides_of(a->q); s.ks = strides_of(a->k); s.vs = strides_of(a->v); s.gs = strides_of(a->dout);
    s.os = strides_of(a->o); s.dqs = strides_of(a->dq); s.dks = strides_of(a->dk); s.dvs = strides_of(a->dv);
    s.log_decay = a->log_decay; s.lengths = a->lengths;
    s.inner = a->inner; s.n = a->n; s.heads = a->heads; s.per_tile = 32 / a->n;
    s.m = a->scale;
    s.nseq = p.nseq;
    s.units = (p.nseq + s.per_tile - 1) / s.per_tile * a->heads;
    // a wave keeps its head: the number of waves is a multiple of the heads
    long long wgs = (s.units + DW - 1) / DW;
    if (wgs > 2048) wgs = 2048;
    wgs = (wgs + a->heads - 1) / a->heads * a->heads;
    const dim3 grid((unsigned)wgs), block(DW * 64);
#define SHORT(T, D) do { if (bwd) hipLaunchKernelGGL((decay_short_kernel<T, D, true>), grid, block, 0, st, s); \
                         else hipLaunchKernelGGL((decay_short_kernel<T, D, false>), grid, block, 0, st, s); } while (0)
#define SHORT_D(T) do { if (a->d == 32) SHORT(T, 32); else if (a->d == 64) SHORT(T, 64); else SHORT(T, 128); } while (0)
    if (a->dtype == VDMI_DT_BF16) SHORT_D(__bf16); else SHORT_D(_Float16);
#undef SHORT_D
#undef SHORT
    VDMI_LAUNCH_CHECK();
    return VDMI_OK;
}

}   // namespace

extern "C" size_t vdmi_decay_attn_workspace_bytes(const vdmi_decay_args* a) {
    if (check_args(a) != VDMI_OK) return 0;
    return plan(a, wants_states(a)).bytes;
}

extern "C" int vdmi_decay_attn_fwd(const vdmi_decay_args* a, vdmi_stream stream) {
    const int ok = check_args(a);
    if (ok != VDMI_OK) return ok;
    if (!a->o.p) return VDMI_E_ARG;
    if (!rows_ok(a->o)) return VDMI_E_ALIGN;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const Plan p = plan(a, wants_states(a));
    if (p.is_short) return launch_short(a, p, false, st);
    if (p.bytes && (!a->workspace || a->workspace_bytes < (int64_t)p.bytes)) return VDMI_E_ARG;
    ScanArgs s = scan_args(a, p);
    role(s, a->q, a->k, a->v, a->o);
    s.s_in = a->state_in;
    s.s_out = a->state_out;
    s.e_out = 1;
    const int r = segment_states(s, a, p, st);
    return r != VDMI_OK ? r : launch_scan<false>(s, a, p, st);
}

extern "C" int vdmi_decay_attn_bwd(const vdmi_decay_args* a, vdmi_stream stream) {
    const int ok = check_args(a);
    if (ok != VDMI_OK) return ok;
    if (!a->dout.p || !a->dq.p || !a->dk.p || !a->dv.p) return VDMI_E_ARG;
    if (!rows_ok(a->dout) || !rows_ok(a->dq) || !rows_ok(a->dk) || !rows_ok(a->dv)) return VDMI_E_ALIGN;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const Plan p = plan(a, wants_states(a));
    if (p.is_short) return launch_short(a, p, true, st);
    if (p.bytes && (!a->workspace || a->workspace_bytes < (int64_t)p.bytes)) return VDMI_E_ARG;
    int r;
    // dq: forward in time, S^T
    ScanArgs s = scan_args(a, p);
    s.s_in = a->state_in;
    s.e_out = 1;
    role(s, a->q, a->k, a->v, a->dq);
    if ((r = segment_states(s, a, p, st)) != VDMI_OK) return r;
    role(s, a->dout, a->v, a->k, a->dq);
    s.rs = 1;
    s.cs = a->d;
    if ((r = launch_scan<false>(s, a, p, st)) != VDMI_OK) return r;
    // dv and dk: backward in time; R = dS / m collects lambda^(i+1) q_i do_i^T
    s = scan_args(a, p);
    s.reverse = 1;
    s.e_u = 1;
    s.s_in = a->dstate_in;
    s.s_in_mul = 1.f / a->scale;
    s.s_out = a->dstate_out;
    s.s_out_mul = a->scale;
    role(s, a->k, a->q, a->dout, a->dv);
    if ((r = segment_states(s, a, p, st)) != VDMI_OK) return r;
    if ((r = launch_scan<false>(s, a, p, st)) != VDMI_OK) return r;
    s.s_out = nullptr;
    role(s, a->v, a->dout, a->q, a->dk);
    s.rs = 1;
    s.cs = a->d;
    return launch_scan<false>(s, a, p, st);
}

extern "C" int vdmi_decay_attn_step(const void* q, const void* k, const void* v, void* o, const int64_t* strides,
                                    const float* log_decay, float* state, int dtype, int64_t seqs, int heads, int d, float scale,
                                    vdmi_stream stream) {
    if (!q || !k || !v || !o || !strides || !log_decay || !state) return VDMI_E_ARG;
    if (dtype != VDMI_DT_BF16 && dtype != VDMI_DT_F16) return VDMI_E_ARG;
    if (!(scale != 0.f) || !(scale - scale == 0.f)) return VDMI_E_ARG;
    if (seqs <= 0 || heads <= 0 || (d != 32 && d != 64 && d != 128) || seqs > 0x7fffffffLL / heads) return VDMI_E_SHAPE;
    if (!aligned16(state)) return VDMI_E_ALIGN;
    StepArgs s = {q, k, v, o, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], strides[6], strides[7],
                  log_decay, state, heads, scale, seqs * heads * (d / 32)};
    const long long wgs = (s.tasks + 3) / 4;
    if (wgs > 0x7fffffffLL) return VDMI_E_SHAPE;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)wgs), block(256);
#define STEP(T) do { if (d == 32) hipLaunchKernelGGL((decay_step_kernel<T, 32>), grid, block, 0, st, s); \
                     else if (d == 64) hipLaunchKernelGGL((decay_step_kernel<T, 64>), grid, block, 0, st, s); \
                     else hipLaunchKernelGGL((decay_step_kernel<T, 128>), grid, block, 0, st, s); } while (0)
    if (dtype == VDMI_DT_BF16) STEP(__bf16); else STEP(_Float16);
#undef STEP
    VDMI_LAUNCH_CHECK();
    return VDMI_OK;
}
