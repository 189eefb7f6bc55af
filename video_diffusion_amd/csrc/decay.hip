// Attention over time with a decay per head: linear attention whose memory of a token fades by lambda = exp(log_decay[head])
// per step.  Per head, with S [d x d] float32:
//     S_t = lambda S_(t-1) + k_t v_t^T,      o_t = m q_t S_t
// over a sequence in tiles of 32 tokens, tokens i, j of a tile, S the state before it:
//     o_i  = m ( sum_(j <= i) lambda^(i-j) (q_i . k_j) v_j  +  lambda^(i+1) q_i S )
//     S'   = lambda^32 S + sum_j lambda^(31-j) k_j v_j^T
// The gradients are the same scan with the operands in other roles:
//     dq : forward in time over (q, k, v) := (do, v, k), with S^T
//     dv : backward in time over (k, q, do) with R = dS / m, where R collects lambda^(i+1) q_i do_i^T
//     dk : backward in time over (v, do, q), with R^T (one walk with dv);   the gradient of the first state is m R there
//
// What bounds it: memory, and the instructions of a tile where long sequences leave a wave alone on its SIMD.  A tile of one
// head takes 2 d (d + 32) products per token and tensor element moved - an order under what the matrix cores do in the time
// the rows take - so the kernels are built to keep loads in flight: a wave works alone on (sequence, head, segment, 32
// columns of v), no barriers, its next tile's rows on their way while the current tile is multiplied.  Layouts
// (v_mfma_f32_32x32x16: lane = row of A / column of B, 8 contraction values):
//   * S^T[key x query] = K Q^T takes both rows as they lie; times the decays (a select: what a later token holds never
//     reaches an earlier one's pairs) it is the B operand of O^T = V^T P^T without leaving the registers;
//   * products that contract over tokens (V^T, K^T) read their transposed operand with ds_read_b64_tr_b16 from the tile's
//     LDS image.  The four-column pieces of that read are taken in an order that swaps bits 2 and 3 of the column index,
//     so that the accumulator registers 8s .. 8s+7 of S and O^T are the eight consecutive features 16s + 8 half ..:
//     the state's registers are then the A operand of q S, whose B operand is a q row as it lies;
//   * the state stays in float32 registers (16 (d / 32) per lane).  Its update has to be as good as float32 (it is handed
//     on): lambda^(31-j) v_j is the sum of three bfloat16 operands or two halfs (under 2^-22 of it is lost).
// Few sequences: the time axis is cut into segments.  A first launch computes every segment's own contribution to the state
// (reading k and v only), a second one runs along the segments, a third computes all outputs.
// Measured, 2 x 8192 tokens, 8 heads of 64 features, bfloat16 (16.8 MB a tensor): segments' sums 11.7 us (2.9 TB/s), along
// the segments 6.5, outputs 20 (3.4 TB/s); backward dq 20, dk and dv 32 (3.7 TB/s) beside another walk for the segments.
// 16384 tokens, 8 heads of 128, half: 24 + 8.4 + 54 us.  There a wave has its SIMD to itself and bounds it by issuing: 72 % of
// its cycles in the outputs and 66 % in the gradients, 18 and 26 % waiting (2 x 8192 x 8 x 64: 60 and 59 %, 25 and 21 %).  Two
// waves per SIMD hide that but take twice the segments, whose states cost as much.
#include "block_common.h"

#include <algorithm>

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
    int rs;                             // the stride of S's rows in s_in and seg: d, or 1 where S is read transposed
    int inner, n, heads, nseg, seg_len, reverse, e_out, e_u;
    float m;
    unsigned tasks;
};

struct GradArgs {                       // dk and dv
    const void* q; const void* k; const void* v; const void* g; void* dk; void* dv;
    Strides qs, ks, vs, gs, dks, dvs;
    const float* log_decay;
    const int* lengths;
    const float* s_in; float* s_out;    // gradients of the last and of the first state
    const float* seg;
    int inner, n, heads, nseg, seg_len;
    float m;
    unsigned tasks;
};

__device__ __forceinline__ int swap23(int l) { return (l & 0x13) | ((l & 4) << 1) | ((l & 8) >> 1); }
__device__ __forceinline__ int acc_row(int reg, int half) { return (reg & 3) + 8 * (reg >> 2) + 4 * half; }

// log2 lambda, bounded so that exponents of zero tokens stay zero (lambda^1 has underflowed long before -1e4); NaN stays
__device__ __forceinline__ float log2_decay(const float* log_decay, int head) {
    const float l2 = log_decay[head] * LOG2E;
    return l2 < -1e4f ? -1e4f : l2;
}

// p * w where w = 0 marks a pair that does not exist: zero whatever p is (0 * inf and 0 * NaN are 0).  v_mul_legacy_f32 as
// the compiler's intrinsic, so that it keeps the waits between a matrix instruction and the first use of its result.
extern "C" __device__ float vdmi_mul_legacy(float, float) __asm("llvm.amdgcn.fmul.legacy");
__device__ __forceinline__ float weigh(float p, float w) { return vdmi_mul_legacy(p, w); }

// lambda^(..) v as a sum of 16-bit operands: three of bfloat16 (8 bits each), two halfs (11 bits each).
// The low halfs (2^-11 of the values at most) are multiplied up by 2^11, so that what is lost of a value is 2^-22 of it or
// 2^-36, where a sum of plain halfs ends at steps of 2^-24.  (The matrix cores take subnormal halfs as what they are: 2^-15,
// 2^-20 and 2^-24 as either operand gave exact products.)  bfloat16 has float's range.
template <typename T> struct Low { static constexpr float SCALE = 1.f; static constexpr bool THREE = true; };
template <> struct Low<_Float16> { static constexpr float SCALE = 2048.f; static constexpr bool THREE = false; };

// two values at a time: the conversions come in pairs
template <typename T>
struct Two {
    typedef __attribute__((ext_vector_type(2))) T t2;
    typedef __attribute__((ext_vector_type(2))) float f2;
    // elements j, j + 1 of h = what T holds of a, b;  a, b become what is left, times SCALE
    static __device__ __forceinline__ void take(x8_t<T>& h, int j, float& a, float& b) {
        const t2 w = __builtin_convertvector((f2{a, b}), t2);
        const f2 back = __builtin_convertvector(w, f2);
        h[j] = w[0];
        h[j + 1] = w[1];
        a = (a - back[0]) * Low<T>::SCALE;
        b = (b - back[1]) * Low<T>::SCALE;
    }
    static __device__ __forceinline__ void round(x8_t<T>& h, int j, float a, float b) {
        const t2 w = __builtin_convertvector((f2{a, b}), t2);
        h[j] = w[0];
        h[j + 1] = w[1];
    }
};

template <typename T>
struct Split {
    x8_t<T> h[2], e[2], f[2];
    // w: the weights of the 32 tokens, in LDS
    __device__ __forceinline__ Split(const x8_t<T>& v0, const x8_t<T>& v1, const float* w, int half) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const f32x4 w0 = *reinterpret_cast<const f32x4*>(w + 16 * s + 4 * half), w1 = *reinterpret_cast<const f32x4*>(w + 16 * s + 8 + 4 * half);
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                float x = (float)(s ? v1 : v0)[j] * (j < 4 ? w0[j & 3] : w1[j & 3]);
                float y = (float)(s ? v1 : v0)[j + 1] * (j < 4 ? w0[(j + 1) & 3] : w1[(j + 1) & 3]);
                Two<T>::take(h[s], j, x, y);
                if (Low<T>::THREE) {
                    Two<T>::take(e[s], j, x, y);
                    Two<T>::round(f[s], j, x, y);
                } else {
                    Two<T>::round(e[s], j, x, y);
                }
            }
        }
    }
    // S[kt] <- whole S[kt] + (columns 32 kt .. of the image at tr)^T (the split rows)
    template <int KT>
    __device__ __forceinline__ void update(f32x16 (&S)[KT], float whole, const char* tr, int pitch) const {
        if constexpr (Low<T>::THREE && KT > 1) {
            // all into S: the products of different kt in turn (no chain of dependent ones)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int r = 0; r < 16; ++r) S[kt][r] *= whole;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                x8_t<T> k[KT];
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) k[kt] = tr_operand<T>(tr + 64 * kt + 16 * s * pitch, 8 * pitch);
#pragma unroll
                for (int t = 0; t < 3; ++t)
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) S[kt] = mfma16(k[kt], t == 0 ? f[s] : t == 1 ? e[s] : h[s], S[kt]);
            }
        } else {
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                const x8_t<T> k0 = tr_operand<T>(tr + 64 * kt, 8 * pitch), k1 = tr_operand<T>(tr + 64 * kt + 16 * pitch, 8 * pitch);
                f32x16 add = mfma16(k0, e[0], zero16());
#pragma unroll
                for (int r = 0; r < 16; ++r) S[kt][r] *= whole;
                S[kt] = mfma16(k0, h[0], S[kt]);
                add = mfma16(k1, e[1], add);
                S[kt] = mfma16(k1, h[1], S[kt]);
                if (Low<T>::THREE) {
                    add = mfma16(k0, f[0], add);
                    S[kt] = mfma16(k1, f[1], S[kt]);
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) S[kt][r] += add[r] * (1.f / Low<T>::SCALE);
            }
        }
    }
};

// What lies in accumulator registers (weighted pairs, a state), contracted over them, as a sum of two 16-bit operands: 2^-17
// of a bfloat16 one is lost, 2^-22 of a half (or 2^-36).  One operand alone would be rounded as coarsely as the result is:
// sqrt(2) of its error in all (2.35e-3 in place of 1.66e-3 in bfloat16).  Kernel time with one and with two operands, forward
// and backward: 2 x 8192 x 8 x 64 99 and 107 us, 16384 x 8 x 128 in half 238 and 300, 32 x 500 x 8 x 64 88 and 105.
// A third bfloat16 operand takes 7 % more (16 frames of 16384 sites 326 and 349 us, 2 x 8192 x 8 x 64 107 and 114) and leaves the
// error at 1.66e-3: what two lose moves one result in some three thousand across a border between two values.
template <typename T>
struct FineOperand {
    x8_t<T> h[2], e[2];
    __device__ __forceinline__ explicit FineOperand(const f32x16& p) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                float x = p[8 * s + j], y = p[8 * s + j + 1];
                Two<T>::take(h[s], j, x, y);
                Two<T>::round(e[s], j, x, y);
            }
    }
    // o + (a0 | a1) times this
    __device__ __forceinline__ f32x16 times(const x8_t<T>& a0, const x8_t<T>& a1, f32x16 o) const {
        f32x16 add = mfma16(a0, e[0], zero16());
        o = mfma16(a0, h[0], o);
        add = mfma16(a1, e[1], add);
        o = mfma16(a1, h[1], o);
#pragma unroll
        for (int r = 0; r < 16; ++r) o[r] += add[r] * (1.f / Low<T>::SCALE);
        return o;
    }
};

// Rows of one head, 32 tokens at a time: a buffer resource per tile, based on the tile's first row in memory, and 32-bit
// lane offsets that stay the same from tile to tile; rows past the tile's last token get an offset past the resource's
// end, which loads as zero and is not stored.  The tokens run backwards in memory where REVERSE.
struct Rows {
    const char* base;
    long long pitch;            // bytes
    unsigned records;           // bytes of a tile

    __device__ __forceinline__ Rows(const void* p, const Strides& s, long long bb, long long ii, int head, int col0, int width)
        : base(static_cast<const char*>(p) + 2 * (bb * s.b + ii * s.i + head * s.h + col0)), pitch(2 * s.n),
          records((unsigned)(31 * 2 * s.n) + 2 * width) {}
    // of a tile that has tokens; nothing is read where it has none
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t tile(int first, bool any = true) const {
        return vdmi_rsrc(base + first * pitch, any ? records : 0u);
    }
    // offset of column byte `col` of token `row` of a tile of cnt tokens
    __device__ __forceinline__ unsigned at(int row, int cnt, bool reverse, int col) const {
        const unsigned off = (unsigned)(reverse ? cnt - 1 - row : row) * (unsigned)pitch + col;
        return row < cnt ? off : NOWHERE;
    }
};

// a wave's place: (sequence, head, segment, 32-column slice) and its tokens
struct Place {
    int slice, head, seg, len, t_begin, t_stop, t_end;
    long long seq, bb, ii;
    template <typename A>
    __device__ __forceinline__ Place(const A& a, unsigned w, unsigned slices, unsigned segs) {
        slice = (int)(w % slices); w /= slices;
        const unsigned r = w / (unsigned)a.heads;
        head = (int)(w - r * (unsigned)a.heads);
        const unsigned sq = r / segs;
        seg = (int)(r - sq * segs);
        const unsigned ob = sq / (unsigned)a.inner;
        seq = sq;
        bb = ob;
        ii = sq - ob * (unsigned)a.inner;
        len = a.n;
        if (a.lengths) len = min(max(a.lengths[seq], 0), a.n);
        t_begin = seg * a.seg_len;
        t_stop = min(a.n, t_begin + a.seg_len);
        t_end = min(len, t_stop);
    }
    // the segment's rows behind the sequence's end become zeros
    template <typename T>
    __device__ __forceinline__ void clear(void* o, const Strides& s, int lane) const {
        x8_t<T> z;
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = (T)0.f;
        T* p = static_cast<T*>(o) + bb * s.b + ii * s.i + head * s.h + 32 * slice + 8 * (lane & 3);
        for (int t = max(len, t_begin) + (lane >> 2); t < t_stop; t += 16) *reinterpret_cast<x8_t<T>*>(p + t * s.n) = z;
    }
};

// transposed reads of a [token][column] image: lane 4 q + p of a 16-lane group supplies row q, four columns; its half's
// contraction values are rows 4 half + 0..3 and + 8 (accumulator-row order), the column pieces in swapped order (see above)
__device__ __forceinline__ int tr_offset(int lane, int pitch) {
    const int g16 = lane >> 4, tq = (lane >> 2) & 3, tp = lane & 3;
    return (4 * (g16 >> 1) + tq) * pitch + (16 * (g16 & 1) + 4 * (((tp & 1) << 1) | (tp >> 1))) * 2;
}

// WHAT: the outputs; only the segments' states
enum { OUTPUTS, STATES };

template <typename T, int D, int WHAT>
__global__ __launch_bounds__(DW * 64, D == 128 && WHAT != STATES ? 1 : 2)
void decay_scan_kernel(const ScanArgs a) {
    constexpr bool STATE_ONLY = WHAT == STATES;
    typedef x8_t<T> x8;
    constexpr int KS = D / 16, KT = D / 32, KP = 2 * D + 16, RS = 512 / D;      // RS: rows that 64 16-byte pieces cover
    __shared__ __attribute__((aligned(16))) char kimg_all[DW][32 * KP];
    __shared__ __attribute__((aligned(16))) char vimg_all[DW][32 * VP];
    __shared__ __attribute__((aligned(16))) float uw_all[DW][32];
    const int lane = threadIdx.x & 63, half = lane >> 5, l31 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    char* kimg = kimg_all[wave];
    char* vimg = vimg_all[wave];
    const unsigned w = blockIdx.x * DW + wave;
    if (w >= a.tasks) return;
    const Place at(a, w, KT, STATE_ONLY && !a.s_out ? a.nseg - 1 : a.nseg);     // nobody reads the last segment's sum
    const bool reverse = a.reverse;
    const Rows qr(a.q, a.qs, at.bb, at.ii, at.head, 0, D), kr(a.k, a.ks, at.bb, at.ii, at.head, 0, D),
        vr(a.v, a.vs, at.bb, at.ii, at.head, 32 * at.slice, 32), orow(a.o, a.os, at.bb, at.ii, at.head, 32 * at.slice, 32);
    if (!STATE_ONLY) at.clear<T>(a.o, a.os, lane);

    x8 kreg[KS], vreg[2], q[KS];
    unsigned kofs[KS], vofs[2], qofs;
    auto offsets = [&](int cnt) {
#pragma unroll
        for (int i = 0; i < KS; ++i) kofs[i] = kr.at(lane / (D / 8) + RS * i, cnt, reverse, 16 * (lane % (D / 8)));
#pragma unroll
        for (int i = 0; i < 2; ++i) vofs[i] = vr.at(16 * i + (lane >> 2), cnt, reverse, 16 * (lane & 3));
        qofs = qr.at(l31, cnt, reverse, 16 * half);
    };
    auto first_row = [&](int t0, int cnt) { return reverse ? at.len - t0 - cnt : t0; };
    auto load_kv = [&](int t0, int cnt) {
        const auto rk = kr.tile(first_row(t0, cnt), cnt > 0), rv = vr.tile(first_row(t0, cnt), cnt > 0);
#pragma unroll
        for (int i = 0; i < KS; ++i) kreg[i] = load16<T>(rk, kofs[i]);
#pragma unroll
        for (int i = 0; i < 2; ++i) vreg[i] = load16<T>(rv, vofs[i]);
    };
    auto load_q = [&](int t0, int cnt) {
        const auto rq = qr.tile(first_row(t0, cnt), cnt > 0);
#pragma unroll
        for (int i = 0; i < KS; ++i) q[i] = load16<T>(rq, qofs + 32 * i);
    };
    const char* ktr = kimg + tr_offset(lane, KP);
    const char* vtr = vimg + tr_offset(lane, VP);

    int cnt = min(32, at.t_end - at.t_begin);
    if (cnt > 0) {
        offsets(cnt);
        load_kv(at.t_begin, cnt);
        if constexpr (!STATE_ONLY) load_q(at.t_begin, cnt);
    }
    const float l2 = log2_decay(a.log_decay, at.head);
    const long long state0 = (at.seq * a.heads + at.head) * (long long)(D * D);
    // this lane's elements of S: row 32 kt + 16 (r >> 3) + 8 half + (r & 7), column 32 slice + swap23(l31)
    const int s_col = (32 * at.slice + swap23(l31)) * (a.rs == 1 ? D : 1);
    f32x16 S[KT];
    {
        const float* src = nullptr;
        float mul = 1.f;
        if (!STATE_ONLY) {
            if (a.nseg > 1) src = a.seg + (state0 * a.nseg + (long long)at.seg * (D * D));
            else if (a.s_in) { src = a.s_in + state0; mul = a.s_in_mul; }
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) S[kt] = zero16();
        if (src && a.rs == 1) {             // a column's rows are contiguous: eight at a time
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>(src + s_col + 32 * kt + 16 * (q >> 1) + 8 * half + 4 * (q & 1));
#pragma unroll
                    for (int e = 0; e < 4; ++e) S[kt][4 * q + e] = x[e] * mul;
                }
        } else if (src) {
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int r = 0; r < 16; ++r) S[kt][r] = src[(32 * kt + 16 * (r >> 3) + 8 * half + (r & 7)) * D + s_col] * mul;
        }
    }
    // decays: of a pair (register = key, lane = query), of the state towards a query, of a token towards the tile's end
    float dw[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int gap = l31 - acc_row(r, half);
        dw[r] = gap >= 0 ? a.m * __builtin_amdgcn_exp2f(l2 * (float)gap) : 0.f;
    }
    const float ow = a.m * __builtin_amdgcn_exp2f(l2 * (float)(l31 + a.e_out));
    float* uw = uw_all[wave];
    auto token_decays = [&](int cnt) {
        if (half == 0) uw[l31] = __builtin_amdgcn_exp2f(l2 * (float)(max(cnt - 1 - l31, 0) + a.e_u));
    };
    token_decays(32);
    float whole = __builtin_amdgcn_exp2f(l2 * 32.f);

    // the rest of a tile's work is one basic block (what the last tile needs comes first, the next tile's rows are asked for
    // whether there is one or not): its phases depend on each other in chains that only overlap if they are scheduled together
    for (int t0 = at.t_begin; t0 < at.t_end; t0 += 32) {
        cnt = min(32, at.t_end - t0);
        const int next = max(min(32, at.t_end - t0 - 32), 0);
        if (cnt < 32) {
            token_decays(cnt);
            whole = __builtin_amdgcn_exp2f(l2 * (float)cnt);
        }
        if (next < 32) offsets(next);
#pragma unroll
        for (int i = 0; i < KS; ++i) *reinterpret_cast<x8*>(kimg + (lane / (D / 8) + RS * i) * KP + 16 * (lane % (D / 8))) = kreg[i];
#pragma unroll
        for (int i = 0; i < 2; ++i) *reinterpret_cast<x8*>(vimg + (16 * i + (lane >> 2)) * VP + 16 * (lane & 3)) = vreg[i];
        wave_lds_order();
        load_kv(t0 + 32, next);
        __builtin_amdgcn_sched_barrier(0);          // not later: a tile's work is what covers them
        const x8 v0 = tr_operand<T>(vtr, 8 * VP), v1 = tr_operand<T>(vtr + 16 * VP, 8 * VP);
        const Split<T> sv(v0, v1, uw, half);
        if (!STATE_ONLY) {
            f32x16 st = zero16(), o = zero16(), low = zero16();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const x8 kf = *reinterpret_cast<const x8*>(kimg + l31 * KP + 32 * ks + 16 * half);
                st = mfma16(kf, q[ks], st);
                const FineOperand<T> state(S[ks >> 1]);
                o = mfma16(state.h[ks & 1], q[ks], o);
                low = mfma16(state.e[ks & 1], q[ks], low);
            }
            load_q(t0 + 32, next);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                st[r] = weigh(st[r], dw[r]);
                o[r] = (o[r] + low[r] * (1.f / Low<T>::SCALE)) * ow;
            }
            o = FineOperand<T>(st).times(v0, v1, o);
            // through LDS (the tile's v image is in registers by now) to 16-byte stores, four lanes on a row's 64 bytes
            wave_lds_order();
            *reinterpret_cast<x8*>(vimg + l31 * VP + 16 * half) = acc_operand<T>(o, 0);
            *reinterpret_cast<x8*>(vimg + l31 * VP + 32 + 16 * half) = acc_operand<T>(o, 1);
            wave_lds_order();
            const auto ro = orow.tile(first_row(t0, cnt));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = 16 * i + (lane >> 2);
                store16<T>(ro, orow.at(row, cnt, reverse, 16 * (lane & 3)), *reinterpret_cast<const x8*>(vimg + row * VP + 16 * (lane & 3)));
            }
        }
        sv.update(S, whole, ktr, KP);
        wave_lds_order();               // the images and weights are read: the next tile may come
    }
    float* dst = nullptr;
    float mul = 1.f;
    if (STATE_ONLY) dst = a.seg + (state0 * a.nseg + (long long)at.seg * (D * D));
    else if (a.s_out && a.nseg == 1) { dst = a.s_out + state0; mul = a.s_out_mul; }
    if (dst) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int r = 0; r < 16; ++r) dst[(32 * kt + 16 * (r >> 3) + 8 * half + (r & 7)) * D + s_col] = S[kt][r] * mul;
    }
}

// dk and dv in one walk backward in time: both read q, k, v and do, and what one of them needs of R = dS / m by columns the
// other needs by rows.  A wave computes 32 columns of dv and the same 32 columns of dk and holds R[all dk][its columns of
// dv] and R^T[all dv][its columns of dk].  Two walks, one for each, are two scans of 20 us and another pass over the segments
// of 18 where this takes 32 (2 x 8192 tokens, 8 heads of 64).  With 64 features dv's half of a tile comes before dk's, which
// fits the registers (whole backward, halves together and apart: 2 x 8192 x 8 x 64 79 and 66 us, in half 91 and 67; 32 x 500 x
// 8 x 64 131 and 73).  With 32 and 128 features it makes no difference (8 x 4000 x 8 x 32: 50.6 and 51.0 us; 16384 x 8 x 128, in
// bfloat16 160 both ways); halves together are the shorter chain there.
template <typename T, int D>
__global__ __launch_bounds__(DW * 64, D <= 64 ? 2 : 1) void decay_grad_kernel(const GradArgs a) {
    typedef x8_t<T> x8;
    constexpr int KS = D / 16, KT = D / 32, KP = 2 * D + 16, RS = 512 / D;
    __shared__ __attribute__((aligned(16))) char qimg_all[DW][32 * KP];
    __shared__ __attribute__((aligned(16))) char gimg_all[DW][32 * KP];
    __shared__ __attribute__((aligned(16))) float uw_all[DW][32];
    __shared__ float fade_all[D == 128 || (D == 64 && !Low<T>::THREE) ? DW : 1][64];
    const int lane = threadIdx.x & 63, half = lane >> 5, l31 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    char* qimg = qimg_all[wave];
    char* gimg = gimg_all[wave];
    const unsigned w = blockIdx.x * DW + wave;
    if (w >= a.tasks) return;
    const Place at(a, w, KT, a.nseg);
    const Rows qr(a.q, a.qs, at.bb, at.ii, at.head, 0, D), kr(a.k, a.ks, at.bb, at.ii, at.head, 0, D),
        vr(a.v, a.vs, at.bb, at.ii, at.head, 0, D), gr(a.g, a.gs, at.bb, at.ii, at.head, 0, D),
        dkr(a.dk, a.dks, at.bb, at.ii, at.head, 32 * at.slice, 32), dvr(a.dv, a.dvs, at.bb, at.ii, at.head, 32 * at.slice, 32);
    at.clear<T>(a.dk, a.dks, lane);
    at.clear<T>(a.dv, a.dvs, lane);

    x8 qreg[KS], greg[KS], k[KS], v[KS];
    // 128 features, and 64 of halfs, leave no registers for the loads' offsets and the pairs' decays: the former are computed
    // again for every tile, the latter read from LDS.  (From scratch memory, where the compiler would put them, each one
    // waits for every load in flight: 2 x 8192 x 8 x 64 in half, 49 us in place of 33.)
    constexpr bool KEEP = D == 32 || (D == 64 && Low<T>::THREE), HALVES = D == 64;
    unsigned qofs[KEEP ? KS : 1], gofs[KEEP ? KS : 1], kofs, vofs;
    auto row_at = [&](const Rows& r, int i, int cnt) { return r.at(lane / (D / 8) + RS * i, cnt, true, 16 * (lane % (D / 8))); };
    auto offsets = [&](int cnt) {
#pragma unroll
        for (int i = 0; KEEP && i < KS; ++i) {
            qofs[i] = row_at(qr, i, cnt);
            gofs[i] = row_at(gr, i, cnt);
        }
        kofs = kr.at(l31, cnt, true, 16 * half);
        vofs = vr.at(l31, cnt, true, 16 * half);
    };
    auto load_qg = [&](int t0, int cnt) {
        const auto rq = qr.tile(at.len - t0 - cnt, cnt > 0), rg = gr.tile(at.len - t0 - cnt, cnt > 0);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            qreg[i] = load16<T>(rq, KEEP ? qofs[i] : row_at(qr, i, cnt));
            greg[i] = load16<T>(rg, KEEP ? gofs[i] : row_at(gr, i, cnt));
        }
    };
    auto load_k = [&](int t0, int cnt) {
        const auto r = kr.tile(at.len - t0 - cnt, cnt > 0);
#pragma unroll
        for (int i = 0; i < KS; ++i) k[i] = load16<T>(r, kofs + 32 * i);
    };
    auto load_v = [&](int t0, int cnt) {
        const auto r = vr.tile(at.len - t0 - cnt, cnt > 0);
#pragma unroll
        for (int i = 0; i < KS; ++i) v[i] = load16<T>(r, vofs + 32 * i);
    };
    const char* qtr = qimg + tr_offset(lane, KP);
    const char* gtr = gimg + tr_offset(lane, KP);

    int cnt = min(32, at.t_end - at.t_begin);
    if (cnt > 0) {
        offsets(cnt);
        load_qg(at.t_begin, cnt);
        load_k(at.t_begin, cnt);
        load_v(at.t_begin, cnt);
    }
    const float l2 = log2_decay(a.log_decay, at.head);
    const long long state0 = (at.seq * a.heads + at.head) * (long long)(D * D);
    const int col = 32 * at.slice + swap23(l31);
    f32x16 R[KT], Rt[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) R[kt] = Rt[kt] = zero16();
    const float* src = a.nseg > 1 ? a.seg + (state0 * a.nseg + (long long)at.seg * (D * D)) : a.s_in ? a.s_in + state0 : nullptr;
    if (src) {
        const float mul = a.nseg > 1 ? 1.f : 1.f / a.m;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = 32 * kt + 16 * (r >> 3) + 8 * half + (r & 7);
                R[kt][r] = src[row * D + col] * mul;
                Rt[kt][r] = src[col * D + row] * mul;
            }
    }
    // the decays of pairs as in the scan; register = query, lane = key, both counted backward in time.  In LDS by gap + 32
    // where there are no registers for them
    float dw[KEEP ? 16 : 1];
    float* fade = fade_all[KEEP ? 0 : wave];
    if constexpr (KEEP) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int gap = l31 - acc_row(r, half);
            dw[r] = gap >= 0 ? a.m * __builtin_amdgcn_exp2f(l2 * (float)gap) : 0.f;
        }
    } else {
        fade[lane] = lane < 32 ? 0.f : a.m * __builtin_amdgcn_exp2f(l2 * (float)(lane - 32));
    }
    const float* fades = fade + 32 + l31 - 4 * half;
    const float ow = a.m * __builtin_amdgcn_exp2f(l2 * (float)l31);
    float* uw = uw_all[wave];
    auto token_decays = [&](int cnt) {
        if (half == 0) uw[l31] = __builtin_amdgcn_exp2f(l2 * (float)(max(cnt - 1 - l31, 0) + 1));
    };
    token_decays(32);
    float whole = __builtin_amdgcn_exp2f(l2 * 32.f);

    for (int t0 = at.t_begin; t0 < at.t_end; t0 += 32) {
        cnt = min(32, at.t_end - t0);
        const int next = max(min(32, at.t_end - t0 - 32), 0);
        if (cnt < 32) {
            token_decays(cnt);
            whole = __builtin_amdgcn_exp2f(l2 * (float)cnt);
        }
        if (next < 32) offsets(next);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            *reinterpret_cast<x8*>(qimg + (lane / (D / 8) + RS * i) * KP + 16 * (lane % (D / 8))) = qreg[i];
            *reinterpret_cast<x8*>(gimg + (lane / (D / 8) + RS * i) * KP + 16 * (lane % (D / 8))) = greg[i];
        }
        wave_lds_order();
        load_qg(t0 + 32, next);
        __builtin_amdgcn_sched_barrier(0);
        // [query x key]: q k, do v;  [column x key]: R k, R^T v
        auto products = [&](const char* img, const x8 (&x)[KS], const f32x16 (&r)[KT], int ks, f32x16& p, f32x16& o, f32x16& low) {
            p = mfma16(*reinterpret_cast<const x8*>(img + l31 * KP + 32 * ks + 16 * half), x[ks], p);
            const FineOperand<T> f(r[ks >> 1]);
            o = mfma16(f.h[ks & 1], x[ks], o);
            low = mfma16(f.e[ks & 1], x[ks], low);
        };
        auto weights = [&](f32x16& p, f32x16& o, const f32x16& low) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                p[r] = weigh(p[r], KEEP ? dw[r] : fades[-acc_row(r, 0)]);
                o[r] = (o[r] + low[r] * (1.f / Low<T>::SCALE)) * ow;
            }
        };
        auto slice = [&](x8& x0, x8& x1, const char* tr) {
            x0 = tr_operand<T>(tr + 64 * at.slice, 8 * KP);
            x1 = tr_operand<T>(tr + 64 * at.slice + 16 * KP, 8 * KP);
        };
        f32x16 p = zero16(), dp = zero16(), ov = zero16(), ok = zero16(), lv = zero16(), lk = zero16();
        x8 g0, g1, q0, q1, rok[2], rov[2];
        if constexpr (HALVES) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) products(qimg, k, R, ks, p, ov, lv);
            load_k(t0 + 32, next);
            __builtin_amdgcn_sched_barrier(0);
            weights(p, ov, lv);
            slice(g0, g1, gtr);
            ov = FineOperand<T>(p).times(g0, g1, ov);
            Split<T>(g0, g1, uw, half).update(R, whole, qtr, KP);
            rov[0] = acc_operand<T>(ov, 0);
            rov[1] = acc_operand<T>(ov, 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) products(gimg, v, Rt, ks, dp, ok, lk);
            load_v(t0 + 32, next);
            __builtin_amdgcn_sched_barrier(0);
            weights(dp, ok, lk);
            slice(q0, q1, qtr);
            ok = FineOperand<T>(dp).times(q0, q1, ok);
            Split<T>(q0, q1, uw, half).update(Rt, whole, gtr, KP);
            rok[0] = acc_operand<T>(ok, 0);
            rok[1] = acc_operand<T>(ok, 1);
        } else {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                products(qimg, k, R, ks, p, ov, lv);
                products(gimg, v, Rt, ks, dp, ok, lk);
            }
            load_k(t0 + 32, next);
            load_v(t0 + 32, next);
            __builtin_amdgcn_sched_barrier(0);
            weights(p, ov, lv);
            weights(dp, ok, lk);
            slice(g0, g1, gtr);
            slice(q0, q1, qtr);
            ov = FineOperand<T>(p).times(g0, g1, ov);
            ok = FineOperand<T>(dp).times(q0, q1, ok);
            rok[0] = acc_operand<T>(ok, 0);
            rok[1] = acc_operand<T>(ok, 1);
            rov[0] = acc_operand<T>(ov, 0);
            rov[1] = acc_operand<T>(ov, 1);
            if (!KEEP) __builtin_amdgcn_sched_barrier(0);
            Split<T>(g0, g1, uw, half).update(R, whole, qtr, KP);
            if (!KEEP) __builtin_amdgcn_sched_barrier(0);
            Split<T>(q0, q1, uw, half).update(Rt, whole, gtr, KP);
        }
        // the images are done with: results through them to 16-byte stores, four lanes on a row's 64 bytes
        wave_lds_order();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            *reinterpret_cast<x8*>(qimg + l31 * VP + 32 * s + 16 * half) = rok[s];
            *reinterpret_cast<x8*>(gimg + l31 * VP + 32 * s + 16 * half) = rov[s];
        }
        wave_lds_order();
        const auto rk = dkr.tile(at.len - t0 - cnt), rv = dvr.tile(at.len - t0 - cnt);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = 16 * i + (lane >> 2);
            store16<T>(rk, dkr.at(row, cnt, true, 16 * (lane & 3)), *reinterpret_cast<const x8*>(qimg + row * VP + 16 * (lane & 3)));
            store16<T>(rv, dvr.at(row, cnt, true, 16 * (lane & 3)), *reinterpret_cast<const x8*>(gimg + row * VP + 16 * (lane & 3)));
        }
        wave_lds_order();
    }
    if (a.s_out && a.nseg == 1) {
        float* dst = a.s_out + state0;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int r = 0; r < 16; ++r) dst[(32 * kt + 16 * (r >> 3) + 8 * half + (r & 7)) * D + col] = R[kt][r] * a.m;
    }
}

// Along the segments of a sequence: sums of single segments -> states at their starts, and the state after the last one.
// One thread per element of S; bound by reading and writing the segment states once (32 segments of 8 heads of 128 x 128:
// 33.5 MB in 8.4 us, 4.0 TB/s, with eight segments' loads ahead; 32 ahead 11.8).
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
// rows, pairs of different sequences weigh nothing, and the backward pass does all three gradients from one read of q, k,
// v and do (dP^T = V dO^T with lane = query for dq; P = Q K^T and dP = dO V^T with lane = key for dv and dk).  A wave
// computes one (tile, head) and ends: enough of them share a SIMD to cover each other's loads.
// A row that is not finite must not reach the other sequences of its tile (zero times infinity in the second product):
// such a tile is computed once per sequence with the others' rows as zeros.  Rows that no sequence of the tile fills
// (32 - n of them where n > 16) are zeros too.
// ------------------------------------------------------------------------------------------------------------------
struct Strides32 { unsigned b, i, n; };            // bytes

struct ShortArgs {
    const void* q; const void* k; const void* v; const void* g;        // g: gradient of o
    void* o; void* dq; void* dk; void* dv;                             // dq null or dk and dv null: not wanted
    Strides32 qs, ks, vs, gs, os, dqs, dks, dvs;
    long long qh, kh, vh, gh, oh, dqh, dkh, dvh;                        // head strides, elements
    const float* log_decay;
    const int* lengths;
    int n, heads, per_tile, tiles;
    unsigned inner, magic, inv_n;       // row / n = row * inv_n >> 16 for row < 32
    int shift;                          // seq / inner = umulhi(seq, magic) >> shift; shift < 0: inner is 1
    float m;
    unsigned nseq;
};

template <typename T, int N>
__device__ __forceinline__ bool finite(const x8_t<T> (&x)[N]) {
    typedef __attribute__((ext_vector_type(2))) unsigned short us2;
    us2 top = {0, 0};
#pragma unroll
    for (int s = 0; s < N; ++s) {
        const vdmi_u4 w = __builtin_bit_cast(vdmi_u4, x[s]);
#pragma unroll
        for (int i = 0; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(us2, w[i] & 0x7fff7fffu));
    }
    return top[0] < Pack<T>::EXP && top[1] < Pack<T>::EXP;
}

// NH heads of D features side by side in memory are one row of W columns, moved as 16-byte pieces with all lanes of a row
// next to each other and transposed to operands through LDS.  Measured over 16 frames of 16384 sites with 8 heads of 32
// features (537 MB forward, 940 MB backward): 123 us and 211 us, 4.4 and 4.5 TB/s; before the pairs were two operands
// each 122 and 197 us, one head at a time (64-byte rows) 127 and 234, every lane loading and storing its own token's row as
// operands (32 bytes of a row per instruction) 150 and 283.
constexpr int short_waves(int d, bool bwd) { return d == 128 && bwd ? 1 : 2; }

template <typename T, int D, int NH, bool BWD>
__global__ __launch_bounds__((short_waves(D, BWD) * 64), D == 128 ? 1 : 2) void decay_short_kernel(const ShortArgs a) {
    typedef x8_t<T> x8;
    constexpr int SW = short_waves(D, BWD), W = D * NH, KS = D / 16, DT = D / 32, P = 2 * W + 16, NT = BWD ? 4 : 3;
    constexpr int PR = W / 8, RPI = 64 / PR, NI = 32 / RPI;       // 16-byte pieces of a row, rows per load, loads
    __shared__ __attribute__((aligned(16))) char img_all[SW][NT][32 * P];       // q, k, v, do; results take their places
    __shared__ float fade_all[SW][64];
    const int lane = threadIdx.x & 63, half = lane >> 5, l31 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const unsigned groups = (unsigned)a.heads / NH, unit = blockIdx.x * SW + wave, tile = unit / groups;
    if (tile >= (unsigned)a.tiles) return;
    const int head0 = (int)(unit - tile * groups) * NH, n = a.n;
    char (*im)[32 * P] = img_all[wave];

    // rows RPI i + lane / PR of the tile, piece lane % PR: their sequence, whether they are the call's, whether live
    const int piece = lane % PR;
    unsigned bb[NI], ii[NI], tt[NI];
    bool mine[NI], live[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const unsigned row = RPI * i + lane / PR, slot = row * a.inv_n >> 16;
        tt[i] = row - slot * n;
        unsigned seq = tile * (unsigned)a.per_tile + slot;
        mine[i] = slot < (unsigned)a.per_tile && seq < a.nseq;     // rows behind the tile's last sequence are nobody's
        seq = min(seq, a.nseq - 1);     // a row that is not there loads another one; nothing of it is stored
        bb[i] = a.shift < 0 ? seq : __umulhi(seq, a.magic) >> a.shift;
        ii[i] = seq - bb[i] * a.inner;
        live[i] = mine[i] && (!a.lengths || (int)tt[i] < a.lengths[seq]);
    }
    auto row_of = [&](const void* p, const Strides32& s, long long h, int i) {
        return const_cast<x8*>(reinterpret_cast<const x8*>(static_cast<const char*>(p) + 2 * head0 * h + (unsigned long long)bb[i] * s.b +
                                                           (unsigned long long)ii[i] * s.i + (unsigned long long)(tt[i] * s.n + 16 * piece)));
    };
    x8 zero8;
#pragma unroll
    for (int j = 0; j < 8; ++j) zero8[j] = (T)0.f;
    // rows of the sequences [s_lo, s_hi) of the tile into the images, the others as zeros; whether all of it is finite
    auto load = [&](int s_lo, int s_hi) {
        x8 x[NT][NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            x[0][i] = *row_of(a.q, a.qs, a.qh, i);
            x[1][i] = *row_of(a.k, a.ks, a.kh, i);
            x[2][i] = *row_of(a.v, a.vs, a.vh, i);
            if constexpr (BWD) x[3][i] = *row_of(a.g, a.gs, a.gh, i);
        }
        if (a.lengths || s_hi - s_lo < a.per_tile || n * a.per_tile < 32) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int slot = (int)((RPI * i + lane / PR) * a.inv_n >> 16);
                if (!live[i] || slot < s_lo || slot >= s_hi) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) x[t][i] = zero8;
                }
            }
        }
        bool fine = true;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (BWD || t == 2) fine = fine & finite<T>(x[t]);
#pragma unroll
            for (int i = 0; i < NI; ++i) *reinterpret_cast<x8*>(im[t] + (RPI * i + lane / PR) * P + 16 * piece) = x[t][i];
        }
        return fine;
    };
    auto store = [&](const char* src, void* dst, const Strides32& s, long long h, int s_lo, int s_hi) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int slot = (int)((RPI * i + lane / PR) * a.inv_n >> 16);
            x8 x = *reinterpret_cast<const x8*>(src + (RPI * i + lane / PR) * P + 16 * piece);
            // whatever the sequence's own tokens made of its padding.  (lengths are read again: live[] kept until here takes
            // the registers of 3 % of the backward.)
            if (a.lengths && (int)tt[i] >= a.lengths[min(tile * (unsigned)a.per_tile + slot, a.nseq - 1)]) x = zero8;
            if (mine[i] && slot >= s_lo && slot < s_hi) *row_of(dst, s, h, i) = x;
        }
    };

    const int slot = (int)(l31 * a.inv_n >> 16), ti = l31 - slot * n;
    const bool in_tile = slot < a.per_tile;
    float* fade = fade_all[wave];
    const int tr_off = tr_offset(lane, P);
    // contraction over the features of two row sets, times the decays of (register, lane) = (key, query) or, by_key, (query,
    // key): pairs within a sequence, the key not after the query
    auto pairs = [&](const char* x, const char* y, bool by_key) {
        f32x16 p = zero16(), p2 = zero16();
#pragma unroll
        for (int s = 0; s < KS; s += 2) {
            const int at = l31 * P + 32 * s + 16 * half;
            p = mfma16(*reinterpret_cast<const x8*>(x + at), *reinterpret_cast<const x8*>(y + at), p);
            p2 = mfma16(*reinterpret_cast<const x8*>(x + at + 32), *reinterpret_cast<const x8*>(y + at + 32), p2);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int t = acc_row(r, half), gap = by_key ? t - l31 : l31 - t;
            const float w = (unsigned)gap <= (unsigned)(by_key ? n - 1 - ti : ti) && in_tile ? fade[32 + gap] : 0.f;
            p[r] = weigh(p[r] + p2[r], w);
        }
        return p;
    };
    // (columns of an image)^T x pairs into the same columns of another one
    auto product = [&](const char* src, const f32x16& p, char* dst) {
        const FineOperand<T> pairs(p);
        f32x16 o[DT];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
            o[dt] = pairs.times(tr_operand<T>(src + tr_off + 64 * dt, 8 * P), tr_operand<T>(src + tr_off + 64 * dt + 16 * P, 8 * P), zero16());
        wave_lds_order();
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int s = 0; s < 2; ++s) *reinterpret_cast<x8*>(dst + l31 * P + 64 * dt + 32 * s + 16 * half) = acc_operand<T>(o[dt], s);
    };
    auto compute = [&](int s_lo, int s_hi) {
#pragma unroll
        for (int j = 0; j < NH; ++j) {
            wave_lds_order();
            // m lambda^gap by gap + 32
            fade[lane] = a.m * __builtin_amdgcn_exp2f(log2_decay(a.log_decay, head0 + j) * (float)max(lane - 32, 0));
            wave_lds_order();
            const int c = 2 * D * j;
            if constexpr (!BWD) {
                product(im[2] + c, pairs(im[1] + c, im[0] + c, false), im[0] + c);
            } else {
                const f32x16 p = pairs(im[2] + c, im[3] + c, false);                    // [key x query]: v do
                const f32x16 pv = pairs(im[0] + c, im[1] + c, true);                    // [query x key]: q k
                const f32x16 pk = pairs(im[3] + c, im[2] + c, true);                    // do v
                if (a.dq) product(im[1] + c, p, im[2] + c);                             // dq, where v was
                if (a.dk) {
                    product(im[3] + c, pv, im[3] + c);                                  // dv, where do was
                    product(im[0] + c, pk, im[0] + c);                                  // dk, where q was
                }
            }
        }
        wave_lds_order();
        if constexpr (!BWD) {
            store(im[0], a.o, a.os, a.oh, s_lo, s_hi);
        } else {
            if (a.dq) store(im[2], a.dq, a.dqs, a.dqh, s_lo, s_hi);
            if (a.dk) {
                store(im[3], a.dv, a.dvs, a.dvh, s_lo, s_hi);
                store(im[0], a.dk, a.dks, a.dkh, s_lo, s_hi);
            }
        }
    };
    const bool fine = load(0, a.per_tile);
    if (a.per_tile == 1 || __builtin_amdgcn_ballot_w64(!fine) == 0) {
        compute(0, a.per_tile);
    } else {
        for (int pass = 0; pass < a.per_tile; ++pass) {
            wave_lds_order();
            load(pass, pass + 1);
            compute(pass, pass + 1);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------
// One more token of every sequence: S <- lambda S + k v^T in place, o = m q S.  Bound by reading and writing S once (8192
// sequences, 8 heads of 32: 545 MB in 100 us, 5.4 TB/s; one sequence, 8 heads of 64: 3.5 us, a launch's time).  A wave
// takes 32 columns of one (sequence, head): 8 rows x 128 contiguous bytes per load, all its loads in flight.
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

// the 32 rows of a tile within a 31-bit offset of each other
bool pitch_ok(const vdmi_rows4& r) { return r.n >= 0 && r.n <= VDMI_DECAY_MAX_PITCH; }

// the short-sequence kernel multiplies batch indexes with 32-bit byte strides
bool strides32_ok(const vdmi_rows4& r) { return r.b >= 0 && r.i >= 0 && r.b < 0x7fffffffLL && r.i < 0x7fffffffLL; }

// the backward divides by it: it and its reciprocal are normal numbers (zero, infinities and NaN are not)
bool scale_ok(float m) { return fabsf(m) >= 0x1p-126f && fabsf(m) <= 0x1p126f; }

int check_args(const vdmi_decay_args* a) {
    if (!a || !a->log_decay) return VDMI_E_ARG;
    if (a->dtype != VDMI_DT_BF16 && a->dtype != VDMI_DT_F16) return VDMI_E_ARG;
    if (!scale_ok(a->scale)) return VDMI_E_ARG;
    if (a->b <= 0 || a->inner <= 0 || a->n <= 0 || a->heads <= 0 || a->heads > 65535) return VDMI_E_SHAPE;
    if (a->d != 32 && a->d != 64 && a->d != 128) return VDMI_E_SHAPE;
    if ((long long)a->b * a->inner > 0x7fffffffLL / a->heads || a->n > (1 << 30)) return VDMI_E_SHAPE;
    if (!a->q.p || !a->k.p || !a->v.p) return VDMI_E_ARG;
    if (!rows_ok(a->q) || !rows_ok(a->k) || !rows_ok(a->v)) return VDMI_E_ALIGN;
    if (!pitch_ok(a->q) || !pitch_ok(a->k) || !pitch_ok(a->v)) return VDMI_E_SHAPE;
    return VDMI_OK;
}

// How the time axis is cut: waves = sequences x heads x d / 32 column slices x segments.  A tile is 1 to 4 us of steps that
// depend on each other, so few sequences are cut until every SIMD of the card has a wave (256 x 4 of them), down to one tile
// per segment; the walk along the segments is serial: beyond 64 of them they are 128 tokens or longer.  Two or three
// segments cost about what they save (k and v are read once more, the states written and read) unless they are long.
// Measured, bfloat16, forward / backward in us (sequences x tokens x heads x features: segments):
//     6 x 701 x 4 x 64:    1: 34/93    2: 34/66    4: 24/45    21: 19/31
//     1 x 1000 x 8 x 128:  1: 78/226   2: 65/146   8: 27/55    31: 22/41
//     2 x 8192 x 8 x 64:   1: 333/958  16: 49/94   32 (1024 waves): 36/65   64: 40/66
//     1 x 4000 x 8 x 32:   32: 20/31   64: 20/28   125: 26/33
//     32 x 500 x 8 x 64:   1: 28/73    2: 40/68        30 x 2048 x 8 x 64:  1: 88/260   2: 99/199
//     62 x 2048 x 8 x 64:  1: 129/322  2: 183/398      1 x 16384 x 8 x 128:  16: 121/280   32 (1024 waves): 78/160   64: 83/185
Plan plan(const vdmi_decay_args* a, bool states) {
    Plan p;
    p.nseq = (long long)a->b * a->inner;
    p.is_short = a->n <= 32 && !states;
    for (const vdmi_rows4* r : {&a->q, &a->k, &a->v, &a->o, &a->dout, &a->dq, &a->dk, &a->dv}) p.is_short = p.is_short && strides32_ok(*r);
    p.nseg = 1;
    p.seg_len = a->n;
    p.bytes = 0;
    if (p.is_short) return p;
    const long long waves = p.nseq * a->heads * (a->d / 32);
    long long want = std::min(1024 / waves, std::min<long long>(a->n / 32, std::max(64, a->n / 128)));
    if (want < 4 && a->n < 4 * a->d * want) want = 1;
    if (want > 1) {
        p.seg_len = (int)(((a->n + want - 1) / want + 31) / 32 * 32);
        p.nseg = (a->n + p.seg_len - 1) / p.seg_len;
    }
    if (p.nseg > 1) p.bytes = (size_t)p.nseq * a->heads * p.nseg * a->d * a->d * sizeof(float);
    return p;
}

bool wants_states(const vdmi_decay_args* a) { return a->state_in || a->state_out || a->dstate_in || a->dstate_out; }

Strides strides_of(const vdmi_rows4& r) { return Strides{r.b, r.i, r.n, r.h}; }

template <int WHAT>
int launch_scan(const ScanArgs& s, const vdmi_decay_args* a, const Plan& p, hipStream_t st) {
    ScanArgs x = s;
    const long long segs = WHAT == STATES && !x.s_out ? p.nseg - 1 : p.nseg;
    const long long tasks = p.nseq * a->heads * segs * (a->d / 32), wgs = (tasks + DW - 1) / DW;
    if (!launch_fits(wgs, DW * 64)) return VDMI_E_SHAPE;
    x.tasks = (unsigned)tasks;
    const dim3 grid((unsigned)wgs), block(DW * 64);
#define SCAN(T, D) hipLaunchKernelGGL((decay_scan_kernel<T, D, WHAT>), grid, block, 0, st, x)
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
    const int r = launch_scan<STATES>(s, a, p, st);
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
    s.rs = a->d;
    s.inner = a->inner; s.n = a->n; s.heads = a->heads;
    s.nseg = p.nseg; s.seg_len = p.seg_len;
    s.m = a->scale;
    return s;
}

Strides32 strides32(const vdmi_rows4& r) { return Strides32{(unsigned)(2 * r.b), (unsigned)(2 * r.i), (unsigned)(2 * r.n)}; }

int launch_short(const vdmi_decay_args* a, const Plan& p, bool bwd, hipStream_t st) {
    ShortArgs s = {};
    s.q = a->q.p; s.k = a->k.p; s.v = a->v.p; s.g = a->dout.p;
    s.o = a->o.p; s.dq = a->dq.p; s.dk = a->dk.p; s.dv = a->dv.p;
    s.qs = strides32(a->q); s.ks = strides32(a->k); s.vs = strides32(a->v); s.gs = strides32(a->dout);
    s.os = strides32(a->o); s.dqs = strides32(a->dq); s.dks = strides32(a->dk); s.dvs = strides32(a->dv);
    s.qh = a->q.h; s.kh = a->k.h; s.vh = a->v.h; s.gh = a->dout.h;
    s.oh = a->o.h; s.dqh = a->dq.h; s.dkh = a->dk.h; s.dvh = a->dv.h;
    s.log_decay = a->log_decay; s.lengths = a->lengths;
    s.n = a->n; s.heads = a->heads; s.per_tile = 32 / a->n;
    s.m = a->scale;
    s.nseq = (unsigned)p.nseq;
    s.tiles = (int)((p.nseq + s.per_tile - 1) / s.per_tile);
    // division by inner of numbers below 2^31: with 2^(l-1) < inner <= 2^l and magic = floor(2^(31+l) / inner) + 1 the
    // error of the quotient stays under 1 / inner
    s.inner = (unsigned)a->inner;
    s.shift = -1;
    if (a->inner > 1) {
        int l = 0;
        while ((1LL << l) < a->inner) ++l;
        s.magic = (unsigned)((1ULL << (31 + l)) / (unsigned)a->inner + 1);
        s.shift = l - 1;
    }
    s.inv_n = 65536u / a->n + 1;
    // two heads of 32 features next to each other in every tensor
    bool two = a->d == 32 && a->heads % 2 == 0;
    for (const vdmi_rows4* r : {&a->q, &a->k, &a->v, &a->o, &a->dout, &a->dq, &a->dk, &a->dv}) two = two && (!r->p || r->h == 32);
#define SHORT(T, D, NH, B) do { constexpr int sw = short_waves(D, B); \
    const long long wgs = ((long long)s.tiles * (a->heads / NH) + sw - 1) / sw; \
    if (!launch_fits(wgs, sw * 64)) return VDMI_E_SHAPE; \
    hipLaunchKernelGGL((decay_short_kernel<T, D, NH, B>), dim3((unsigned)wgs), dim3(sw * 64), 0, st, s); } while (0)
#define SHORT_D(T, B) do { if (two) SHORT(T, 32, 2, B); else if (a->d == 32) SHORT(T, 32, 1, B); else if (a->d == 64) SHORT(T, 64, 1, B); \
                           else SHORT(T, 128, 1, B); } while (0)
    if (a->dtype == VDMI_DT_BF16) { if (bwd) SHORT_D(__bf16, true); else SHORT_D(__bf16, false); }
    else { if (bwd) SHORT_D(_Float16, true); else SHORT_D(_Float16, false); }
#undef SHORT_D
#undef SHORT
    VDMI_LAUNCH_CHECK();
    return VDMI_OK;
}

int launch_grad(const vdmi_decay_args* a, const Plan& p, hipStream_t st) {
    GradArgs g = {};
    g.q = a->q.p; g.k = a->k.p; g.v = a->v.p; g.g = a->dout.p; g.dk = a->dk.p; g.dv = a->dv.p;
    g.qs = strides_of(a->q); g.ks = strides_of(a->k); g.vs = strides_of(a->v); g.gs = strides_of(a->dout);
    g.dks = strides_of(a->dk); g.dvs = strides_of(a->dv);
    g.log_decay = a->log_decay; g.lengths = a->lengths;
    g.s_in = a->dstate_in; g.s_out = a->dstate_out;
    g.seg = static_cast<const float*>(a->workspace);
    g.inner = a->inner; g.n = a->n; g.heads = a->heads; g.nseg = p.nseg; g.seg_len = p.seg_len;
    g.m = a->scale;
    const long long tasks = p.nseq * a->heads * p.nseg * (a->d / 32), wgs = (tasks + DW - 1) / DW;
    if (!launch_fits(wgs, DW * 64)) return VDMI_E_SHAPE;
    g.tasks = (unsigned)tasks;
    const dim3 grid((unsigned)wgs), block(DW * 64);
#define GRAD(T, D) hipLaunchKernelGGL((decay_grad_kernel<T, D>), grid, block, 0, st, g)
#define GRAD_D(T) do { if (a->d == 32) GRAD(T, 32); else if (a->d == 64) GRAD(T, 64); else GRAD(T, 128); } while (0)
    if (a->dtype == VDMI_DT_BF16) GRAD_D(__bf16); else GRAD_D(_Float16);
#undef GRAD
#undef GRAD_D
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
    if (!pitch_ok(a->o)) return VDMI_E_SHAPE;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const Plan p = plan(a, wants_states(a));
    if (p.is_short) return launch_short(a, p, false, st);
    if (p.bytes && (!a->workspace || a->workspace_bytes < (int64_t)p.bytes)) return VDMI_E_ARG;
    if (p.bytes && !aligned16(a->workspace)) return VDMI_E_ALIGN;
    ScanArgs s = scan_args(a, p);
    role(s, a->q, a->k, a->v, a->o);
    s.s_in = a->state_in;
    s.s_out = a->state_out;
    s.e_out = 1;
    const int r = segment_states(s, a, p, st);
    return r != VDMI_OK ? r : launch_scan<OUTPUTS>(s, a, p, st);
}

extern "C" int vdmi_decay_attn_bwd(const vdmi_decay_args* a, vdmi_stream stream) {
    const int ok = check_args(a);
    if (ok != VDMI_OK) return ok;
    // dk and dv come from one walk, which also ends in the gradient of the first state
    const bool want_q = a->dq.p, want_kv = a->dk.p;
    if (!a->dout.p || !(want_q || want_kv) || !a->dk.p != !a->dv.p || (a->dstate_out && !want_kv)) return VDMI_E_ARG;
    if (!rows_ok(a->dout) || (want_q && !rows_ok(a->dq)) || (want_kv && (!rows_ok(a->dk) || !rows_ok(a->dv)))) return VDMI_E_ALIGN;
    if (!pitch_ok(a->dout) || !pitch_ok(a->dq) || !pitch_ok(a->dk) || !pitch_ok(a->dv)) return VDMI_E_SHAPE;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const Plan p = plan(a, wants_states(a));
    if (p.is_short) return launch_short(a, p, true, st);
    if (p.bytes && (!a->workspace || a->workspace_bytes < (int64_t)p.bytes || !a->fwd_workspace)) return VDMI_E_ARG;
    // S^T is read 16 bytes at a time
    if (!aligned16(a->state_in) || (p.bytes && (!aligned16(a->workspace) || !aligned16(a->fwd_workspace)))) return VDMI_E_ALIGN;
    if (want_q) {
        // dq: forward in time over (do, v, k) with S^T; the states at the segments' starts are the forward's
        ScanArgs s = scan_args(a, p);
        s.seg = const_cast<float*>(static_cast<const float*>(a->fwd_workspace));
        s.s_in = a->state_in;
        s.e_out = 1;
        s.rs = 1;
        role(s, a->dout, a->v, a->k, a->dq);
        const int r = launch_scan<OUTPUTS>(s, a, p, st);
        if (r != VDMI_OK || !want_kv) return r;
    }
    // dv and dk: backward in time; R = dS / m collects lambda^(i+1) q_i do_i^T
    if (p.nseg > 1) {
        ScanArgs s = scan_args(a, p);
        s.reverse = 1;
        s.e_u = 1;
        s.s_in = a->dstate_in;
        s.s_in_mul = 1.f / a->scale;
        s.s_out = a->dstate_out;
        s.s_out_mul = a->scale;
        role(s, a->k, a->q, a->dout, a->dv);
        const int r = segment_states(s, a, p, st);
        if (r != VDMI_OK) return r;
    }
    return launch_grad(a, p, st);
}

extern "C" int vdmi_decay_attn_step(const void* q, const void* k, const void* v, void* o, const int64_t* strides,
                                    const float* log_decay, float* state, int dtype, int64_t seqs, int heads, int d, float scale,
                                    vdmi_stream stream) {
    if (!q || !k || !v || !o || !strides || !log_decay || !state) return VDMI_E_ARG;
    if (dtype != VDMI_DT_BF16 && dtype != VDMI_DT_F16) return VDMI_E_ARG;
    if (!scale_ok(scale)) return VDMI_E_ARG;
    if (seqs <= 0 || heads <= 0 || (d != 32 && d != 64 && d != 128) || seqs > 0x7fffffffLL / heads) return VDMI_E_SHAPE;
    if (!aligned16(state)) return VDMI_E_ALIGN;
    StepArgs s = {q, k, v, o, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], strides[6], strides[7],
                  log_decay, state, heads, scale, seqs * heads * (d / 32)};
    const long long wgs = (s.tasks + 3) / 4;
    if (!launch_fits(wgs, 256)) return VDMI_E_SHAPE;
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
