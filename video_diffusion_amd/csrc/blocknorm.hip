// The norms before and after a block with its gate and residual scale, in one pass over the rows:
//     sum = alpha x + gate_b * P(h) * post_weight          (after a block; without h: sum = x)
//     y   = N(sum) * weight * (1 + scale_b) + shift_b      (before the next one)
// N and P are the root-mean-square norm t / sqrt(mean t^2 + eps) or the layer norm (t - mean) / sqrt(var + eps); P may be
// absent.  gate, scale and shift belong to a sample (its rows_per_sample consecutive rows) or to all rows.
// Backward, with a = weight (1 + scale_b), c = gate_b post_weight, n = N(sum), p = P(h), f the norms' factors:
//     ds = dout + f_n (dy a - mean(dy a) - n mean(dy a n)),   dx = alpha ds,
//     dh = f_p (ds c - mean(ds c) - p mean(ds c p))           (the plain means for the layer norm only)
// and per column, over the rows of a sample: S1 = sum dy n, S2 = sum dy, S3 = sum ds p, from which
//     dscale_b = weight S1, dshift_b = S2, dgate_b = post_weight S3, dweight = sum_b (1 + scale_b) S1, dpost_weight = sum_b gate_b S3.
// Everything between loads and stores is float32; the second norm sees the sum before it is rounded for storage, forward
// and backward (which computes it again from x and h: reading them costs what reading the stored sum would).
//
// What bounds it: memory (x, h, out, y once; backward x, h, dout, dy, dx, dh once).  262144 bfloat16 rows of 256 columns:
// forward 102 us (537 MB, 5.3 TB/s), backward 181 us (805 MB, 4.4 TB/s) and 10 us for the column sums; 3711 float32 rows of
// 2048: 29 us (4.2 TB/s) and 42 us (4.3 TB/s), sums 10 us.  L lanes hold a row in registers, P
// pieces of eight columns each; a workgroup stays in one sample, so the parameters are products in registers and the column
// sums are kept there too, added over the workgroup's rows and written once; a second launch adds the workgroups' sums in
// a fixed order.
#include "block_common.h"

#include <algorithm>

namespace {

struct NormArgs {
    const void* x; const void* h; const void* dout; const void* dy;
    void* out; void* y; void* dx; void* dh;
    long long ldx, ldh, ldo, ldy, lddo, lddy, lddx, lddh;
    const float* pw; const float* gate; const float* w; const float* scale; const float* shift;
    long long gate_bs, scale_bs, shift_bs;
    long long rows_per_sample, sample0; // sample0: the launch's first one
    float* part;                        // [sample][parts][3][c] or null
    int c, kind, pkind, parts, rows_per_wg;     // kinds: 0 rms, 1 layer, -1 none
    float eps, alpha;
};

template <int L>
struct RowSum {                         // sums over the L lanes of a row; L == 256: the workgroup, one row at a time
    float (*slots)[2][4];
    int turn = 0;
    __device__ __forceinline__ void two(float& a, float& b) {
        if constexpr (L <= 64) {
            a = vdmi_group_sum<L>(a);
            b = vdmi_group_sum<L>(b);
        } else {
            a = vdmi_group_sum<64>(a);
            b = vdmi_group_sum<64>(b);
            const int wave = threadIdx.x >> 6;
            // two sets of slots: a set is written again only after the barrier of the other one, which every wave passes
            // after it has read the first
            if ((threadIdx.x & 63) == 0) {
                slots[turn][0][wave] = a;
                slots[turn][1][wave] = b;
            }
            __syncthreads();
            a = (slots[turn][0][0] + slots[turn][0][1]) + (slots[turn][0][2] + slots[turn][0][3]);
            b = (slots[turn][1][0] + slots[turn][1][1]) + (slots[turn][1][2] + slots[turn][1][3]);
            turn ^= 1;
        }
    }
};

// A lane's pieces of eight consecutive columns, loaded and stored 16 bytes at a time at any alignment of the elements.
// TAIL: the columns are no multiple of eight; the row's last piece then begins eight columns before its end and holds some
// columns twice.  Both copies are computed and stored alike, sums take those from own[] on.  (160000 bfloat16 rows of 301
// columns, forward / backward: 113 / 189 us; the last piece element by element 157 / 362; the whole row so 189 / 440.)
// Rows of less than eight columns begin before their start: they go element by element from own[] on.
template <bool TAIL, int L, int P>
struct Columns {
    int c, start[P], own[P];
    __device__ __forceinline__ Columns(int c, int l) : c(c) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int at = (p * L + l) * 8;
            start[p] = TAIL ? min(at, c - 8) : at;
            own[p] = at < c ? at - start[p] : 8;
        }
    }
    __device__ __forceinline__ bool there(int p) const { return TAIL ? own[p] < 8 : start[p] < c; }
    // of element i = 8 p + e
    __device__ __forceinline__ bool mine(int i) const { return TAIL ? (i & 7) >= own[i >> 3] : there(i >> 3); }
    // what element i adds to a sum (elements that are not there are zeros)
    __device__ __forceinline__ float part(float v, int i) const { return !TAIL || mine(i) ? v : 0.f; }
};

template <typename T, bool TAIL, int L, int P>
__device__ __forceinline__ void load_row(float (&v)[P * 8], const T* r, float absent, const Columns<TAIL, L, P>& at) {
    constexpr int W = 16 / sizeof(T);
    typedef T wide __attribute__((ext_vector_type(W), aligned(sizeof(T))));
    T x[P * 8];
#pragma unroll
    for (int i = 0; i < P * 8; ++i) x[i] = (T)absent;
    if (!TAIL || at.c >= 8) {
#pragma unroll
        for (int p = 0; p < P; ++p)
            if (at.there(p)) {
#pragma unroll
                for (int i = 0; i < 8 / W; ++i) {
                    const wide a = *reinterpret_cast<const wide*>(r + at.start[p] + W * i);
#pragma unroll
                    for (int e = 0; e < W; ++e) x[8 * p + W * i + e] = a[e];
                }
            }
    } else {
#pragma unroll
        for (int e = 1; e < 8; ++e)
            if (at.mine(e)) x[e] = r[at.start[0] + e];
    }
#pragma unroll
    for (int i = 0; i < P * 8; ++i) v[i] = (float)x[i];
}

template <typename T, bool TAIL, int L, int P>
__device__ __forceinline__ void store_row(const float (&v)[P * 8], T* r, const Columns<TAIL, L, P>& at) {
    constexpr int W = 16 / sizeof(T);
    typedef T wide __attribute__((ext_vector_type(W), aligned(sizeof(T))));
    if (!TAIL || at.c >= 8) {
#pragma unroll
        for (int p = 0; p < P; ++p)
            if (at.there(p)) {
#pragma unroll
                for (int i = 0; i < 8 / W; ++i) {
                    wide a;
#pragma unroll
                    for (int e = 0; e < W; ++e) a[e] = (T)v[8 * p + W * i + e];
                    *reinterpret_cast<wide*>(r + at.start[p] + W * i) = a;
                }
            }
    } else {
#pragma unroll
        for (int e = 1; e < 8; ++e)
            if (at.mine(e)) r[at.start[0] + e] = (T)v[e];
    }
}

// the lane's columns of a parameter row, `absent` where there is none
template <bool TAIL, int L, int P>
__device__ __forceinline__ void load_params(float (&v)[P * 8], const float* src, float absent, const Columns<TAIL, L, P>& at) {
    if (src) {
        load_row<float, TAIL, L, P>(v, src, absent, at);
    } else {
#pragma unroll
        for (int i = 0; i < P * 8; ++i) v[i] = absent;
    }
}

// v -> its norm in place; returns the factor
template <bool TAIL, int L, int P>
__device__ __forceinline__ float normalise(float (&v)[P * 8], RowSum<L>& sum, int kind, float inv_c, float eps,
                                           const Columns<TAIL, L, P>& at) {
    if (kind == 1) {
        float s = 0.f, z = 0.f;
#pragma unroll
        for (int i = 0; i < P * 8; ++i) s += at.part(v[i], i);
        sum.two(s, z);
        const float mean = s * inv_c;
#pragma unroll
        for (int i = 0; i < P * 8; ++i) v[i] = at.there(i >> 3) ? v[i] - mean : 0.f;
    }
    float s = 0.f, z = 0.f;
#pragma unroll
    for (int i = 0; i < P * 8; ++i) s += at.part(v[i] * v[i], i);
    sum.two(s, z);
    const float f = 1.f / __builtin_sqrtf(s * inv_c + eps);
#pragma unroll
    for (int i = 0; i < P * 8; ++i) v[i] *= f;
    return f;
}

// g (gradient of a norm's result n) -> f (g - mean g - n mean(g n)); the plain mean for the layer norm
template <bool TAIL, int L, int P>
__device__ __forceinline__ void norm_gradient(float (&g)[P * 8], const float (&n)[P * 8], float f, RowSum<L>& sum, int kind,
                                              float inv_c, const Columns<TAIL, L, P>& at) {
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int i = 0; i < P * 8; ++i) { s += at.part(g[i], i); t += at.part(g[i] * n[i], i); }
    sum.two(s, t);
    s = kind == 1 ? s * inv_c : 0.f;
    t *= inv_c;
#pragma unroll
    for (int i = 0; i < P * 8; ++i) g[i] = at.there(i >> 3) ? f * (g[i] - s - n[i] * t) : 0.f;
}

template <typename T, bool TAIL, int L, int P, bool BWD>
__global__ __launch_bounds__(256, P == 1 ? 4 : 1) void block_norm_kernel(const NormArgs a) {
    constexpr int N = P * 8, ROWS = 256 / L;
    __shared__ float slots[2][2][4];
    __shared__ float cols[BWD && ROWS > 1 ? ROWS * L * N : 1];
    RowSum<L> sum{slots};
    const int l = threadIdx.x % L, group = threadIdx.x / L, c = a.c;
    const unsigned there = blockIdx.x / a.parts;
    const long long sample = a.sample0 + there;
    const int part = (int)(blockIdx.x - there * a.parts);
    const long long first = (long long)part * a.rows_per_wg;
    const long long last = min(first + a.rows_per_wg, a.rows_per_sample);
    const float inv_c = 1.f / (float)c;
    const Columns<TAIL, L, P> at(c, l);
    // per column: a = weight (1 + scale), gate * post_weight, shift
    float wa[N], pg[N], sh[BWD ? 1 : N];
    load_params<TAIL, L, P>(wa, a.w, 1.f, at);
    load_params<TAIL, L, P>(pg, a.pw, 1.f, at);
    if (a.scale) {
        float t[N];
        load_params<TAIL, L, P>(t, a.scale + sample * a.scale_bs, 0.f, at);
#pragma unroll
        for (int i = 0; i < N; ++i) wa[i] *= 1.f + t[i];
    }
    if (a.gate) {
        float t[N];
        load_params<TAIL, L, P>(t, a.gate + sample * a.gate_bs, 0.f, at);
#pragma unroll
        for (int i = 0; i < N; ++i) pg[i] *= t[i];
    }
    if constexpr (!BWD) load_params<TAIL, L, P>(sh, a.shift ? a.shift + sample * a.shift_bs : nullptr, 0.f, at);
    float s1[BWD ? N : 1], s2[BWD ? N : 1], s3[BWD ? N : 1];
    if constexpr (BWD) {
#pragma unroll
        for (int i = 0; i < N; ++i) s1[i] = s2[i] = s3[i] = 0.f;
    }
    // every group of a workgroup walks the same number of rows (the sums of L == 256 meet at barriers; ROWS is 1 there)
    for (long long r0 = first; r0 < last; r0 += ROWS) {
        const long long r = r0 + group;
        if (r >= last) continue;        // L <= 64: lanes of other rows are not involved in this one's sums
        const long long row = sample * a.rows_per_sample + r;
        float v[N], h[N];
        load_row<T, TAIL, L, P>(v, static_cast<const T*>(a.x) + row * a.ldx, 0.f, at);
        if (a.h) load_row<T, TAIL, L, P>(h, static_cast<const T*>(a.h) + row * a.ldh, 0.f, at);
        float fh = 1.f;
        if constexpr (!BWD) {
            if (a.h) {
                if (a.pkind >= 0) normalise<TAIL, L, P>(h, sum, a.pkind, inv_c, a.eps, at);
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = a.alpha * v[i] + pg[i] * h[i];
                store_row<T, TAIL, L, P>(v, static_cast<T*>(a.out) + row * a.ldo, at);
            }
            if (a.y) {
                normalise<TAIL, L, P>(v, sum, a.kind, inv_c, a.eps, at);
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = v[i] * wa[i] + sh[i];
                store_row<T, TAIL, L, P>(v, static_cast<T*>(a.y) + row * a.ldy, at);
            }
        } else {
            float ds[N], g[N];
            if (a.dout) load_row<T, TAIL, L, P>(ds, static_cast<const T*>(a.dout) + row * a.lddo, 0.f, at);
            if (a.dy) load_row<T, TAIL, L, P>(g, static_cast<const T*>(a.dy) + row * a.lddy, 0.f, at);
            if (a.h) {
                if (a.pkind >= 0) fh = normalise<TAIL, L, P>(h, sum, a.pkind, inv_c, a.eps, at);
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = a.alpha * v[i] + pg[i] * h[i];
            }
            if (a.dy) {
                const float f = normalise<TAIL, L, P>(v, sum, a.kind, inv_c, a.eps, at);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    s1[i] += g[i] * v[i];
                    s2[i] += g[i];
                    g[i] *= wa[i];
                }
                norm_gradient<TAIL, L, P>(g, v, f, sum, a.kind, inv_c, at);
#pragma unroll
                for (int i = 0; i < N; ++i) ds[i] = a.dout ? ds[i] + g[i] : g[i];
            }
            if (a.dx) {
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = (a.h ? a.alpha : 1.f) * ds[i];
                store_row<T, TAIL, L, P>(v, static_cast<T*>(a.dx) + row * a.lddx, at);
            }
            if (a.h) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    s3[i] += ds[i] * h[i];
                    ds[i] *= pg[i];
                }
                if (a.dh) {
                    if (a.pkind >= 0) norm_gradient<TAIL, L, P>(ds, h, fh, sum, a.pkind, inv_c, at);
                    store_row<T, TAIL, L, P>(ds, static_cast<T*>(a.dh) + row * a.lddh, at);
                }
            }
        }
    }
    if constexpr (BWD) {
        if (a.part) {
            float* dst = a.part + (sample * a.parts + part) * 3 * (long long)c;
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                const float* s = k == 0 ? s1 : k == 1 ? s2 : s3;
                if constexpr (ROWS == 1) {
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (at.mine(i)) dst[(long long)k * c + at.start[i >> 3] + (i & 7)] = s[i];
                } else {
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (!TAIL || at.mine(i)) cols[(group * N + i - (TAIL ? at.own[i >> 3] : 0)) * L + l] = s[i];
                    __syncthreads();
                    for (int q = threadIdx.x; q < L * N; q += 256) {
                        const int i = q / L, col = ((i >> 3) * L + q % L) * 8 + (i & 7);     // by the pieces' places
                        float t = 0.f;
                        for (int gr = 0; gr < ROWS; ++gr) t += cols[(gr * N + i) * L + q % L];
                        if (col < c) dst[(long long)k * c + col] = t;
                    }
                }
            }
        }
    }
}

// The column sums of the workgroups of a sample -> [sample][3][c] and the sample's own gradients; then, over the samples,
// the gradients of the weights and of gates, scales and shifts that all samples share.  16 columns x 64 partial sums per
// workgroup, combined in a fixed order.
struct SumArgs {
    const float* part;                  // [samples][parts][3][c]
    float* by_sample;                   // [samples][3][c] or null (one sample: its sums are used at once)
    const float* pw; const float* gate; const float* w; const float* scale;
    long long gate_bs, scale_bs, shift_bs;
    float* dpw; float* dgate; float* dw; float* dscale; float* dshift;
    int c, parts;
    long long samples, sample0;         // sample0: the launch's first one
};

__device__ __forceinline__ void add64(float (&v)[3], float (*buf)[3][16], int pl, int col) {
#pragma unroll
    for (int k = 0; k < 3; ++k) buf[pl][k][col] = v[k];
    __syncthreads();
    for (int n = 32; n > 0; n >>= 1) {
        if (pl < n) {
#pragma unroll
            for (int k = 0; k < 3; ++k) buf[pl][k][col] += buf[pl + n][k][col];
        }
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) v[k] = buf[0][k][col];
}

__global__ __launch_bounds__(1024) void norm_sums_kernel(const SumArgs a) {
    __shared__ float buf[64][3][16];
    const int lc = threadIdx.x & 15, pl = threadIdx.x >> 4, col = blockIdx.y * 16 + lc;
    const long long sample = a.sample0 + blockIdx.x;
    float v[3] = {0.f, 0.f, 0.f};
    if (col < a.c) {
        const float* p = a.part + sample * a.parts * 3 * (long long)a.c + col;
        for (int i = pl; i < a.parts; i += 64)
#pragma unroll
            for (int k = 0; k < 3; ++k) v[k] += p[((long long)i * 3 + k) * a.c];
    }
    add64(v, buf, pl, lc);
    if (pl != 0 || col >= a.c) return;
    const float w = a.w ? a.w[col] : 1.f, pw = a.pw ? a.pw[col] : 1.f;
    if (a.dscale && (a.scale_bs || a.samples == 1)) a.dscale[sample * a.scale_bs + col] = w * v[0];
    if (a.dshift && (a.shift_bs || a.samples == 1)) a.dshift[sample * a.shift_bs + col] = v[1];
    if (a.dgate && (a.gate_bs || a.samples == 1)) a.dgate[sample * a.gate_bs + col] = pw * v[2];
    if (a.samples == 1) {
        if (a.dw) a.dw[col] = (a.scale ? 1.f + a.scale[col] : 1.f) * v[0];
        if (a.dpw) a.dpw[col] = (a.gate ? a.gate[col] : 1.f) * v[2];
    } else {
#pragma unroll
        for (int k = 0; k < 3; ++k) a.by_sample[(sample * 3 + k) * a.c + col] = v[k];
    }
}

__global__ __launch_bounds__(1024) void norm_sample_sums_kernel(const SumArgs a) {
    __shared__ float buf[64][3][16];
    const int lc = threadIdx.x & 15, pl = threadIdx.x >> 4, col = blockIdx.x * 16 + lc;
    float v[3] = {0.f, 0.f, 0.f}, u[3] = {0.f, 0.f, 0.f};       // v: for weights and shared shift, u: shared scale and gate
    if (col < a.c) {
        for (long long b = pl; b < a.samples; b += 64) {
            const float* p = a.by_sample + b * 3 * (long long)a.c + col;
            const float t1 = p[0], t2 = p[a.c], t3 = p[2 * (long long)a.c];
            v[0] += (a.scale ? 1.f + a.scale[b * a.scale_bs + col] : 1.f) * t1;
            v[1] += t2;
            v[2] += (a.gate ? a.gate[b * a.gate_bs + col] : 1.f) * t3;
            u[0] += t1;
            u[2] += t3;
        }
    }
    add64(v, buf, pl, lc);
    __syncthreads();
    add64(u, buf, pl, lc);
    if (pl != 0 || col >= a.c) return;
    if (a.dw) a.dw[col] = v[0];
    if (a.dpw) a.dpw[col] = v[2];
    if (a.dshift && !a.shift_bs) a.dshift[col] = v[1];
    if (a.dscale && !a.scale_bs) a.dscale[col] = (a.w ? a.w[col] : 1.f) * u[0];
    if (a.dgate && !a.gate_bs) a.dgate[col] = (a.pw ? a.pw[col] : 1.f) * u[2];
}

// Lanes and pieces of a row: a wave or less holds up to 1024 columns, 16 per lane; wider rows spread over the workgroup
// (3711 float32 rows of 2048 columns forward: 29 us, 4.2 TB/s; with a wave per row and 32 columns per lane 95 us).  Kernels
// of one piece per lane stay within 128 registers, four waves on a SIMD (301 columns backward: 189 us, with three 289).
struct Shape { bool tail; int lanes, pieces; };

Shape shape_of(const vdmi_block_norm_args* a) {
    const int g = (a->c + 7) / 8;
    Shape s;
    s.tail = a->c % 8 != 0;
    s.lanes = g <= 8 ? 8 : g <= 16 ? 16 : g <= 32 ? 32 : g <= 128 ? 64 : 256;
    s.pieces = (g + s.lanes - 1) / s.lanes;
    if (s.pieces == 3) s.pieces = 4;
    return s;
}

struct NormPlan { long long samples, rps; int parts, rows_per_wg; bool sums; size_t part_bytes, bytes; };

NormPlan norm_plan(const vdmi_block_norm_args* a, bool bwd) {
    NormPlan p;
    const bool per_sample = (a->gate && a->gate_stride) || (a->scale && a->scale_stride) || (a->shift && a->shift_stride);
    p.samples = per_sample ? a->rows / a->rows_per_sample : 1;
    p.rps = per_sample ? a->rows_per_sample : a->rows;
    const Shape s = shape_of(a);
    const long long at_once = 256 / s.lanes;
    // about four workgroups per CU backward (each writes its column sums), eight forward
    long long per = (p.samples * p.rps + (bwd ? 1024 : 2048) - 1) / (bwd ? 1024 : 2048);
    if (bwd && s.lanes == 256 && per < 8) per = 8;      // a workgroup writes 12 c bytes of sums: not for fewer rows
    per = (per + at_once - 1) / at_once * at_once;
    const long long most = (p.rps + at_once - 1) / at_once * at_once;
    if (per > most) per = most;
    p.rows_per_wg = (int)per;
    p.parts = (int)((p.rps + per - 1) / per);
    p.sums = bwd && (a->dpost_weight || a->dgate || a->dweight || a->dscale || a->dshift);
    p.part_bytes = p.sums ? (size_t)p.samples * p.parts * 3 * a->c * sizeof(float) : 0;
    p.bytes = p.part_bytes + (p.sums && p.samples > 1 ? (size_t)p.samples * 3 * a->c * sizeof(float) : 0);
    return p;
}

int check_norm(const vdmi_block_norm_args* a, bool bwd) {
    if (!a || !a->x) return VDMI_E_ARG;
    if (a->dtype != VDMI_DT_BF16 && a->dtype != VDMI_DT_F16 && a->dtype != VDMI_DT_F32) return VDMI_E_ARG;
    if (a->kind < 0 || a->kind > 1 || a->post_kind < -1 || a->post_kind > 1) return VDMI_E_ARG;
    if (!(a->eps >= 0.f) || !(a->eps < 1e30f) || !(a->alpha - a->alpha == 0.f)) return VDMI_E_ARG;
    if (a->c <= 0 || a->c > 8192 || a->rows <= 0 || a->rows > 0x7fffffffLL) return VDMI_E_SHAPE;
    if (a->rows_per_sample <= 0 || a->rows % a->rows_per_sample) return VDMI_E_SHAPE;
    for (int64_t s : {a->gate_stride, a->scale_stride, a->shift_stride})
        if (s != 0 && s != a->c) return VDMI_E_SHAPE;
    if (a->ldx < a->c || (a->h && a->ldh < a->c)) return VDMI_E_SHAPE;
    if (!a->h && (a->post_weight || a->gate)) return VDMI_E_ARG;
    if (!bwd) {
        if (!a->h != !a->out) return VDMI_E_ARG;               // the sum is written where there is one
        if (!a->out && !a->y) return VDMI_E_ARG;
        if ((a->out && a->ldo < a->c) || (a->y && a->ldy < a->c)) return VDMI_E_SHAPE;
    } else {
        if (!a->dout && !a->dy) return VDMI_E_ARG;
        if (a->dh && !a->h) return VDMI_E_ARG;
        if ((a->dpost_weight && !a->post_weight) || (a->dgate && !a->gate) || (a->dweight && !a->weight) ||
            (a->dscale && !a->scale) || (a->dshift && !a->shift)) return VDMI_E_ARG;
        if ((a->dout && a->lddo < a->c) || (a->dy && a->lddy < a->c) || (a->dx && a->lddx < a->c) || (a->dh && a->lddh < a->c))
            return VDMI_E_SHAPE;
    }
    // elements of the type: nothing narrower is read
    const uintptr_t mask = a->dtype == VDMI_DT_F32 ? 3u : 1u;
    for (const void* p : {a->x, a->h, (const void*)a->out, (const void*)a->y, a->dout, a->dy, (const void*)a->dx, (const void*)a->dh})
        if (reinterpret_cast<uintptr_t>(p) & mask) return VDMI_E_ALIGN;
    return VDMI_OK;
}

template <typename T, bool BWD>
int launch_norm(const NormArgs& n, const Shape& s, unsigned grid, hipStream_t st) {
#define NORM(L, P) do { if (s.tail) hipLaunchKernelGGL((block_norm_kernel<T, true, L, P, BWD>), dim3(grid), dim3(256), 0, st, n); \
                        else hipLaunchKernelGGL((block_norm_kernel<T, false, L, P, BWD>), dim3(grid), dim3(256), 0, st, n); } while (0)
    switch (s.lanes * 8 + s.pieces) {
        case 8 * 8 + 1: NORM(8, 1); break;
        case 16 * 8 + 1: NORM(16, 1); break;
        case 32 * 8 + 1: NORM(32, 1); break;
        case 64 * 8 + 1: NORM(64, 1); break;
        case 64 * 8 + 2: NORM(64, 2); break;
        case 256 * 8 + 1: NORM(256, 1); break;
        case 256 * 8 + 2: NORM(256, 2); break;
        case 256 * 8 + 4: NORM(256, 4); break;
        default: return VDMI_E_SHAPE;
    }
#undef NORM
    VDMI_LAUNCH_CHECK();
    return VDMI_OK;
}

NormArgs norm_args(const vdmi_block_norm_args* a, const NormPlan& p) {
    NormArgs n = {};
    n.x = a->x; n.h = a->h; n.ldx = a->ldx; n.ldh = a->ldh;
    n.pw = a->post_weight; n.gate = a->gate; n.w = a->weight; n.scale = a->scale; n.shift = a->shift;
    n.gate_bs = a->gate_stride; n.scale_bs = a->scale_stride; n.shift_bs = a->shift_stride;
    n.rows_per_sample = p.rps;
    n.c = a->c; n.kind = a->kind; n.pkind = a->post_kind; n.parts = p.parts; n.rows_per_wg = p.rows_per_wg;
    n.eps = a->eps; n.alpha = a->alpha;
    return n;
}

// workgroups of one launch: 2^23 of 256 threads and 2^21 of 1024 stay below its 2^32 threads
constexpr long long AT_ONCE = 1LL << 23;

template <bool BWD>
int run_norm(const vdmi_block_norm_args* a, NormArgs n, const NormPlan& p, hipStream_t st) {
    const Shape s = shape_of(a);
    const long long samples = std::max(AT_ONCE / p.parts, 1LL);         // parts: 2048 at most
    for (n.sample0 = 0; n.sample0 < p.samples; n.sample0 += samples) {
        const unsigned grid = (unsigned)(std::min(samples, p.samples - n.sample0) * p.parts);
        const int r = a->dtype == VDMI_DT_BF16  ? launch_norm<__bf16, BWD>(n, s, grid, st)
                      : a->dtype == VDMI_DT_F16 ? launch_norm<_Float16, BWD>(n, s, grid, st)
                                                : launch_norm<float, BWD>(n, s, grid, st);
        if (r != VDMI_OK) return r;
    }
    return VDMI_OK;
}

}   // namespace

extern "C" int vdmi_block_norm_fwd(const vdmi_block_norm_args* a, vdmi_stream stream) {
    const int ok = check_norm(a, false);
    if (ok != VDMI_OK) return ok;
    vdmi_block_norm_args f = *a;            // what the backward alone uses plays no part in the choice of a kernel
    f.dout = f.dy = nullptr;
    f.dx = f.dh = nullptr;
    const NormPlan p = norm_plan(&f, false);
    NormArgs n = norm_args(&f, p);
    n.out = f.out; n.y = f.y; n.ldo = f.ldo; n.ldy = f.ldy;
    return run_norm<false>(&f, n, p, static_cast<hipStream_t>(stream));
}

extern "C" size_t vdmi_block_norm_bwd_workspace_bytes(const vdmi_block_norm_args* a) {
    if (check_norm(a, true) != VDMI_OK) return 0;
    vdmi_block_norm_args f = *a;
    f.out = f.y = nullptr;
    return norm_plan(&f, true).bytes;
}

extern "C" int vdmi_block_norm_bwd(const vdmi_block_norm_args* a, vdmi_stream stream) {
    const int ok = check_norm(a, true);
    if (ok != VDMI_OK) return ok;
    vdmi_block_norm_args f = *a;
    f.out = f.y = nullptr;
    const NormPlan p = norm_plan(&f, true);
    if (p.bytes && (!f.workspace || f.workspace_bytes < (int64_t)p.bytes)) return VDMI_E_ARG;
    if (p.bytes && !aligned16(f.workspace)) return VDMI_E_ALIGN;
    hipStream_t st = static_cast<hipStream_t>(stream);
    NormArgs n = norm_args(&f, p);
    n.dout = f.dout; n.dy = f.dy; n.dx = f.dx; n.dh = f.dh;
    n.lddo = f.lddo; n.lddy = f.lddy; n.lddx = f.lddx; n.lddh = f.lddh;
    n.part = p.sums ? static_cast<float*>(f.workspace) : nullptr;
    const int r = run_norm<true>(&f, n, p, st);
    if (r != VDMI_OK || !p.sums) return r;
    SumArgs s = {};
    s.part = n.part;
    s.by_sample = n.part + p.part_bytes / sizeof(float);
    s.pw = f.post_weight; s.gate = f.gate; s.w = f.weight; s.scale = f.scale;
    s.gate_bs = f.gate_stride; s.scale_bs = f.scale_stride; s.shift_bs = f.shift_stride;
    s.dpw = f.dpost_weight; s.dgate = f.dgate; s.dw = f.dweight; s.dscale = f.dscale; s.dshift = f.dshift;
    s.c = f.c; s.parts = p.parts; s.samples = p.samples;
    const unsigned gx = (unsigned)((f.c + 15) / 16);
    for (s.sample0 = 0; s.sample0 < p.samples; s.sample0 += AT_ONCE / 4) {
        hipLaunchKernelGGL(norm_sums_kernel, dim3((unsigned)std::min(AT_ONCE / 4, p.samples - s.sample0), gx), dim3(1024), 0, st, s);
        VDMI_LAUNCH_CHECK();
    }
    const bool across = p.samples > 1 && (f.dweight || f.dpost_weight || (f.dscale && !f.scale_stride) ||
                                          (f.dshift && !f.shift_stride) || (f.dgate && !f.gate_stride));
    if (!across) return VDMI_OK;
    hipLaunchKernelGGL(norm_sample_sums_kernel, dim3(gx), dim3(1024), 0, st, s);
    VDMI_LAUNCH_CHECK();
    return VDMI_OK;
}
