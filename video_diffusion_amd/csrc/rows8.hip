// Activation checkpoints in 8 bits: rows of activations kept for the backward pass as e4m3 codes (4 exponent and 3 fraction
// bits, largest 448) with a power of two per 32 consecutive channels, and their use there.
//   pack    e = the least exponent with max |x| <= 448 2^e over the group's finite values, in -118 .. 119 (so that every
//           code times 2^e is a bfloat16);  code = e4m3(x 2^-e), round to nearest even: off by 2^-4 of the value at most
//           (2^-10 2^e below 2^-6 2^e).  Infinities and NaN become NaN; magnitudes beyond 448 2^119 (2.9e38) become that.
//   unpack  code 2^e, to halfs at most 65504
//   weight gradient of a Linear from the kept input: dw[o][i] = sum_r dy[r][o] code[r][i] 2^e, on the matrix cores, codes
//           widened to bfloat16 (exactly) on their way into LDS - half the bytes of bfloat16 rows.
#include "block_common.h"

namespace {

// ---- pack: a lane holds 8 channels, four lanes a group ------------------------------------------------------------
// What bounds it: memory.  262144 bfloat16 rows of 256 channels (203 MB): 42 us, 4.8 TB/s; back 31 us, 6.6 TB/s.
struct PackArgs {
    const void* x;
    unsigned char* codes;       // [rows][c]
    unsigned char* exps;        // [rows][groups]: e + 127
    long long ldx, total;       // total = rows * groups * 4 lanes
    int c, groups;
};

template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T* p) {
    if constexpr (sizeof(T) == 4) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[4 + e] = b[e]; }
    } else {
        typedef __attribute__((ext_vector_type(8))) T t8;
        const t8 a = *reinterpret_cast<const t8*>(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)a[e];
    }
}

template <typename T>
__global__ __launch_bounds__(256) void rows8_pack_kernel(const PackArgs a) {
    const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long group = idx >> 2;
    const long long row = group / a.groups;
    const int g = (int)(group - row * a.groups), col = 32 * g + 8 * (int)(idx & 3);
    const bool on = idx < a.total && col < a.c;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if (on) load8<T>(v, static_cast<const T*>(a.x) + row * a.ldx + col);
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float m = fabsf(v[e]);
        top = m < __builtin_inff() ? fmaxf(top, m) : top;
    }
    top = fmaxf(top, vdmi_dpp<0xB1>(top));
    top = fmaxf(top, vdmi_dpp<0x4E>(top));
    const unsigned bits = __float_as_uint(top);
    int e2 = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    e2 = min(max(e2, -118), 119);
    const float inv = __uint_as_float((unsigned)(127 - e2) << 23);
#pragma unroll
    for (int e = 0; e < 8; ++e)
        v[e] = fabsf(v[e]) < __builtin_inff() ? fminf(fmaxf(v[e] * inv, -448.f), 448.f) : __builtin_nanf("");
    uint2 w;
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
    w.x = (unsigned)lo;
    w.y = (unsigned)hi;
    if (on) {
        *reinterpret_cast<uint2*>(a.codes + row * a.c + col) = w;
        if ((idx & 3) == 0) a.exps[group] = (unsigned char)(e2 + 127);
    }
}

__device__ __forceinline__ void widen8(float (&v)[8], uint2 w, unsigned exp) {
    const float s = __uint_as_float(exp << 23);
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, true);
    const auto c = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, true);
    v[0] = a[0] * s; v[1] = a[1] * s; v[2] = b[0] * s; v[3] = b[1] * s;
    v[4] = c[0] * s; v[5] = c[1] * s; v[6] = d[0] * s; v[7] = d[1] * s;
}

// the same to bfloat16, two codes an instruction: exact, since every code times its power of two is a bfloat16
__device__ __forceinline__ Pack<__bf16>::x8 widen8_bf16(vdmi_u2 w, unsigned exp) {
    const float s = __uint_as_float(exp << 23);
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, s, true);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, s, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, s, true);
    return Pack<__bf16>::x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

struct UnpackArgs {
    const unsigned char* codes;
    const unsigned char* exps;
    void* x;
    long long ldx, total;       // total = rows * c / 8
    int c, groups;
};

template <typename T>
__global__ __launch_bounds__(256) void rows8_unpack_kernel(const UnpackArgs a) {
    const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
    if (idx >= a.total) return;
    const int per = a.c >> 3;
    const long long row = idx / per;
    const int p = (int)(idx - row * per);
    const uint2 w = *reinterpret_cast<const uint2*>(a.codes + idx * 8);
    float v[8];
    widen8(v, w, a.exps[row * a.groups + (p >> 2)]);
    if constexpr (__is_same(T, _Float16)) {
        // halfs from 63488 on have the code of 65536, which is not a half: what is finite stays finite
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fabsf(v[e]) > 65504.f ? copysignf(65504.f, v[e]) : v[e];
    }
    T* dst = static_cast<T*>(a.x) + row * a.ldx + 8 * p;
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<f32x4*>(dst) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(dst + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
        typedef __attribute__((ext_vector_type(8))) T t8;
        t8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (T)v[e];
        *reinterpret_cast<t8*>(dst) = o;
    }
}

// ---- weight gradient -----------------------------------------------------------------------------------------------
// The contraction index (the row) is the slow one in memory for both operands: stages of 64 rows go into LDS as they lie
// and the fragments are read with ds_read_b64_tr_b16.  A workgroup owns 128 x 128 of dw for a share of the rows, four waves
// 64 x 64 each; LDS rows are 320 bytes apart (the four rows x two column blocks of a half wave's read fall into different
// banks).  Shares are added in a fixed order by a second launch.  The bias gradient sum_r dy comes from the staged pieces.
// What bounds it: LDS - a wave reads 4 KB of fragments for four products of 32 cycles, what LDS gives four waves in that
// time, and the staging comes on top.  131072 rows, 512 -> 1536 channels: 243 us (850 TFLOP/s) in the first launches of a run
// and after some 150 of them, 330 to 354 in between (launches 8 to 15; 297 on average over 20) - the same launches on the same
// data, so the card's answer to the load, not the kernel's - and 17 us for the shares' sums; bfloat16 rows through
// vdmi_rows_wgrad 414, the library's product 709.  A 256 x 128 tile (128 x 64 per wave, three quarters of the LDS reads, one
// workgroup per CU) took 341, one stage ahead in registers in place of two 392.
constexpr int WK = 64, WT = 128, WPITCH = 320;

struct Wgrad8Args {
    const unsigned char* codes; const unsigned char* exps;
    const __bf16* dy;
    float* part;                // [split][o tiles][i tiles][128][128]
    float* bpart;               // [split][o tiles][128] or null
    long long lddy, rows, per;  // per: rows of a share
    int cin, cout, groups, to, ti, splits;
};

typedef Pack<__bf16>::x8 b8;

__global__ __launch_bounds__(256, 2) void rows8_wgrad_kernel(const Wgrad8Args a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];          // [buffer][dy | x][64][320]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, l31 = lane & 31;
    // workgroups go round the eight XCDs, each with its own L2: all tiles of a share of the rows on one of them
    const unsigned tiles = a.to * a.ti, k = a.splits % 8 == 0 ? blockIdx.x >> 3 : blockIdx.x, share = k / tiles;
    const int tile = (int)(k - share * tiles), it = tile / a.to, ot = tile - it * a.to;
    const long long split = a.splits % 8 == 0 ? (blockIdx.x & 7) + 8 * share : share;
    const int o0 = ot * WT, i0 = it * WT;
    const long long r_begin = split * a.per, r_end = min(r_begin + a.per, a.rows);
    // staging: piece tid + 256 j is (row (tid >> 4) + 16 j, columns 8 (tid & 15) ..): a thread's column is fixed
    const int prow = tid >> 4, pc = tid & 15;
    // byte offsets within a stage; columns past the operands' ends load zeros, and so do rows past the share's end
    const unsigned aoff = o0 + 8 * pc < a.cout ? (unsigned)(prow * a.lddy + o0 + 8 * pc) * 2 : NOWHERE;
    const unsigned boff = i0 + 8 * pc < a.cin ? (unsigned)(prow * a.cin + i0 + 8 * pc) : NOWHERE;
    const unsigned eoff = i0 + 8 * pc < a.cin ? (unsigned)(prow * a.groups + ((i0 + 8 * pc) >> 5)) : NOWHERE;
    struct Staged { b8 a[4]; vdmi_u2 b[4]; unsigned e[4]; } ra, rb;
    float bias[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) bias[e] = 0.f;
    auto load = [&](Staged& v, long long r0) {
        const unsigned n = (unsigned)max(min(r_end - r0, (long long)WK), 0ll);
        const auto da = vdmi_rsrc(a.dy + r0 * a.lddy, n * (unsigned)a.lddy * 2), db = vdmi_rsrc(a.codes + r0 * a.cin, n * a.cin),
                   de = vdmi_rsrc(a.exps + r0 * a.groups, n * a.groups);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v.a[j] = load16<__bf16>(da, aoff + 32 * j * (unsigned)a.lddy);
            v.b[j] = __builtin_amdgcn_raw_buffer_load_b64(db, boff + 16 * j * a.cin, 0, 0);
            v.e[j] = __builtin_amdgcn_raw_buffer_load_b8(de, eoff + 16 * j * a.groups, 0, 0);
        }
    };
    const bool sums = a.bpart && it == 0;
    auto store = [&](const Staged& v, int buf, int j) {
        char* la = lds + buf * (2 * WK * WPITCH) + (prow + 16 * j) * WPITCH + 16 * pc;
        *reinterpret_cast<b8*>(la) = v.a[j];
        *reinterpret_cast<b8*>(la + WK * WPITCH) = widen8_bf16(v.b[j], v.e[j]);
    };
    auto add_bias = [&](const Staged& v) {
        if (sums) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) bias[e] += (float)v.a[j][e];
        }
    };
    const int g16 = lane >> 4, tq = (lane >> 2) & 3, tp = lane & 3;
    const int tr_off = (8 * (g16 >> 1) + tq) * WPITCH + (16 * (g16 & 1) + 4 * tp) * 2;
    const int wo = 64 * (wave & 1), wi = 64 * (wave >> 1);
    f32x16 acc[2][2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n) acc[m][n] = zero16();
    // products of the stage in `buf`; the next one's pieces go into the other buffer between them.  The order is held: loads
    // first (they need the whole stage), then every step's fragments ahead of the products before it.
    auto stage = [&](int buf, const Staged& next) {
        const char* ta = lds + buf * (2 * WK * WPITCH) + tr_off + 2 * wo;
        const char* tb = lds + buf * (2 * WK * WPITCH) + WK * WPITCH + tr_off + 2 * wi;
        b8 A[2][2], B[2][2];
        auto fragments = [&](int ks) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                A[ks & 1][m] = tr_operand<__bf16>(ta + ks * 16 * WPITCH + 64 * m, 4 * WPITCH);
                B[ks & 1][m] = tr_operand<__bf16>(tb + ks * 16 * WPITCH + 64 * m, 4 * WPITCH);
            }
        };
        __builtin_amdgcn_sched_barrier(0);
        fragments(0);
#pragma unroll
        for (int ks = 0; ks < WK / 16; ++ks) {
            if (ks + 1 < WK / 16) fragments(ks + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int n = 0; n < 2; ++n) acc[m][n] = mfma16(A[ks & 1][m], B[ks & 1][n], acc[m][n]);
            store(next, buf ^ 1, ks);
            __builtin_amdgcn_sched_barrier(0);
        }
        add_bias(next);
        __syncthreads();
    };
    // two stages' rows are in flight in registers while a third is multiplied from LDS: one stage's products take less time
    // than its loads.  Loads past the share's end are zeros.
    if (r_begin < r_end) {
        load(ra, r_begin);
        load(rb, r_begin + WK);
#pragma unroll
        for (int j = 0; j < 4; ++j) store(ra, 0, j);
        add_bias(ra);
        __syncthreads();
        for (long long r0 = r_begin; r0 < r_end; r0 += 2 * WK) {
            load(ra, r0 + 2 * WK);
            stage(0, rb);
            load(rb, r0 + 3 * WK);
            stage(1, ra);
        }
    }
    float* part = a.part + ((split * a.to + ot) * a.ti + it) * (long long)(WT * WT);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                part[(wo + 32 * m + (r & 3) + 8 * (r >> 2) + 4 * half) * WT + wi + 32 * n + l31] = acc[m][n][r];
    if (a.bpart && it == 0) {                   // 16 threads hold a column's rows
        float* buf = reinterpret_cast<float*>(lds);
#pragma unroll
        for (int e = 0; e < 8; ++e) buf[prow * 128 + 8 * pc + e] = bias[e];
        __syncthreads();
        if (tid < 128) {
            float t = 0.f;
            for (int j = 0; j < 16; ++j) t += buf[j * 128 + tid];
            a.bpart[(split * a.to + ot) * 128 + tid] = t;
        }
    }
}

// The shares' sums: 32 x four consecutive columns of dw per workgroup, eight threads on each with every eighth share, their
// sums added in order; the workgroups behind those of dw do the same for 32 columns of db.
__global__ __launch_bounds__(256) void rows8_reduce_kernel(const float* part, const float* bpart, float* dw, float* db, int splits,
                                                           int to, int ti, int cout, int cin, unsigned dw_wgs) {
    __shared__ f32x4 sums[8][32];
    const int slot = threadIdx.x & 31, g = threadIdx.x >> 5;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (blockIdx.x < dw_wgs) {
        const long long e = ((long long)blockIdx.x * 32 + slot) * 4;        // cin is a multiple of 8: within a row
        const int o = (int)(e / cin), i = (int)(e - (long long)o * cin);
        if (o < cout) {
            const long long all = (long long)WT * WT * to * ti;
            const float* p = part + ((long long)(o / WT) * ti + i / WT) * (WT * WT) + (o % WT) * WT + i % WT;
#pragma unroll 4
            for (int k = g; k < splits; k += 8) s += *reinterpret_cast<const f32x4*>(p + k * all);
        }
        sums[g][slot] = s;
        __syncthreads();
        if (g == 0 && o < cout) {
#pragma unroll
            for (int j = 1; j < 8; ++j) s += sums[j][slot];
            *reinterpret_cast<f32x4*>(dw + e) = s;
        }
    } else {
        const long long q = (long long)(blockIdx.x - dw_wgs) * 32 + slot;
        if (q < cout)
            for (int k = g; k < splits; k += 8) s[0] += bpart[(long long)k * to * WT + q];
        sums[g][slot] = s;
        __syncthreads();
        if (g == 0 && q < cout) {
#pragma unroll
            for (int j = 1; j < 8; ++j) s[0] += sums[j][slot][0];
            db[q] = s[0];
        }
    }
}

struct Wgrad8Plan { int to, ti, splits; long long per; size_t part, bytes; };

int wgrad8_plan(int cin, int cout, int64_t rows, Wgrad8Plan* p) {
    if (cin <= 0 || cout <= 0 || rows <= 0 || cin % 8 || cout % 8 || cin > (1 << 20) || cout > (1 << 20)) return VDMI_E_SHAPE;
    p->to = (cout + WT - 1) / WT;
    p->ti = (cin + WT - 1) / WT;
    const long long tiles = (long long)p->to * p->ti, stages = (rows + WK - 1) / WK;
    // Shares of the rows: 1, 2, 4 or a multiple of 8 (whole XCDs).  512 workgroups run at once (80 KB of LDS each); a stage of
    // 64 rows takes 0.76 us of a workgroup that has a CU to itself and 1.1 us of two on one CU; a share's partial sums are
    // 128 KB of traffic per tile, at 4 TB/s.  Shares: measured us (with the second launch), rows x cin x cout
    //     131072 x 512 x 1536:  8: 293   16: 292   32: 276   48: 288   64: 299        300 x 512 x 512:  1: 13   2: 12   4: 11
    //     131072 x 256 x 256:   8: 203   32: 60   64: 39   128: 37        4096 x 1024 x 1024:  1: 59   2: 36   4: 27   8: 32
    long long splits = 1;
    double best = 1e30;
    for (long long k = 1; k <= 256 && k <= stages; k += k < 2 ? 1 : k < 4 ? 2 : k < 8 ? 4 : 8) {
        const long long per = (stages + k - 1) / k;
        const long long rounds = k % 8 ? (tiles * k + 511) / 512 : (tiles * (k / 8) + 63) / 64;
        const double us = rounds * per * (tiles * k <= 256 ? 0.76 : 1.1) + 128e3 * tiles * k / 4e6;
        if (us < best) { best = us; splits = k; }
    }
    const long long per = (stages + splits - 1) / splits;
    p->per = per * WK;
    p->splits = (int)splits;            // the last ones may be empty: a multiple of 8 stays one
    // the shares' sums: 128 elements of dw a workgroup, 32 of db
    if (!launch_fits(tiles * p->splits, 256) || !launch_fits((long long)cin * cout / 128 + cout / 32 + 2, 256)) return VDMI_E_SHAPE;
    p->part = (size_t)tiles * p->splits * WT * WT * sizeof(float);
    p->bytes = p->part + (size_t)p->splits * p->to * WT * sizeof(float);
    return VDMI_OK;
}

std::atomic<uint64_t> g_wgrad8_lds{0};

int check_rows8(const void* x, const void* codes, const void* exps, int dtype, int64_t rows, int c, int64_t ldx) {
    if (!x || !codes || !exps) return VDMI_E_ARG;
    if (dtype != VDMI_DT_BF16 && dtype != VDMI_DT_F16 && dtype != VDMI_DT_F32) return VDMI_E_ARG;
    if (rows <= 0 || c <= 0 || c % 8 || c > (1 << 20) || ldx < c || ldx % 8) return VDMI_E_SHAPE;
    // a thread takes eight channels, of the last group also those that are not there
    if (rows > (1LL << 32) || !launch_fits((rows * ((c + 31) / 32) * 4 + 255) / 256, 256)) return VDMI_E_SHAPE;
    if (!aligned16(x) || (reinterpret_cast<uintptr_t>(codes) & 7u)) return VDMI_E_ALIGN;
    return VDMI_OK;
}

}   // namespace

extern "C" int vdmi_rows8_pack(const void* x, int64_t ldx, void* codes, void* exps, int dtype, int64_t rows, int c,
                               vdmi_stream stream) {
    const int ok = check_rows8(x, codes, exps, dtype, rows, c, ldx);
    if (ok != VDMI_OK) return ok;
    const int groups = (c + 31) / 32;
    const PackArgs a = {x, static_cast<unsigned char*>(codes), static_cast<unsigned char*>(exps), ldx, rows * groups * 4, c, groups};
    const dim3 grid((unsigned)((a.total + 255) / 256)), block(256);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == VDMI_DT_BF16) hipLaunchKernelGGL(rows8_pack_kernel<__bf16>, grid, block, 0, st, a);
    else if (dtype == VDMI_DT_F16) hipLaunchKernelGGL(rows8_pack_kernel<_Float16>, grid, block, 0, st, a);
    else hipLaunchKernelGGL(rows8_pack_kernel<float>, grid, block, 0, st, a);
    VDMI_LAUNCH_CHECK();
    return VDMI_OK;
}

extern "C" int vdmi_rows8_unpack(const void* codes, const void* exps, void* x, int64_t ldx, int dtype, int64_t rows, int c,
                                 vdmi_stream stream) {
    const int ok = check_rows8(x, codes, exps, dtype, rows, c, ldx);
    if (ok != VDMI_OK) return ok;
    const UnpackArgs a = {static_cast<const unsigned char*>(codes), static_cast<const unsigned char*>(exps), x, ldx, rows * (c / 8), c,
                          (c + 31) / 32};
    const dim3 grid((unsigned)((a.total + 255) / 256)), block(256);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == VDMI_DT_BF16) hipLaunchKernelGGL(rows8_unpack_kernel<__bf16>, grid, block, 0, st, a);
    else if (dtype == VDMI_DT_F16) hipLaunchKernelGGL(rows8_unpack_kernel<_Float16>, grid, block, 0, st, a);
    else hipLaunchKernelGGL(rows8_unpack_kernel<float>, grid, block, 0, st, a);
    VDMI_LAUNCH_CHECK();
    return VDMI_OK;
}

extern "C" size_t vdmi_rows8_wgrad_workspace_bytes(int cin, int cout, int64_t rows) {
    Wgrad8Plan p;
    return wgrad8_plan(cin, cout, rows, &p) == VDMI_OK ? p.bytes : 0;
}

extern "C" int vdmi_rows8_wgrad(const void* codes, const void* exps, const void* dy, int64_t lddy, float* dw, float* db, int cin,
                                int cout, int64_t rows, void* workspace, vdmi_stream stream) {
    if (!codes || !exps || !dy || !dw || !workspace) return VDMI_E_ARG;
    Wgrad8Plan p;
    const int ok = wgrad8_plan(cin, cout, rows, &p);
    if (ok != VDMI_OK) return ok;
    if (lddy < cout || lddy % 8 || lddy > VDMI_ROWS8_MAX_PITCH) return VDMI_E_SHAPE;
    if (!aligned16(dy) || !aligned16(dw) || !aligned16(workspace) || (reinterpret_cast<uintptr_t>(codes) & 7u)) return VDMI_E_ALIGN;
    const int lds = 4 * WK * WPITCH;
    if (vdmi_set_max_lds(reinterpret_cast<const void*>(&rows8_wgrad_kernel), g_wgrad8_lds, lds) != 0) return VDMI_E_LDS;
    hipStream_t st = static_cast<hipStream_t>(stream);
    Wgrad8Args a;
    a.codes = static_cast<const unsigned char*>(codes); a.exps = static_cast<const unsigned char*>(exps);
    a.dy = static_cast<const __bf16*>(dy);
    a.part = static_cast<float*>(workspace);
    a.bpart = db ? a.part + p.part / sizeof(float) : nullptr;
    a.lddy = lddy; a.rows = rows; a.per = p.per;
    a.cin = cin; a.cout = cout; a.groups = (cin + 31) / 32; a.to = p.to; a.ti = p.ti; a.splits = p.splits;
    hipLaunchKernelGGL(rows8_wgrad_kernel, dim3((unsigned)(p.to * p.ti * p.splits)), dim3(256), lds, st, a);
    VDMI_LAUNCH_CHECK();
    const long long dw_wgs = ((long long)cout * cin + 127) / 128;
    hipLaunchKernelGGL(rows8_reduce_kernel, dim3((unsigned)(dw_wgs + (db ? (cout + 31) / 32 : 0))), dim3(256), 0, st, a.part, a.bpart,
                       dw, db, p.splits, p.to, p.ti, cout, cin, (unsigned)dw_wgs);
    VDMI_LAUNCH_CHECK();
    return VDMI_OK;
}
