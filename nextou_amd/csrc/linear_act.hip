// K10 — point-wise products with their epilogue, forward and backward (gfx950): float32, bfloat16 and float16 rows of any width.
//
//   z[p, gN+n] = sum_k x[p, gK+k] w[gN+n, k] + b[gN+n]          y = act(z) + residual
//   dz = gy act'(z)     dx[p, gK+k] = sum_n dz[p, gN+n] w[gN+n, k]     dw[gN+n, k] = sum_p dz[p, gN+n] x[p, gK+k]     db = sum_p dz
//
// Sums are held in float32; y, dz (16-bit types only: the matrix units read 16-bit operands) and the gradients are rounded once each.
#include "common.h"

namespace nextou {
namespace {

using bf16_t = __bf16;
using f16_t = _Float16;
using f32x16 = __attribute__((ext_vector_type(16))) float;
using u32x4 = __attribute__((ext_vector_type(4))) unsigned;

enum Act { kActNone = 0, kActRelu = 1, kActLeaky = 2, kActGelu = 3, kActHardswish = 4 };

// ---- activations --------------------------------------------------------------------------------------------------------------------
constexpr float kInvSqrt2 = 0.70710678118654752f, kInvSqrt2Pi = 0.39894228040143268f;

// The normal distribution's tail Phi(-|z|), and e = exp(-z^2 / 2) beside it.  float32 rows: the library's erfc (relative accuracy all the
// way).  16-bit rows: Abramowitz and Stegun 7.1.26 (|error| <= 1.5e-7 of erf): five multiply-adds, one exp and one reciprocal, since the epilogue
// of a product that the matrix units finish in microseconds is bound by exactly these instructions.
template <bool FAST>
__device__ __forceinline__ float normal_tail(float z, float* e) {
    if constexpr (FAST) {
        const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * kInvSqrt2, fabsf(z), 1.f));
        float q = fmaf(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
        q = fmaf(q, t, 0.5f * 1.421413741f);
        q = fmaf(q, t, 0.5f * -0.284496736f);
        q = fmaf(q, t, 0.5f * 0.254829592f);
        *e = __builtin_amdgcn_exp2f(z * z * (-0.5f * 1.44269504f));
        return q * t * *e;
    } else {
        *e = expf(-0.5f * z * z);
        return 0.5f * erfcf(fabsf(z) * kInvSqrt2);
    }
}

// (one branch for a piece, not one for every element)
template <bool FAST, int E>
__device__ __forceinline__ void activate(float (&f)[E], int act, float slope) {
    if (act == kActRelu) {
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] = f[i] <= 0.f ? 0.f : f[i];             // (NaN stays NaN)
    } else if (act == kActLeaky) {
        if (slope > 0.f && slope <= 1.f) {
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] = fmaxf(f[i], f[i] * slope);
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] = f[i] > 0.f ? f[i] : f[i] * slope;
        }
    } else if (act == kActGelu) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            // z Phi(z) = max(z, 0) - |z| Phi(-|z|); the tail is 0 long before 1e4 (and stays so at infinity)
            float e;
            const float z = f[i], tail = normal_tail<FAST>(z, &e);
            f[i] = fmaf(-fminf(fabsf(z), 1e4f), tail, z < 0.f ? 0.f : z);
        }
    } else if (act == kActHardswish) {
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] *= fminf(fmaxf(f[i] + 3.f, 0.f), 6.f) * (1.f / 6.f);      // (6 times a large z would leave the range)
    }
}

template <bool FAST>
__device__ __forceinline__ float act_slope(float z, int act, float slope) {
    switch (act) {
        case kActRelu: return z <= 0.f ? 0.f : 1.f;
        case kActLeaky: return z > 0.f ? 1.f : slope;
        case kActGelu: {
            const float c = z > 40.f ? 40.f : (z < -40.f ? -40.f : z);      // beyond that z phi(z) is 0 and must not become inf * 0
            float e;
            const float tail = normal_tail<FAST>(c, &e);
            return fmaf(c * kInvSqrt2Pi, e, c < 0.f ? tail : 1.f - tail);
        }
        case kActHardswish: return z <= -3.f ? 0.f : (z >= 3.f ? 1.f : fmaf(2.f, z, 3.f) * (1.f / 6.f));
        default: return 1.f;
    }
}

// ---- element types ------------------------------------------------------------------------------------------------------------------
// 16-byte pieces at any element-aligned address: the target takes unaligned global accesses, the type says so to the compiler
struct __attribute__((packed, aligned(2))) Piece16 {
    u32x4 v;
};
__device__ __forceinline__ u32x4 load16(const void* p) { return static_cast<const Piece16*>(p)->v; }
__device__ __forceinline__ void store16(void* p, u32x4 v) { static_cast<Piece16*>(p)->v = v; }

template <typename T> struct Num;
template <> struct Num<float> {
    static constexpr int E = 4;                   // elements of a 16-byte piece
    static constexpr bool fast = false;
    using Pre = float;
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned u = v[i];
            f[i] = __builtin_bit_cast(float, u);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[4]) {
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(unsigned, f[i]);
        return v;
    }
    static __device__ __forceinline__ float pre(float z) { return z; }
    static __device__ __forceinline__ u32x4 pack_pre(const float (&f)[4]) { return pack(f); }
    static __device__ __forceinline__ void unpack_pre(u32x4 v, float (&f)[4]) { unpack(v, f); }
    // one k step: lane half h holds 4 consecutive k of its half, so A and B agree whatever k that is
    static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
        float x[4], y[4];
        unpack(a, x);
        unpack(b, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[i], c, 0, 0, 0);
        return c;
    }
};

// What the backward needs of z: float32 for float32 rows, float16 for BOTH 16-bit types (the derivative saturates far inside float16's
// range, and float16's 11 bits keep the saved value's rounding out of the gradients).  A positive z never becomes zero: the sign decides.
__device__ __forceinline__ f16_t pre_half(float z) {
    const float c = z > 65504.f ? 65504.f : (z < -65504.f ? -65504.f : z);
    f16_t h = (f16_t)c;
    if (z > 0.f && h == (f16_t)0.f) h = __builtin_bit_cast(f16_t, (unsigned short)1);
    return h;
}

template <typename T> struct Num16 {
    static constexpr int E = 8;
    static constexpr bool fast = true;
    using Pre = f16_t;
    using V8 = __attribute__((ext_vector_type(8))) T;
    using H8 = __attribute__((ext_vector_type(8))) f16_t;
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[8]) {
        const V8 t = __builtin_bit_cast(V8, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)t[i];
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
        V8 t;
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = (T)f[i];
        return __builtin_bit_cast(u32x4, t);
    }
    static __device__ __forceinline__ f16_t pre(float z) { return pre_half(z); }
    static __device__ __forceinline__ u32x4 pack_pre(const float (&f)[8]) {
        H8 t;
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = pre_half(f[i]);
        return __builtin_bit_cast(u32x4, t);
    }
    static __device__ __forceinline__ void unpack_pre(u32x4 v, float (&f)[8]) {
        const H8 t = __builtin_bit_cast(H8, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)t[i];
    }
};
template <> struct Num<bf16_t> : Num16<bf16_t> {
    static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
    }
};
template <> struct Num<f16_t> : Num16<f16_t> {
    static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
    }
};

// elements [c, c + E) of a row of C columns (zeros behind its end); nothing outside the row is read
template <typename T>
__device__ __forceinline__ u32x4 load_piece(const T* row, long c, long C) {
    constexpr int E = Num<T>::E;
    if (c + E <= C) return load16(row + c);
    T e[E];
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = c + i < C ? row[c + i] : (T)0.f;
    return __builtin_bit_cast(u32x4, e);
}

// The same without a branch around the load, so that many can be in flight (C >= E): the last whole piece of the row is fetched where the
// wanted one would pass its end, and tail_fixed() moves the wanted elements down when the value is used.
template <typename T>
__device__ __forceinline__ u32x4 load_tail(const T* row, long c, long C) {
    return load16(row + min(c, C - Num<T>::E));
}
// (In 32-bit steps.  A form with 64-bit shifts by a register stood in a build whose float32 few_rows_kernel gave wrong results in about one of thirty
// runs; this form and another LDS layout came in one step, and the results have been right since.  Which of the two it was is not known.)
template <typename T>
__device__ __forceinline__ u32x4 tail_fixed(u32x4 v, long c, long C) {
    constexpr int E = Num<T>::E;
    int drop = (int)max(0l, min((long)E, c + E - C));                   // elements: 0 ... E
    unsigned a0 = v[0], a1 = v[1], a2 = v[2], a3 = v[3];
    if constexpr (E == 8) {
        const bool odd = drop & 1;
        const unsigned b0 = a0 >> 16 | a1 << 16, b1 = a1 >> 16 | a2 << 16, b2 = a2 >> 16 | a3 << 16, b3 = a3 >> 16;
        a0 = odd ? b0 : a0, a1 = odd ? b1 : a1, a2 = odd ? b2 : a2, a3 = odd ? b3 : a3;
        drop >>= 1;
    }
    const bool one = drop & 1, two = drop & 2, all = drop & 4;
    a0 = one ? a1 : a0, a1 = one ? a2 : a1, a2 = one ? a3 : a2, a3 = one ? 0 : a3;
    a0 = two ? a2 : a0, a1 = two ? a3 : a1, a2 = two ? 0 : a2, a3 = two ? 0 : a3;
    return u32x4{all ? 0 : a0, all ? 0 : a1, all ? 0 : a2, all ? 0 : a3};
}

// ---- rows times rows: out[m, n] = sum_k A[m, k] B[n, k], both k-contiguous ------------------------------------------------------------
// The forward (A = x, B = w, with the epilogue) and the data gradient (A = dz, B = the transposed weight).
//
// A workgroup of WR x WC waves computes BM x BN outputs; a wave its (BM / WR) x (BN / WC) block out of 32 x 32 matrix-unit tiles, n in the
// tile's rows: a lane ends up with four consecutive n of one m.  k advances in stages of CH 16-byte pieces per row (CH = 8: 64 sixteen-bit
// or 32 float values), two stages kept in LDS as [row][piece] with the piece index XORed by the row, so that the sixteen lanes that are served
// together (16 rows, one piece) fall on all sixteen 16-byte columns of the 64 banks.  In float32 a piece feeds four matrix instructions, in 16 bits one: the same addresses.
//
// DMA = 1: every row starts on 16 bytes and K is a whole number of pieces; stages go from memory to LDS without registers
// (global_load_lds), one barrier a stage.  Rows behind the end are read from the last row (their outputs are not
// stored), pieces behind K from sixteen zero bytes.
// DMA = 0: any alignment and any K; a stage waits in registers while the previous one is multiplied.
//
// Epilogue: the sums go through LDS (the wave's own part of it, 32 rows at a time) so that a lane then holds E consecutive columns of a
// row: bias, activation, residual and the stores are 16-byte accesses of whole lines.
//
// In long products the matrix unit is busy 55 % of the cycles, at a clock that falls to 1.6-1.8 GHz; the waves wait a third of their cycles, 2 % of
// them for LDS, the rest at the stage barriers for loads (8192 x 4096 -> 4096 fetches its operands four times).  Measured: 8192^3 bfloat16 971 us =
// 1130 TFLOP/s, 16384 x 2048 -> 8192 with gelu and z written 642 us, 8192 x 4096 -> 4096 float16 with hardswish 266 us = 1030 TFLOP/s; a library
// product alone of these sizes takes 790, 464 and 191 us.  256 x 128 tiles, four waves of 128 x 128, and four shorter stages in LDS were slower.
__device__ u32x4 g_zero_piece;      // stays zero

struct Epilogue {
    const void* bias;      // per output column (all groups), or NULL
    int bias_f32;
    const void* residual;
    long ldr;
    void* pre;             // dense rows, or NULL
    int act;
    float slope;
};

constexpr int CH = 8, NBUF = 2;     // pieces of a row in a stage, stages in LDS
__device__ __forceinline__ int swizzle(int row, int piece) { return piece ^ ((row >> 1) & 7); }

// LDS written by a wave is read by the same wave's other lanes behind this (its LDS instructions run in order)
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A 32-row strip of a wave's block into LDS: row = lane & 31, and the lane's four consecutive columns per 8 of each 32-column tile
template <int SN, typename F>
__device__ __forceinline__ void put_strip(float* strip, int ld, int lane, F value) {
    const int r32 = lane & 31, half = lane >> 5;
#pragma unroll
    for (int i = 0; i < SN; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<float4*>(strip + r32 * ld + i * 32 + q * 8 + half * 4) =
                make_float4(value(i, q * 4), value(i, q * 4 + 1), value(i, q * 4 + 2), value(i, q * 4 + 3));
    wave_sync();
}

constexpr int kXcds = 8;

// Workgroup -> (m tile, n tile).  The hardware deals workgroups out over the 8 XCDs in turn; each XCD gets a contiguous run of items, and
// items walk 8 m tiles for every n tile, so that what runs together on an XCD shares panels of both operands in its L2.
__device__ __forceinline__ bool tile_of(int block, int grid, int mt, int nt, int* m, int* n) {
    const int per = grid / kXcds;
    const long item = (long)(block % kXcds) * per + block / kXcds;
    if (item >= (long)mt * nt) return false;
    const int band = (int)(item / (8l * nt)), in = (int)(item % (8l * nt));
    const int rows = min(8, mt - band * 8);
    *m = band * 8 + in % rows;
    *n = in / rows;
    return true;
}

// One output row of the epilogue: where its residual, its z and the row itself begin, and how many columns there are in all
template <typename T>
struct OutRow {
    const T* residual;
    typename Num<T>::Pre* pre;
    T* out;
    int C;
    __device__ __forceinline__ OutRow(const Epilogue& e, T* first, long ldo, long m, int C) : C(C) {
        residual = e.residual ? static_cast<const T*>(e.residual) + m * e.ldr : nullptr;
        pre = e.pre ? static_cast<typename Num<T>::Pre*>(e.pre) + m * C : nullptr;
        out = first + m * ldo;
    }
    __device__ __forceinline__ u32x4 fetch(int col) const { return load_tail(residual, col, C); }       // C >= E
};

template <typename T>
__device__ __forceinline__ void finish_piece(float (&f)[Num<T>::E], u32x4 residual, const OutRow<T>& row, int col, int valid, int act, float slope) {
    constexpr int E = Num<T>::E;
    if (row.pre) {
        typename Num<T>::Pre* p = row.pre + col;
        if (valid == E) store16(p, Num<T>::pack_pre(f));
        else
            for (int i = 0; i < E; ++i)
                if (i < valid) p[i] = Num<T>::pre(f[i]);
    }
    activate<Num<T>::fast>(f, act, slope);
    if (row.residual) {
        float r[E];
        if (col + E <= row.C) Num<T>::unpack(residual, r);
        else if (row.C >= E) Num<T>::unpack(tail_fixed<T>(residual, col, row.C), r);
        else
            for (int i = 0; i < E; ++i) r[i] = i < valid ? (float)row.residual[col + i] : 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] += r[i];
    }
    T* out = row.out + col;
    if (valid == E) store16(out, Num<T>::pack(f));
    else
        for (int i = 0; i < E; ++i)
            if (i < valid) out[i] = (T)f[i];
}

// bias of columns col ... col + E - 1 of C (no branch around a load: eight of them in a row would cost eight memory latencies)
template <typename T>
__device__ __forceinline__ void load_bias(float (&b)[Num<T>::E], const Epilogue& e, int col, int C) {
    constexpr int E = Num<T>::E;
#pragma unroll
    for (int i = 0; i < E; ++i) b[i] = 0.f;
    if (!e.bias) return;
    if (e.bias_f32) {
        const float* p = static_cast<const float*>(e.bias);
#pragma unroll
        for (int i = 0; i < E; ++i) b[i] = p[min(col + i, C - 1)];
    } else {
        const T* p = static_cast<const T*>(e.bias);
#pragma unroll
        for (int i = 0; i < E; ++i) b[i] = (float)p[min(col + i, C - 1)];
    }
}

template <typename T, int BM, int BN, int WR, int WC, int DMA>
__global__ __launch_bounds__(64 * WR * WC, (BM / WR) * (BN / WC) > 128 * 64 ? 1 : 2) void rows_gemm_kernel(
    const T* __restrict__ A, const T* __restrict__ B, T* __restrict__ out, long M, int N, int K, long lda, long ldb, long ldo, long bg, int mt, int nt,
    Epilogue e) {
    constexpr int E = Num<T>::E, KE = CH * E, THREADS = 64 * WR * WC, WAVES = WR * WC;
    constexpr int TM = BM / WR, TN = BN / WC, SM = TM / 32, SN = TN / 32;
    constexpr int STAGE = (BM + BN) * CH;                        // pieces
    extern __shared__ u32x4 smem[];
    int mi, ni;
    if (!tile_of(blockIdx.x, gridDim.x, mt, nt, &mi, &ni)) return;
    const int g = blockIdx.y;
    const long m0 = (long)mi * BM;
    const int n0 = ni * BN;
    A += (long)g * K;
    B += g * bg;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave / WC, wn = wave % WC;
    const int stages = (K + KE - 1) / KE;

    f32x16 acc[SN][SM];
#pragma unroll
    for (int i = 0; i < SN; ++i)
#pragma unroll
        for (int j = 0; j < SM; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    auto multiply = [&](const u32x4* buf, int steps) __attribute__((always_inline)) {
        const u32x4* as = buf + (wm * TM) * CH;
        const u32x4* bs = buf + (BM + wn * TN) * CH;
        const int r32 = lane & 31, half = lane >> 5;
#pragma unroll
        for (int ks = 0; ks < CH / 2; ++ks) {
            if (ks < steps) {
                u32x4 a[SM], b[SN];
#pragma unroll
                for (int j = 0; j < SM; ++j) a[j] = as[(j * 32 + r32) * CH + swizzle(r32, ks * 2 + half)];
#pragma unroll
                for (int i = 0; i < SN; ++i) b[i] = bs[(i * 32 + r32) * CH + swizzle(r32, ks * 2 + half)];
#pragma unroll
                for (int i = 0; i < SN; ++i)
#pragma unroll
                    for (int j = 0; j < SM; ++j) acc[i][j] = Num<T>::mma(b[i], a[j], acc[i][j]);
            }
        }
    };
    const int last_steps = ((K - (stages - 1) * KE) + 2 * E - 1) / (2 * E);

    if constexpr (DMA) {
        // a wave's instruction fills 64 pieces: 64 / CH rows; A's BM rows first, then B's
        constexpr int RPI = 64 / CH, INSTR = (BM + BN) / RPI / WAVES;
        const char* src[INSTR];
        int piece[INSTR];
#pragma unroll
        for (int i = 0; i < INSTR; ++i) {
            const int row = (i * WAVES + wave) * RPI + lane / CH;          // INSTR x WAVES x RPI rows, A rows below BM
            const int in = row < BM ? row : row - BM;
            piece[i] = swizzle(in, lane % CH);
            src[i] = row < BM ? reinterpret_cast<const char*>(A + min(m0 + in, M - 1) * lda)
                              : reinterpret_cast<const char*>(B + (long)min(n0 + in, N - 1) * ldb);
        }
        const int pieces = K / E;
        auto fetch = [&](int s) __attribute__((always_inline)) {
            u32x4* buf = smem + (s & 1) * STAGE;
            const bool whole = (s + 1) * CH <= pieces;
#pragma unroll
            for (int i = 0; i < INSTR; ++i) {
                const int pc = s * CH + piece[i];
                const char* from = src[i] + (long)pc * 16;
                if (!whole && pc >= pieces) from = reinterpret_cast<const char*>(&g_zero_piece);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                                 (__attribute__((address_space(3))) void*)(buf + (i * WAVES + wave) * 64), 16, 0, 0);
            }
        };
        // The operands of a k step are read from LDS while the step before it is multiplied, across the stages as well: the barrier that
        // hands a stage over stands in front of the LAST step's multiplication, whose operands are in registers by then, so the buffer
        // just read is free for the stage after the next, and the first operands of the next stage arrive behind the multiplication.
        u32x4 a[2][SM], b[2][SN];
        auto read = [&](int s, int ks, u32x4 (&ra)[SM], u32x4 (&rb)[SN]) __attribute__((always_inline)) {
            const u32x4* at = smem + (s & 1) * STAGE + (lane & 31) * CH + swizzle(lane & 31, ks * 2 + (lane >> 5));
#pragma unroll
            for (int j = 0; j < SM; ++j) ra[j] = at[(wm * TM + j * 32) * CH];
#pragma unroll
            for (int i = 0; i < SN; ++i) rb[i] = at[(BM + wn * TN + i * 32) * CH];
        };
        auto mma = [&](u32x4 (&ra)[SM], u32x4 (&rb)[SN]) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < SN; ++i)
#pragma unroll
                for (int j = 0; j < SM; ++j) acc[i][j] = Num<T>::mma(rb[i], ra[j], acc[i][j]);
        };
        fetch(0);
        if (stages > 1) {
            fetch(1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(INSTR) : "memory");      // loads return in order: stage 0 is there
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        read(0, 0, a[0], b[0]);
        for (int s = 0; s < stages; ++s) {
#pragma unroll
            for (int ks = 0; ks + 1 < CH / 2; ++ks) {
                read(s, ks + 1, a[(ks + 1) & 1], b[(ks + 1) & 1]);
                __builtin_amdgcn_sched_barrier(0);
                mma(a[ks & 1], b[ks & 1]);
            }
            // this wave has its last operands of stage s, and its loads of stage s + 1; then everybody has
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (s + 2 < stages) fetch(s + 2);
            if (s + 1 < stages) read(s + 1, 0, a[0], b[0]);
            __builtin_amdgcn_sched_barrier(0);
            mma(a[1], b[1]);
        }
    } else {
        constexpr int PIECES = STAGE / THREADS;
        u32x4 held[PIECES];
        const int pc = tid % CH;                  // THREADS is a multiple of CH: the same piece of every row
        auto fetch = [&](int s) __attribute__((always_inline)) {
            const long k = (long)s * KE + pc * E;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int row = (i * THREADS + tid) / CH;
                const T* at = row < BM ? A + min(m0 + row, M - 1) * lda : B + (long)min(n0 + (row - BM), N - 1) * ldb;
                held[i] = K >= E ? load_tail(at, k, K) : load_piece(at, k, K);
            }
        };
        auto keep = [&](int s) __attribute__((always_inline)) {
            u32x4* buf = smem + (s & 1) * STAGE;
            const bool whole = (s + 1) * KE <= K || K < E;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int row = (i * THREADS + tid) / CH;
                buf[row * CH + swizzle(row < BM ? row : row - BM, pc)] = whole ? held[i] : tail_fixed<T>(held[i], (long)s * KE + pc * E, K);
            }
        };
        fetch(0);
        keep(0);
        __syncthreads();
        for (int s = 0; s < stages; ++s) {
            if (s + 1 < stages) fetch(s + 1);
            multiply(smem + (s & 1) * STAGE, s + 1 < stages ? CH / 2 : last_steps);
            if (s + 1 < stages) keep(s + 1);      // into the buffer that the multiplication before this one read
            __syncthreads();
        }
    }

    // epilogue
    constexpr int LD = TN + 4;                    // floats
    static_assert(32 * LD * 4 * WAVES <= STAGE * 16 * NBUF, "a wave's strip has to fit into the stages' LDS");
    float* strip = reinterpret_cast<float*>(smem) + wave * 32 * LD;
    if constexpr (DMA) __syncthreads();
    constexpr int LPR = TN / E, RPI = 64 / LPR;   // lanes per row, rows per pass
    const int col = n0 + wn * TN + (lane % LPR) * E;
    const int valid = min(E, N - col);
    const int oc = g * N + col, C = (int)gridDim.y * N;
    float bias[E];
    load_bias<T>(bias, e, oc, C);
#pragma unroll
    for (int j = 0; j < SM; ++j) {
        const long mj = m0 + wm * TM + j * 32 + lane / LPR;
        u32x4 add[32 / RPI];
#pragma unroll
        for (int r = 0; r < 32 / RPI; ++r)
            if (e.residual && valid > 0 && C >= E) add[r] = OutRow<T>(e, out, ldo, min(mj + r * RPI, M - 1), C).fetch(oc);
        put_strip<SN>(strip, LD, lane, [&](int i, int r) { return acc[i][j][r]; });
#pragma unroll
        for (int r = 0; r < 32 / RPI; ++r) {
            const long m = mj + r * RPI;
            float f[E];
#pragma unroll
            for (int q = 0; q < E; q += 4) {
                const float4 v = *reinterpret_cast<const float4*>(strip + (r * RPI + lane / LPR) * LD + (lane % LPR) * E + q);
                f[q] = v.x, f[q + 1] = v.y, f[q + 2] = v.z, f[q + 3] = v.w;
            }
#pragma unroll
            for (int q = 0; q < E; ++q) f[q] += bias[q];
            if (m < M && valid > 0) finish_piece<T>(f, add[r], OutRow<T>(e, out, ldo, m, C), oc, valid, e.act, e.slope);
        }
        wave_sync();
    }
}

template <typename T, int BM, int BN, int WR, int WC, int DMA>
int launch_rows_gemm(const T* A, const T* B, T* out, long M, int N, int K, int groups, long lda, long ldb, long ldo, long bg, const Epilogue& e,
                     hipStream_t s) {
    const int mt = (int)cdiv64(M, BM), nt = cdiv(N, BN);
    const size_t lds = (size_t)(BM + BN) * CH * 16 * NBUF;
    auto* kernel = &rows_gemm_kernel<T, BM, BN, WR, WC, DMA>;
    if (lds > 65536) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    const int64_t blocks = cdiv64((int64_t)mt * nt, kXcds) * kXcds;
    // (rows of a stride of 0 make such calls possible: their number is not bound by the memory that x takes)
    NEXTOU_REQUIRE(blocks * 64 * WR * WC < (1ll << 32), "linear_act: %ld rows of %d columns are more than one launch takes", M, N);
    const dim3 grid((unsigned)blocks, (unsigned)groups);
    hipLaunchKernelGGL((rows_gemm_kernel<T, BM, BN, WR, WC, DMA>), grid, dim3(64 * WR * WC), lds, s, A, B, out, M, N, K, lda, ldb, ldo, bg,
                       mt, nt, e);
    return 0;
}

bool on16(const void* p, long ld, size_t size) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * (long)size % 16 == 0; }

// ---- the weight gradient: out[n, k] = sum_p G[p, n] X[p, k], both reduced over their ROWS ------------------------------------------------
// A stage is KP rows of BC columns of each operand, as they lie in memory.  16 bits: the matrix unit wants 8 consecutive p of one column per
// lane, which ds_read_tr16_b64 delivers: the 16 lanes of a group name 4 rows x 16 columns (8 bytes each) and each receives one column's
// four values.  The 64-byte granules of a row are XORed by the row so that the four rows fall on different banks.  float32: the
// instruction takes one p per lane half, plain 4-byte reads.
// k is put in the tile's rows, so a lane ends up with consecutive k and the epilogue above stores whole lines of the weight's layout.
// p is split over blockIdx.z when there are few tiles: float32 partial blocks, added in a fixed order by split_sum_kernel.
// Measured: 16384 rows, 8192 x 2048 bfloat16 612 us = 900 TFLOP/s (256 tiles; 776 us with 128); 21504 rows, 1056 x 264 67 us = 179 TFLOP/s, where
// 3 x 9 tiles of 128 hold 264 x 1056 columns to 69 % and 486 workgroups read x nine times and dz three times: 192 MB come from memory for 57, the
// waves wait half of their cycles.
template <typename T, int BC>
__device__ __forceinline__ int col_swizzle(int row, int piece) {
    if constexpr (sizeof(T) == 4) return piece;
    else if constexpr (BC == 64) return piece ^ (((row >> 1) & 1) << 2);
    else return piece ^ ((row & 3) << 2);
}

template <typename T, int BC, int WR, int WC, int DMA>
__global__ __launch_bounds__(64 * WR * WC, 2) void cols_gemm_kernel(const T* __restrict__ G, const T* __restrict__ X, T* __restrict__ out,
                                                                    float* __restrict__ partial, long P, int N, int K, long ldg, long ldx, int nt,
                                                                    int kt, long rows_per_split) {
    constexpr int E = Num<T>::E, CP = BC / E, THREADS = 64 * WR * WC, WAVES = WR * WC;
    constexpr int KP = sizeof(T) == 4 ? 32 : 64, HALF = KP * CP, STAGE = 2 * HALF;       // pieces; G's tile, then X's
    constexpr int TM = BC / WR, TN = BC / WC, SM = TM / 32, SN = TN / 32;
    extern __shared__ u32x4 smem[];
    int ni, ki;
    if (!tile_of(blockIdx.x, gridDim.x, nt, kt, &ni, &ki)) return;
    const int g = blockIdx.y, n0 = ni * BC, k0 = ki * BC;
    const long p_from = (long)blockIdx.z * rows_per_split, p_to = min(P, p_from + rows_per_split);
    G += (long)g * N;
    X += (long)g * K;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave / WC, wn = wave % WC;
    const int stages = (int)((p_to - p_from + KP - 1) / KP);

    f32x16 acc[SN][SM];
#pragma unroll
    for (int i = 0; i < SN; ++i)
#pragma unroll
        for (int j = 0; j < SM; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    // 16 bits: k step ks of the 32 columns from c0 of a tile, one column per lane
    auto columns = [&](const u32x4* tile, int ks, int c0) __attribute__((always_inline)) {
        using S4 = __attribute__((ext_vector_type(4))) short;
        const int row = ks * 16 + 8 * (lane >> 5) + ((lane >> 2) & 3), col = c0 + 16 * ((lane >> 4) & 1) + (lane & 3) * 4;
        const char* at = reinterpret_cast<const char*>(tile) + (row * CP + col_swizzle<T, BC>(row, col / 8)) * 16 + (col & 4) * 2;
        // four rows further: the same swizzle
        const S4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) S4*)at);
        const S4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) S4*)(at + 4 * CP * 16));
        return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto read = [&](const u32x4* buf, int ks, u32x4 (&a)[SM], u32x4 (&b)[SN]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < SM; ++j) a[j] = columns(buf, ks, wm * TM + j * 32);
#pragma unroll
        for (int i = 0; i < SN; ++i) b[i] = columns(buf + HALF, ks, wn * TN + i * 32);
    };
    auto mma = [&](u32x4 (&a)[SM], u32x4 (&b)[SN]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < SN; ++i)
#pragma unroll
            for (int j = 0; j < SM; ++j) acc[i][j] = Num<T>::mma(b[i], a[j], acc[i][j]);
    };
    auto multiply = [&](const u32x4* buf) __attribute__((always_inline)) {
        if constexpr (sizeof(T) == 4) {
            const float* gs = reinterpret_cast<const float*>(buf);
            const float* xs = gs + KP * BC;
            const int r32 = lane & 31, half = lane >> 5;
#pragma unroll 8
            for (int kk = 0; kk < KP / 2; ++kk) {
                float a[SM], b[SN];
#pragma unroll
                for (int j = 0; j < SM; ++j) a[j] = gs[(kk * 2 + half) * BC + wm * TM + j * 32 + r32];
#pragma unroll
                for (int i = 0; i < SN; ++i) b[i] = xs[(kk * 2 + half) * BC + wn * TN + i * 32 + r32];
#pragma unroll
                for (int i = 0; i < SN; ++i)
#pragma unroll
                    for (int j = 0; j < SM; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(b[i], a[j], acc[i][j], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int ks = 0; ks < KP / 16; ++ks) {
                u32x4 a[SM], b[SN];
                read(buf, ks, a, b);
                mma(a, b);
            }
        }
    };

    if constexpr (DMA) {
        constexpr int INSTR = STAGE / 64 / WAVES;
        auto fetch = [&](int s) __attribute__((always_inline)) {
            u32x4* buf = smem + (s & 1) * STAGE;
#pragma unroll
            for (int i = 0; i < INSTR; ++i) {
                const int q = (i * WAVES + wave) * 64 + lane, in = q < HALF ? q : q - HALF;
                const int row = in / CP, piece = col_swizzle<T, BC>(row, in % CP);
                const long p = p_from + (long)s * KP + row;
                const int c = (q < HALF ? n0 : k0) + piece * E;
                const char* from = reinterpret_cast<const char*>(&g_zero_piece);
                if (p < p_to && c < (q < HALF ? N : K)) from = reinterpret_cast<const char*>(q < HALF ? G + p * ldg + c : X + p * ldx + c);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                                 (__attribute__((address_space(3))) void*)(buf + (i * WAVES + wave) * 64), 16, 0, 0);
            }
        };
        if constexpr (sizeof(T) == 2) {                // handed over as in rows_gemm_kernel, in front of the last k step's multiplication
            constexpr int STEPS = KP / 16;
            u32x4 a[2][SM], b[2][SN];
            fetch(0);
            if (stages > 1) {
                fetch(1);
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(INSTR) : "memory");
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            read(smem, 0, a[0], b[0]);
            for (int s = 0; s < stages; ++s) {
#pragma unroll
                for (int ks = 0; ks + 1 < STEPS; ++ks) {
                    read(smem + (s & 1) * STAGE, ks + 1, a[(ks + 1) & 1], b[(ks + 1) & 1]);
                    __builtin_amdgcn_sched_barrier(0);
                    mma(a[ks & 1], b[ks & 1]);
                }
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                if (s + 2 < stages) fetch(s + 2);
                if (s + 1 < stages) read(smem + ((s + 1) & 1) * STAGE, 0, a[0], b[0]);
                __builtin_amdgcn_sched_barrier(0);
                mma(a[1], b[1]);
            }
        } else {
            fetch(0);
            for (int s = 0; s < stages; ++s) {
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                if (s + 1 < stages) fetch(s + 1);
                multiply(smem + (s % NBUF) * STAGE);
            }
        }
        __syncthreads();
    } else {
        constexpr int PIECES = STAGE / THREADS;
        u32x4 held[PIECES];
        const bool cols_whole = n0 + BC <= N && k0 + BC <= K, narrow = N < E || K < E;
        auto fetch = [&](int s) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int q = i * THREADS + tid, in = q < HALF ? q : q - HALF;
                const int c = (q < HALF ? n0 : k0) + (in % CP) * E, C = q < HALF ? N : K;
                const long p = min(p_from + (long)s * KP + in / CP, p_to - 1);
                const T* at = q < HALF ? G + p * ldg : X + p * ldx;
                held[i] = narrow ? load_piece(at, c, C) : load_tail(at, c, C);
            }
        };
        auto keep = [&](int s) __attribute__((always_inline)) {
            u32x4* buf = smem + (s & 1) * STAGE;
            const long left = p_to - p_from - (long)s * KP;
            const bool whole = (cols_whole || narrow) && left >= KP;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int q = i * THREADS + tid, in = q < HALF ? q : q - HALF, row = in / CP;
                u32x4 v = held[i];
                if (!whole) {
                    if (!narrow) v = tail_fixed<T>(v, (q < HALF ? n0 : k0) + (in % CP) * E, q < HALF ? N : K);
                    if (row >= left) v = u32x4{0, 0, 0, 0};
                }
                buf[q - in + row * CP + col_swizzle<T, BC>(row, in % CP)] = v;
            }
        };
        fetch(0);
        keep(0);
        __syncthreads();
        for (int s = 0; s < stages; ++s) {
            if (s + 1 < stages) fetch(s + 1);
            multiply(smem + (s & 1) * STAGE);
            if (s + 1 < stages) keep(s + 1);
            __syncthreads();
        }
    }

    constexpr int LD = TN + 4;
    static_assert(32 * LD * 4 * WAVES <= STAGE * 16 * NBUF, "a wave's strip has to fit into the stages' LDS");
    float* strip = reinterpret_cast<float*>(smem) + wave * 32 * LD;
    const long block = (long)g * N * K;
    if (partial) partial += ((long)blockIdx.z * gridDim.y) * N * K + block;
    else out += block;
#pragma unroll
    for (int j = 0; j < SM; ++j) {
        put_strip<SN>(strip, LD, lane, [&](int i, int r) { return acc[i][j][r]; });
        constexpr int LPR = TN / 4, RPI = 64 / LPR;
        const int k = k0 + wn * TN + (lane % LPR) * 4;
#pragma unroll
        for (int r = 0; r < 32; r += RPI) {
            const int row = r + lane / LPR, n = n0 + wm * TM + j * 32 + row;
            const float4 v = *reinterpret_cast<const float4*>(strip + row * LD + (lane % LPR) * 4);
            const float f[4] = {v.x, v.y, v.z, v.w};
            if (n < N) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (k + q < K) {
                        if (partial) partial[(long)n * K + k + q] = f[q];
                        else out[(long)n * K + k + q] = (T)f[q];
                    }
            }
        }
        wave_sync();
    }
}

// out[i] = sum over splits of partial[split][i], in a fixed order: `parts` threads take a contiguous run of the splits each (one when there
// are few: then every thread reads whole lines), and their sums are added in order.  Two such sums in one launch: the bias's and the weight's.
struct SplitSum {
    const float* partial;
    void* out;
    int out_f32, splits, parts;
    long n;
    unsigned blocks;
};

template <typename T>
__global__ __launch_bounds__(256) void split_sum_kernel(SplitSum first, SplitSum second) {
    __shared__ float sums[256];
    const bool is_first = blockIdx.x < first.blocks;
    const SplitSum& a = is_first ? first : second;
    const int per = 256 / a.parts, part = threadIdx.x / per;
    const long i = (long)(is_first ? blockIdx.x : blockIdx.x - first.blocks) * per + threadIdx.x % per;
    const int from = (int)((long)a.splits * part / a.parts), to = (int)((long)a.splits * (part + 1) / a.parts);
    float t = 0.f;
    if (i < a.n) {
#pragma unroll 8
        for (int s = from; s < to; ++s) t += a.partial[s * a.n + i];
    }
    sums[threadIdx.x] = t;
    __syncthreads();
    if (part != 0 || i >= a.n) return;
    for (int q = 1; q < a.parts; ++q) t += sums[q * per + threadIdx.x];
    if (a.out_f32) static_cast<float*>(a.out)[i] = t;
    else static_cast<T*>(a.out)[i] = (T)t;
}

// ---- the backward's preparation: the activation's gradient with the column sums, and the transposed weight ----------------------------------
// w (groups * N, K) -> wt (groups * K, ldt >= N), columns behind N zero: the data gradient's second operand with n contiguous
template <typename T>
__device__ __forceinline__ void transpose_weight(T (&tile)[64][66], const T* __restrict__ w, T* __restrict__ wt, int N, int K, int ldt, unsigned block) {
    const int nt = (ldt + 63) / 64, kt = (K + 63) / 64;
    const int n0 = (int)(block % nt) * 64, k0 = (int)(block / nt % kt) * 64;
    const long g = block / nt / kt;
    w += g * N * K;
    wt += g * K * ldt;
    constexpr int E = Num<T>::E, LPR = 64 / E;
#pragma unroll
    for (int j = 0; j < 64 * LPR / 256; ++j) {
        const int i = j * 256 + threadIdx.x, r = i / LPR, c = i % LPR * E;
        T v[E];
        u32x4 piece{0, 0, 0, 0};
        if (n0 + r < N && k0 + c < K) piece = load_piece(w + (long)(n0 + r) * K, k0 + c, K);
        __builtin_memcpy(v, &piece, 16);
#pragma unroll
        for (int q = 0; q < E; ++q) tile[r][c + q] = v[q];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 64 * LPR / 256; ++j) {
        const int i = j * 256 + threadIdx.x, r = i / LPR, c = i % LPR * E;
        if (k0 + r >= K || n0 + c >= ldt) continue;             // ldt is a whole number of pieces
        T v[E];
        u32x4 piece;
#pragma unroll
        for (int q = 0; q < E; ++q) v[q] = tile[c + q][r];
        __builtin_memcpy(&piece, v, 16);
        store16(wt + (long)(k0 + r) * ldt + n0 + c, piece);
    }
}

// dz = gy act'(saved) as dense rows of ld_dz columns (a multiple of 16 bytes, so that both products fetch it without registers; the columns
// behind C are zeros), and per-workgroup column sums of the unrounded dz.  A workgroup holds `lanes` 16-byte pieces of a row and 256 / lanes
// rows at a time; the pieces walk fastest over the workgroups.  Reads gy and the saved tensor, writes dz: HBM-bound
// (21504 x 1056 bfloat16 with gelu: 136 MB in 40 us, 3.4 TB/s).  The rounding of dz to 16 bits is the matrix units': the gradients of a bfloat16
// layer are 0.0023 off the 64-bit ones in norm, where the rounding of the outputs alone gives 0.0017; a second 16-bit part would double both
// products.  The weight is transposed by the workgroups behind `act_blocks`, in the same
// launch (5 us less than in one of its own).
// KIND 0: no activation (only the sums), 1: saved is z, 2: saved is y and only its sign matters
template <typename T, int KIND>
__global__ __launch_bounds__(256) void act_grad_kernel(const T* __restrict__ gy, const void* __restrict__ saved, T* __restrict__ dz,
                                                       float* __restrict__ sums, long P, long C, long ldg, long ld_dz, int lanes, long rows_per_block,
                                                       int act, float slope, int col_blocks, unsigned act_blocks, const T* __restrict__ w,
                                                       T* __restrict__ wt, int N, int K, int ldt) {
    constexpr int E = Num<T>::E;
    __shared__ union {
        float part[256][E + 1];
        T tile[64][66];
    } lds;
    if (blockIdx.x >= act_blocks) {
        transpose_weight<T>(lds.tile, w, wt, N, K, ldt, blockIdx.x - act_blocks);
        return;
    }
    auto& part = lds.part;
    const int rows = 256 / lanes, r = threadIdx.x / lanes, piece = (int)(blockIdx.x % col_blocks) * lanes + threadIdx.x % lanes;
    const long c = (long)piece * E, row_block = blockIdx.x / col_blocks;
    const long from = row_block * rows_per_block, to = min(P, from + rows_per_block);
    float acc[E];
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = 0.f;
    if (r < rows && c < ld_dz) {
        const int valid = (int)max(0l, min((long)E, C - c));
#pragma unroll 4
        for (long p = from + r; p < to; p += rows) {
            float f[E];
            Num<T>::unpack(load_piece(gy + p * ldg + c, 0, valid), f);
            if constexpr (KIND == 1) {
                float s[E];
                Num<T>::unpack_pre(load_piece(static_cast<const typename Num<T>::Pre*>(saved) + p * C + c, 0, valid), s);
#pragma unroll
                for (int i = 0; i < E; ++i) f[i] *= act_slope<Num<T>::fast>(s[i], act, slope);
            }
            if constexpr (KIND == 2) {
                float s[E];
                Num<T>::unpack(load_piece(static_cast<const T*>(saved) + p * C + c, 0, valid), s);
#pragma unroll
                for (int i = 0; i < E; ++i) f[i] *= act == kActRelu ? (s[i] <= 0.f ? 0.f : 1.f) : (s[i] > 0.f ? 1.f : slope);
            }
            if constexpr (KIND != 0) {
                if (dz) {
#pragma unroll
                    for (int i = 0; i < E; ++i)
                        if (i >= valid) f[i] = 0.f;
                    store16(dz + p * ld_dz + c, Num<T>::pack(f));
                }
            }
#pragma unroll
            for (int i = 0; i < E; ++i) acc[i] += f[i];
        }
    }
    if (!sums) return;
#pragma unroll
    for (int i = 0; i < E; ++i) part[threadIdx.x][i] = acc[i];
    __syncthreads();
    if (r == 0 && c < C) {
        for (int i = 0; i < E && c + i < C; ++i) {
            float t = 0.f;
            for (int q = 0; q < rows; ++q) t += part[q * lanes + threadIdx.x][i];
            sums[row_block * C + c + i] = t;
        }
    }
}

// ---- many rows, short k: the weight stays in LDS ---------------------------------------------------------------------------------------
// With k of a few hundred, the products above spend their time on stages and barriers while memory waits.  Here a workgroup (one per CU, 8
// waves) keeps a panel of the weight in LDS for all its rows, and every wave for itself takes 32 rows at a time: its piece of x goes straight from
// memory into the matrix unit's operand registers (lane = row, 16 bytes of k), all of k at once, and is used for every 32 columns of the
// panel.  x is read once per panel, no barrier after the panel is there, and two waves a SIMD cover each other's loads.
// The panel is `pg` whole groups, or `pn` columns of one group when that is too large for LDS.
// Panel rows lie an odd number of pieces apart, so that eight consecutive rows fall on all banks.
// Results stay in registers: the lane halves of a 32 x 32 tile hold alternate groups of four columns; in 16 bits an exchange between the
// halves makes that eight consecutive columns, so residual, z and output move as 16-byte pieces.
// 172032 rows 132 -> 528 bfloat16 87 us = 2.6 TB/s, 6 groups of 44 -> 44 float32 120 us = 3.0 TB/s; a copy reaches 4.9.  No unit is full (bfloat16: VALU
// 37 % of the cycles, matrix unit 15, waves waiting 26; float32 24, 38, 20), and 10-14 % more is written than the output (lines that two 16-byte
// pieces of different waves complete).  1024 threads, two tiles at a time, output lines gathered in LDS,
// and stores past the caches (215 us) were no faster.
// KS: k steps (two pieces each), zeros behind K; LOW: the steps that are whole in every K of this size.
template <int E, int N>
__device__ __forceinline__ const float (&piece(const float (&f)[N], int q))[E] {
    return *reinterpret_cast<const float(*)[E]>(&f[q * E]);
}

constexpr int kPanelThreads = 512;                              // two waves a SIMD, 256 registers each

template <typename T, int LOW, int KS>
__global__ __launch_bounds__(kPanelThreads, 2) void panel_gemm_kernel(const T* __restrict__ X, const T* __restrict__ W, T* __restrict__ out, long M,
                                                                          int N, int K, int groups, long ldx, long ldw, long ldo, long wg, int pg,
                                                                          int pn, int parts, Epilogue e) {
    constexpr int E = Num<T>::E, THREADS = kPanelThreads, WAVES = THREADS / 64, PITCH = 2 * KS + 1;
    extern __shared__ u32x4 smem[];
    const int npg = (N + pn - 1) / pn;                          // panels per group (1 when a panel holds whole groups)
    const int g0 = (int)blockIdx.y / npg * pg, g1 = min(groups, g0 + pg);
    const int n0 = (int)blockIdx.y % npg * pn, n1 = min(N, n0 + pn), rows = n1 - n0, rows32 = (rows + 31) / 32 * 32;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r32 = lane & 31, half = lane >> 5;
    float* biases = reinterpret_cast<float*>(smem + pg * pn * PITCH);
    {
        constexpr int AHEAD = 4;                                // loads in flight per thread
        const int total = (g1 - g0) * rows * KS * 2;
        for (int i = threadIdx.x; i < total; i += AHEAD * THREADS) {
            u32x4 v[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int q = min(i + j * THREADS, total - 1), row = q / (KS * 2);
                v[j] = load_tail(W + (g0 + row / rows) * wg + (long)(n0 + row % rows) * ldw, q % (KS * 2) * E, K);
            }
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int q = i + j * THREADS, pc = q % (KS * 2);
                if (q < total) smem[q / (KS * 2) * PITCH + pc] = tail_fixed<T>(v[j], pc * E, K);
            }
        }
    }
    for (int i = threadIdx.x; i < (g1 - g0) * rows32; i += THREADS) {
        const int n = i % rows32;
        const long c = (long)(g0 + i / rows32) * N + n0 + n;
        float b = 0.f;
        if (e.bias && n < rows) b = e.bias_f32 ? static_cast<const float*>(e.bias)[c] : (float)static_cast<const T*>(e.bias)[c];
        biases[i] = b;
    }
    __syncthreads();
    const long tiles = (M + 31) / 32;
    const int C = groups * N;
    // items: (32 rows, group, part of the panel's columns), rows slowest
    const int per_row = (g1 - g0) * parts;
    auto fetch = [&](long item, u32x4 (&x)[KS]) __attribute__((always_inline)) {
        const T* at = X + min(item / per_row * 32 + r32, M - 1) * ldx + (long)(g0 + (int)(item % per_row) / parts) * K;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) x[ks] = ks < LOW ? load16(at + half * E + ks * 2 * E) : load_tail(at, (ks * 2 + half) * E, K);
    };
    const long items = tiles * per_row, stride = (long)gridDim.x * WAVES, first = (long)blockIdx.x * WAVES + wave;
    u32x4 x[2][KS];                                             // this item's x and the next one's
    if (first < items) fetch(first, x[0]);
    auto one = [&](long item, u32x4 (&xi)[KS], u32x4 (&xn)[KS]) __attribute__((always_inline)) {
        fetch(min(item + stride, items - 1), xn);
        if (K != 2 * KS * E) {                                  // KS is the next size above: zeros behind K
#pragma unroll
            for (int ks = LOW; ks < KS; ++ks) xi[ks] = tail_fixed<T>(xi[ks], (ks * 2 + half) * E, K);
        }
        const long m = item / per_row * 32 + r32;
        const OutRow<T> orow(e, out, ldo, min(m, M - 1), C);
        const int g = g0 + (int)(item % per_row) / parts, part = (int)(item % parts);
        const int cols = (rows32 / 32 + parts - 1) / parts * 32, c_from = part * cols, c_to = min(rows, c_from + cols);
        const u32x4* panel = smem + (g - g0) * rows * PITCH + half;
        const float* bs = biases + (g - g0) * rows32;
        for (int c0 = c_from; c0 < c_to; c0 += 32) {
            const u32x4* wrow = panel + min(c0 + r32, rows - 1) * PITCH;
            u32x4 w[4];                                         // the panel's pieces are read three k steps ahead of the matrix unit
#pragma unroll
            for (int ks = 0; ks < 3; ++ks) w[ks] = wrow[min(ks, KS - 1) * 2];
            f32x16 acc;                                         // bias first: the sums start from it
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 v = *reinterpret_cast<const float4*>(bs + c0 + q * 8 + half * 4);
                acc[q * 4] = v.x, acc[q * 4 + 1] = v.y, acc[q * 4 + 2] = v.z, acc[q * 4 + 3] = v.w;
            }
            const int col0 = g * N + n0 + c0 + half * E;
            u32x4 add[16 / E];
            if (e.residual) {
#pragma unroll
                for (int q = 0; q < 16 / E; ++q) add[q] = orow.fetch(min(col0 + q * 2 * E, C - 1));
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (ks + 3 < KS) w[(ks + 3) % 4] = wrow[(ks + 3) * 2];
                __builtin_amdgcn_sched_barrier(0);
                acc = Num<T>::mma(w[ks % 4], xi[ks], acc);
            }
            float f[16];                                        // piece q: columns 16 q + 8 half + 0..7 (16 bits), 8 q + 4 half + 0..3 (float32)
            if constexpr (E == 8) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float lower = acc[i / 4 * 8 + i % 4], upper = acc[i / 4 * 8 + 4 + i % 4];
                    const auto both = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, lower), __builtin_bit_cast(unsigned, upper), false,
                                                                       false);
                    const unsigned lo = both[0], hi = both[1];
                    f[i / 4 * 8 + i % 4] = __builtin_bit_cast(float, lo);
                    f[i / 4 * 8 + 4 + i % 4] = __builtin_bit_cast(float, hi);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) f[i] = acc[i];
            }
            // whole pieces, predicated by the lane's row and columns; where the columns end inside a piece, its elements one by one (a
            // branch that is the same for all lanes, taken for the last tile of an odd width)
            const bool mine = m < M, ragged = rows % E != 0 && c0 + 32 > rows;
            const int left = rows - c0 - half * E;              // columns from this lane's first
            if (e.pre) {
#pragma unroll
                for (int q = 0; q < 16 / E; ++q) {
                    typename Num<T>::Pre* at = orow.pre + col0 + q * 2 * E;
                    if (mine && left >= q * 2 * E + E) store16(at, Num<T>::pack_pre(piece<E>(f, q)));
                    else if (ragged && mine) {
#pragma unroll
                        for (int i = 0; i < E; ++i)
                            if (left > q * 2 * E + i) at[i] = Num<T>::pre(f[q * E + i]);
                    }
                }
            }
            activate<Num<T>::fast>(f, e.act, e.slope);
            if (e.residual) {
                const bool end = g * N + n0 + c0 + 32 > C;      // pieces that pass the row's end were fetched from in front of it
#pragma unroll
                for (int q = 0; q < 16 / E; ++q) {
                    float r[E];
                    Num<T>::unpack(end ? tail_fixed<T>(add[q], min(col0 + q * 2 * E, C - 1), C) : add[q], r);
#pragma unroll
                    for (int i = 0; i < E; ++i) f[q * E + i] += r[i];
                }
            }
#pragma unroll
            for (int q = 0; q < 16 / E; ++q) {
                T* at = orow.out + col0 + q * 2 * E;
                if (mine && left >= q * 2 * E + E) store16(at, Num<T>::pack(piece<E>(f, q)));
                else if (ragged && mine) {
#pragma unroll
                    for (int i = 0; i < E; ++i)
                        if (left > q * 2 * E + i) at[i] = (T)f[q * E + i];
                }
            }
        }
    };
    for (long item = first; item < items; item += 2 * stride) {
        one(item, x[0], x[1]);
        if (item + stride < items) one(item + stride, x[1], x[0]);
    }
}

constexpr int kPanelLds = 160 * 1024;

// A panel for these sizes; 0 columns: the rows do not fit the registers
struct PanelPlan {
    int ks, pg, pn, pitch, panels;
    size_t lds;
};
PanelPlan plan_panel(int N, int K, int groups, size_t S) {
    PanelPlan p{};
    const int E = (int)(16 / S), steps = cdiv(K, 2 * E);
    static const int sizes[] = {3, 6, 9, 13, 17};
    for (int ks : sizes)
        if (!p.ks && steps <= ks) p.ks = ks;
    if (K < E || groups * N < E) p.ks = 0;
    if (!p.ks) return p;
    p.pitch = 2 * p.ks + 1;
    const int room = (kPanelLds - 128) / (p.pitch * 16 + 4);    // columns, each with its bias (those in whole 32s)
    if (N <= room) {
        p.pn = N;
        p.pg = kPanelLds / (N * p.pitch * 16 + cdiv(N, 32) * 128);
        if (p.pg < 1) p.pg = 1;
        if (p.pg > groups) p.pg = groups;
        p.pg = cdiv(groups, cdiv(groups, p.pg));
        p.panels = cdiv(groups, p.pg);
    } else {
        p.pg = 1;
        const int per = cdiv(N, room / 32 * 32);
        p.pn = cdiv(cdiv(N, per), 32) * 32;
        p.panels = groups * cdiv(N, p.pn);
    }
    p.lds = (size_t)p.pg * (p.pn * p.pitch * 16 + cdiv(p.pn, 32) * 128);
    return p;
}

template <typename T, int LOW, int KS>
void launch_panel(const T* A, const T* B, T* out, long M, int N, int K, int groups, long lda, long ldb, long ldo, long bg, const Epilogue& e,
                  const PanelPlan& p, hipStream_t s) {
    constexpr int THREADS = kPanelThreads;
    auto* kernel = &panel_gemm_kernel<T, LOW, KS>;
    if (p.lds > 65536) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)p.lds);
    const int per_cu = p.lds <= kPanelLds / 2 ? 2 : 1;
    int64_t wgs = cdiv(256 * per_cu, p.panels);
    if (wgs > cdiv64(M, THREADS / 2)) wgs = cdiv64(M, THREADS / 2);
    // 32 rows are a large item for a wave that gets one or two of them: the columns in up to four parts, where that evens the waves out
    const int64_t items = cdiv64(M, 32) * p.pg, waves = wgs * (THREADS / 64);
    int parts = 1;
    for (int q = 2; q <= 4 && q * 3 <= cdiv(p.pn, 32); ++q)
        if (cdiv64(items * q, waves) * parts < cdiv64(items * parts, waves) * q) parts = q;
    hipLaunchKernelGGL((panel_gemm_kernel<T, LOW, KS>), dim3((unsigned)wgs, (unsigned)p.panels), dim3(THREADS), p.lds, s, A, B, out, M, N,
                       K, groups, lda, ldb, ldo, bg, p.pg, p.pn, parts, e);
}

template <typename T>
void panel_gemm(const T* A, const T* B, T* out, long M, int N, int K, int groups, long lda, long ldb, long ldo, long bg, const Epilogue& e,
                const PanelPlan& p, hipStream_t s) {
    switch (p.ks) {
        case 3: return launch_panel<T, 0, 3>(A, B, out, M, N, K, groups, lda, ldb, ldo, bg, e, p, s);
        case 6: return launch_panel<T, 3, 6>(A, B, out, M, N, K, groups, lda, ldb, ldo, bg, e, p, s);
        case 9: return launch_panel<T, 6, 9>(A, B, out, M, N, K, groups, lda, ldb, ldo, bg, e, p, s);
        case 13: return launch_panel<T, 9, 13>(A, B, out, M, N, K, groups, lda, ldb, ldo, bg, e, p, s);
        default: return launch_panel<T, 13, 17>(A, B, out, M, N, K, groups, lda, ldb, ldo, bg, e, p, s);
    }
}

// ---- few rows: k split over the waves ----------------------------------------------------------------------------------------------
// A single row, or a few hundred: too few tiles of the kernels above for 256 CUs, and what counts is how soon the weight arrives.  A workgroup
// takes 32 rows x 32 columns; its 8 waves take every eighth batch of four k steps (128 bytes of a row), two batches in flight, each for
// itself: whole 128-byte runs, eight lanes to a row, turned into the operands' order (one row per lane) through LDS of the wave's own.  (Fetched
// in the operands' order every lane is a request of its own: 11.6 against 7.9 us for 336 x 1296 -> 324 in bfloat16.)  The partial tiles are added through
// LDS in wave order, then the epilogue runs over whole row pieces, whose bias and residual were fetched before anything else: a
// dependent trip to memory costs as much as the whole product.  One launch, no workspace.
// Bound by latency: one row 1024 -> 4096 bfloat16 6.1 us (8.4 MB), 336 rows 1296 -> 324 8.5 us.
template <typename T>
__global__ __launch_bounds__(512) void few_rows_kernel(const T* __restrict__ X, const T* __restrict__ W, T* __restrict__ out, long M, int N, int K,
                                                       long ldx, long ldw, long ldo, long wg, Epilogue e) {
    constexpr int E = Num<T>::E, LD = 36, U = 4, WAVES = 8, LPR = 32 / E;
    __shared__ u32x4 turn[WAVES][2][32 * 8];              // 64 KB; afterwards the partial tiles
    const int g = blockIdx.z, n0 = blockIdx.x * 32, C = (int)gridDim.z * N;
    const long m0 = (long)blockIdx.y * 32;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r32 = lane & 31, half = lane >> 5, r8 = lane >> 3, p8 = lane & 7;
    const T *wrow[U], *xrow[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        wrow[u] = W + g * wg + (long)min(n0 + u * 8 + r8, N - 1) * ldw;
        xrow[u] = X + min(m0 + u * 8 + r8, M - 1) * ldx + (long)g * K;
    }
    const int batches = (K + 2 * U * E - 1) / (2 * U * E), rounds = (batches + WAVES - 1) / WAVES;
    u32x4 w[3][U], x[3][U];
    auto fetch = [&](int round, u32x4 (&wb)[U], u32x4 (&xb)[U]) __attribute__((always_inline)) {       // behind K: the row's end
        const int k = min(((round * WAVES + wave) * 8 + p8) * E, K - E);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            wb[u] = load16(wrow[u] + k);
            xb[u] = load16(xrow[u] + k);
        }
    };
    fetch(0, w[0], x[0]);
    // this thread's piece of the result
    const int prow = threadIdx.x / LPR % 32, pc = threadIdx.x % LPR * E, col = min(g * N + n0 + pc, C - 1), valid = min(E, N - n0 - pc);
    const bool mine = threadIdx.x < 32 * LPR && m0 + prow < M && valid > 0;
    const OutRow<T> orow(e, out, ldo, min(m0 + prow, M - 1), C);
    u32x4 add;
    float bias[E];
    if (e.residual && C >= E) add = orow.fetch(col);
    load_bias<T>(bias, e, col, C);
    fetch(1, w[1], x[1]);
    f32x16 acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0.f;
    auto multiply = [&](int round, u32x4 (&wb)[U], u32x4 (&xb)[U]) __attribute__((always_inline)) {
        const int k0 = (round * WAVES + wave) * U * 2 * E;
        if (k0 + U * 2 * E > K) {              // zeros behind K
#pragma unroll
            for (int u = 0; u < U; ++u) {
                wb[u] = tail_fixed<T>(wb[u], k0 + p8 * E, K);
                xb[u] = tail_fixed<T>(xb[u], k0 + p8 * E, K);
            }
        }
        u32x4 *wt = turn[wave][0], *xt = turn[wave][1];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            wt[(u * 8 + r8) * 8 + swizzle(u * 8 + r8, p8)] = wb[u];
            xt[(u * 8 + r8) * 8 + swizzle(u * 8 + r8, p8)] = xb[u];
        }
        wave_sync();
#pragma unroll
        for (int u = 0; u < U; ++u)
            acc = Num<T>::mma(wt[r32 * 8 + swizzle(r32, u * 2 + half)], xt[r32 * 8 + swizzle(r32, u * 2 + half)], acc);
        wave_sync();
    };
    for (int r = 0;;) {
        fetch(r + 2, w[2], x[2]);
        multiply(r, w[0], x[0]);
        if (++r == rounds) break;
        fetch(r + 2, w[0], x[0]);
        multiply(r, w[1], x[1]);
        if (++r == rounds) break;
        fetch(r + 2, w[1], x[1]);
        multiply(r, w[2], x[2]);
        if (++r == rounds) break;
    }
    __syncthreads();
    float(*part)[32][LD] = reinterpret_cast<float(*)[32][LD]>(&turn[0][0][0]);
    static_assert(sizeof(float) * WAVES * 32 * LD <= sizeof(turn), "the partial tiles lie in the waves' LDS");
    put_strip<1>(&part[wave][0][0], LD, lane, [&](int, int r) { return acc[r]; });
    __syncthreads();
    if (!mine) return;
    float f[E];
#pragma unroll
    for (int q = 0; q < E; q += 4) {
        float4 t = *reinterpret_cast<const float4*>(&part[0][prow][pc + q]);
#pragma unroll
        for (int v = 1; v < WAVES; ++v) {
            const float4 o = *reinterpret_cast<const float4*>(&part[v][prow][pc + q]);
            t.x += o.x, t.y += o.y, t.z += o.z, t.w += o.w;
        }
        f[q] = t.x + bias[q], f[q + 1] = t.y + bias[q + 1], f[q + 2] = t.z + bias[q + 2], f[q + 3] = t.w + bias[q + 3];
    }
    finish_piece<T>(f, add, orow, g * N + n0 + pc, valid, e.act, e.slope);
}

template <typename T>
void launch_few_rows(const T* A, const T* B, T* out, long M, int N, int K, int groups, long lda, long ldb, long ldo, long bg, const Epilogue& e,
                     hipStream_t s) {
    const dim3 grid((unsigned)cdiv(N, 32), (unsigned)cdiv64(M, 32), (unsigned)groups);
    hipLaunchKernelGGL(few_rows_kernel<T>, grid, dim3(512), 0, s, A, B, out, M, N, K, lda, ldb, ldo, bg, e);
}

// ---- plans ---------------------------------------------------------------------------------------------------------------------------
size_t elem_bytes(int dtype) { return dtype == 0 ? 4 : 2; }
size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// The panel kernel from 65536 rows on: then each of its 2048 waves has 32 rows.  Panel against tiles, us: 65536 rows bfloat16 132 -> 132 15.5 / 27.8,
// 264 -> 528 48 / 69; 172032 rows 132 -> 528 91 / 164, float32 249 / 330; fewer rows leave waves idle, 21504 rows 132 -> 264 17.4 / 16.0, float32
// 132 -> 132 34 / 20.  Wide ones: 65536 rows 264 -> 2112 128 / 211, 132 -> 4096 169 / 380, float32 132 -> 4096 868 / 857; the panels of long rows are
// narrow, each reads all of x again: 264 -> 4096 421 / 390, 172032 rows 1119 / 982 (not worth a rule of its own).  Rows of more than 17 k steps leave no registers for the next rows: 172032 rows 384 -> 384 132 / 117, 400 -> 1600 593 / 484.
constexpr long kPanelRows = 65536;
// k split over the waves where fewer than 64 tiles of 64 x 64 would be there, and up to 160 with rows of 4 KB and more.  Split against tiles, us:
// bfloat16 336 rows 528 -> 528 5.9 / 7.0, 1000 rows 132 -> 132 5.0 / 6.2, 256 rows 2048 -> 2048 14.0 / 19.7; 700 rows 528 -> 528 10.9 / 7.3,
// 512 rows 2048 -> 2048 25.5 / 20.3.  32 rows fill no tile, whatever their number of columns: 8192 -> 2048 15 / 66.
bool few_rows(long M, int N, int K, int groups, size_t S) {
    const long tiles = cdiv64(M, 64) * cdiv(N, 64) * groups;
    return K >= (int)(16 / S) && (M <= 32 || tiles < 64 || (tiles <= 160 && (long)K * (long)S >= 4096));
}

// Rounds of the CUs that square tiles of three sizes need, in units of a 64 x 64 tile's matrix work; what a CU holds at a time is one 256, two
// 128 or four 64 tiles.  Weighted by what they reach when they fill the card (16 bits, 16384 x 2048 -> 8192 in bfloat16: 1030, 900, 620 TFLOP/s;
// float32, 4096^3: 140, 130, 119) and, in float32, by the k that the first stage and the epilogue cost beside K (65536 x 264 -> 1056 448, 391,
// 379 us; 172032 x 264 -> 132 279, 242, 184; 65536 x 528 -> 528 453, 379, 362; in 16 bits the sizes stay within 5 % of the best without it).
int tile_size(long M, int N, int K, int groups, bool dma, size_t S) {
    const auto rounds = [&](long t, long at_a_time) { return (cdiv64(M, t) * cdiv64(N, t) * groups + 256 * at_a_time - 1) / (256 * at_a_time); };
    const bool f32 = S == 4;
    const double c256 = 16.0 * rounds(256, 1) * (f32 ? (K + 113) / 1.40 : K / 1.03), c128 = 8.0 * rounds(128, 2) * (f32 ? (K + 72) / 1.30 : K / 0.9),
                 c64 = 4.0 * rounds(64, 4) * (f32 ? (K + 55) / 1.19 : K / 0.62);
    if (dma && c256 <= c128 && c256 <= c64) return 256;
    return c128 <= c64 ? 128 : 64;
}

template <typename T>
int rows_gemm(const T* A, const T* B, T* out, long M, int N, int K, int groups, long lda, long ldb, long ldo, long bg, const Epilogue& e,
               hipStream_t s) {
    constexpr size_t S = sizeof(T);
    const bool dma = on16(A, lda, S) && on16(B, ldb, S) && (long)K * S % 16 == 0 && bg * (long)S % 16 == 0;
    const PanelPlan p = plan_panel(N, K, groups, S);
    if (p.ks && M >= kPanelRows) {
        panel_gemm<T>(A, B, out, M, N, K, groups, lda, ldb, ldo, bg, e, p, s);
        return 0;
    }
    if (few_rows(M, N, K, groups, S)) {
        launch_few_rows<T>(A, B, out, M, N, K, groups, lda, ldb, ldo, bg, e, s);
        return 0;
    }
    const int tile = tile_size(M, N, K, groups, dma, S);
    if (tile == 256) return launch_rows_gemm<T, 256, 256, 2, 4, 1>(A, B, out, M, N, K, groups, lda, ldb, ldo, bg, e, s);
    if (dma && tile == 128) return launch_rows_gemm<T, 128, 128, 2, 2, 1>(A, B, out, M, N, K, groups, lda, ldb, ldo, bg, e, s);
    if (dma) return launch_rows_gemm<T, 64, 64, 2, 2, 1>(A, B, out, M, N, K, groups, lda, ldb, ldo, bg, e, s);
    if (tile == 128) return launch_rows_gemm<T, 128, 128, 2, 2, 0>(A, B, out, M, N, K, groups, lda, ldb, ldo, bg, e, s);
    return launch_rows_gemm<T, 64, 64, 2, 2, 0>(A, B, out, M, N, K, groups, lda, ldb, ldo, bg, e, s);
}

// The weight gradient's tiles and split: 128-column tiles, 64 where a side is that small, 256 (16 bits, aligned rows) where those alone give
// most of the CUs a tile; p in as many parts as give every CU two workgroups (one of the 256 tiles), each at least four stages long.
struct ColsPlan {
    int bc, nt, kt, splits;
    long rows_per_split;
};
ColsPlan plan_cols(int64_t P, int N, int K, int groups, int dtype, bool dma) {
    ColsPlan p;
    p.bc = N > 64 && K > 64 ? 128 : 64;
    if (dtype != 0 && dma && cdiv64(N, 256) * cdiv64(K, 256) * groups >= 192) p.bc = 256;
    p.nt = cdiv(N, p.bc);
    p.kt = cdiv(K, p.bc);
    const int64_t tiles = (int64_t)p.nt * p.kt * groups, kp = dtype == 0 ? 32 : 64;
    int64_t splits = (p.bc == 256 ? 256 : 512) / tiles, most = cdiv64(P, 4 * kp);      // rounded down: one workgroup too many is a second round
    if (splits < 1) splits = 1;
    if (splits > most) splits = most;
    if (splits > 512) splits = 512;
    p.rows_per_split = cdiv64(cdiv64(P, splits), kp) * kp;
    p.splits = (int)cdiv64(P, p.rows_per_split);
    return p;
}

template <typename T, int BC, int WR, int WC, int DMA>
void launch_cols_gemm(const T* G, const T* X, T* out, float* partial, long P, int N, int K, int groups, long ldg, long ldx, const ColsPlan& p,
                      hipStream_t s) {
    constexpr int KP = sizeof(T) == 4 ? 32 : 64;
    const size_t lds = (size_t)2 * 2 * KP * BC * sizeof(T);
    auto* kernel = &cols_gemm_kernel<T, BC, WR, WC, DMA>;
    if (lds > 65536) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    const dim3 grid((unsigned)(cdiv64((int64_t)p.nt * p.kt, kXcds) * kXcds), (unsigned)groups, (unsigned)p.splits);
    hipLaunchKernelGGL((cols_gemm_kernel<T, BC, WR, WC, DMA>), grid, dim3(64 * WR * WC), lds, s, G, X, out, p.splits > 1 ? partial : nullptr, P, N,
                       K, ldg, ldx, p.nt, p.kt, p.rows_per_split);
}

SplitSum split_sum(const float* partial, void* out, int out_f32, long n, int splits) {
    const int parts = splits >= 64 ? 16 : (splits >= 16 && n < 65536 ? 4 : 1);
    return SplitSum{partial, out, out_f32, splits, parts, n, (unsigned)cdiv64(n, 256 / parts)};
}

// `padded`: G's rows are followed by zeros up to whole pieces.  Returns the split
template <typename T>
int cols_gemm(const T* G, const T* X, T* out, float* partial, long P, int N, int K, int groups, long ldg, long ldx, bool padded, int dtype,
              hipStream_t s) {
    constexpr size_t S = sizeof(T);
    const bool dma = on16(G, ldg, S) && on16(X, ldx, S) && (long)K * S % 16 == 0 && ((long)N * S % 16 == 0 || (padded && groups == 1));
    const ColsPlan p = plan_cols(P, N, K, groups, dtype, dma);
    if constexpr (S == 2)
        if (p.bc == 256) {
            launch_cols_gemm<T, 256, 2, 4, 1>(G, X, out, partial, P, N, K, groups, ldg, ldx, p, s);
            return p.splits;
        }
    if (p.bc == 128 && dma) launch_cols_gemm<T, 128, 2, 2, 1>(G, X, out, partial, P, N, K, groups, ldg, ldx, p, s);
    else if (p.bc == 128) launch_cols_gemm<T, 128, 2, 2, 0>(G, X, out, partial, P, N, K, groups, ldg, ldx, p, s);
    else if (dma) launch_cols_gemm<T, 64, 2, 2, 1>(G, X, out, partial, P, N, K, groups, ldg, ldx, p, s);
    else launch_cols_gemm<T, 64, 2, 2, 0>(G, X, out, partial, P, N, K, groups, ldg, ldx, p, s);
    return p.splits;
}

// Workspace of a backward call: [dz][transposed weight][column sums][split blocks]
struct BwdPlan {
    int64_t ld_dz;
    int ldt, lanes, col_blocks, row_blocks;
    int64_t rows_per_block;
    size_t dz, wt, sums, split, total;
};
BwdPlan plan_bwd(int64_t P, int N, int K, int groups, int dtype, int act, bool want_gx, bool want_gw, bool want_gb) {
    BwdPlan b{};
    const size_t S = elem_bytes(dtype);
    const int E = dtype == 0 ? 4 : 8;
    const int64_t C = (int64_t)groups * N;
    b.ld_dz = cdiv64(C, E) * E;
    b.ldt = cdiv(N, E) * E;
    // lanes per row: the division of the row's pieces (at least 16 together, 256 bytes) that leaves the fewest of 256 threads idle
    const int64_t pieces = b.ld_dz / E;
    int64_t best = 0;
    for (int64_t cb = cdiv64(pieces, 256); cb == 1 || (cb <= cdiv64(pieces, 256) + 16 && cdiv64(pieces, cb) >= 16); ++cb) {
        const int64_t lanes = cdiv64(pieces, cb), used = 256 / lanes * pieces * 1000 / cb;
        if (used > best + best / 50) best = used, b.col_blocks = (int)cb, b.lanes = (int)lanes;
    }
    const int rows = 256 / b.lanes;                       // rows a workgroup holds at a time; at least 8 of them each, about 1024 workgroups
    int64_t blocks = cdiv64(1024, b.col_blocks), most = cdiv64(P, 8 * rows);
    if (blocks > most) blocks = most;
    b.rows_per_block = cdiv64(P, blocks);
    b.row_blocks = (int)cdiv64(P, b.rows_per_block);
    b.dz = act != kActNone && (want_gx || want_gw) ? align256((size_t)P * b.ld_dz * S) : 0;
    b.wt = want_gx ? align256((size_t)groups * K * b.ldt * S) : 0;
    b.sums = want_gb ? align256((size_t)b.row_blocks * C * 4) : 0;
    if (want_gw) {           // room for either split: which tiles it is depends on the rows' alignment as well
        const int a = plan_cols(P, N, K, groups, dtype, false).splits, c = plan_cols(P, N, K, groups, dtype, true).splits, splits = a > c ? a : c;
        b.split = splits > 1 ? (size_t)splits * groups * N * K * 4 : 0;
    }
    b.total = b.dz + b.wt + b.sums + b.split;
    return b;
}

template <typename T>
int launch_fwd(const T* x, const T* w, T* y, int64_t P, int N, int K, int groups, int64_t ldx, int64_t ldy, const Epilogue& e, hipStream_t s) {
    if (int r = rows_gemm<T>(x, w, y, P, N, K, groups, ldx, K, ldy, (long)N * K, e, s)) return r;
    return check_launch("linear_act_fwd");
}

template <typename T>
int launch_bwd(const T* gy, const T* x, const T* w, const void* saved, int kind, T* gx, T* gw, void* gb, int gb_f32, char* ws, int64_t P, int N,
               int K, int groups, int64_t ldg, int64_t ldx, int dtype, int act, float slope, hipStream_t s) {
    const BwdPlan b = plan_bwd(P, N, K, groups, dtype, act, gx != nullptr, gw != nullptr, gb != nullptr);
    const int64_t C = (int64_t)groups * N;
    T* dz = b.dz ? reinterpret_cast<T*>(ws) : nullptr;
    T* wt = reinterpret_cast<T*>(ws + b.dz);
    float* sums = gb ? reinterpret_cast<float*>(ws + b.dz + b.wt) : nullptr;
    float* split = reinterpret_cast<float*>(ws + b.dz + b.wt + b.sums);
    const unsigned act_blocks = dz || sums ? (unsigned)b.col_blocks * b.row_blocks : 0;
    const unsigned wt_blocks = gx ? (unsigned)cdiv(b.ldt, 64) * cdiv(K, 64) * groups : 0;
    if (act_blocks + wt_blocks) {
        auto* kernel = kind == 0 ? &act_grad_kernel<T, 0> : (kind == 1 ? &act_grad_kernel<T, 1> : &act_grad_kernel<T, 2>);
        hipLaunchKernelGGL(kernel, dim3(act_blocks + wt_blocks), dim3(256), 0, s, gy, saved, dz, sums, (long)P, (long)C, (long)ldg, (long)b.ld_dz,
                           b.lanes, (long)b.rows_per_block, act, slope, b.col_blocks, act_blocks, w, wt, N, K, b.ldt);
    }
    const bool padded = dz != nullptr;
    if (padded) {
        gy = dz;
        ldg = b.ld_dz;
    }
    if (gx) {
        const Epilogue none{};
        // the zeros behind N in dz and in wt's rows are multiplied along: whole pieces
        if (int r = rows_gemm<T>(gy, wt, gx, P, K, padded && groups == 1 ? b.ldt : N, groups, ldg, b.ldt, (long)groups * K, (long)K * b.ldt, none, s))
            return r;
    }
    const int splits = gw ? cols_gemm<T>(gy, x, gw, split, P, N, K, groups, ldg, ldx, padded, dtype, s) : 1;
    SplitSum first{}, second{};
    first.parts = second.parts = 1;
    if (gb) first = split_sum(sums, gb, gb_f32, C, b.row_blocks);
    if (splits > 1) second = split_sum(split, gw, 0, (long)groups * N * K, splits);
    if (first.blocks + second.blocks)
        hipLaunchKernelGGL(split_sum_kernel<T>, dim3(first.blocks + second.blocks), dim3(256), 0, s, first, second);
    return check_launch("linear_act_bwd");
}

int check_sizes(const char* who, int64_t P, int N, int K, int groups, int dtype, int act) {
    NEXTOU_REQUIRE(P > 0 && P <= (1ll << 36) && N > 0 && K > 0 && groups > 0 && groups <= 65535 && (int64_t)groups * N <= (1ll << 21) &&
                       (int64_t)groups * K <= (1ll << 21) && cdiv64(P, 64) * cdiv(N > K ? N : K, 64) < (1ll << 31),
                   "%s: bad sizes (P %lld, N %d, K %d, groups %d)", who, (long long)P, N, K, groups);
    // Rows narrower than a piece go through 64-row tiles however many there are; a launch takes fewer than 2^32 threads
    const int E = dtype == 0 ? 4 : 8;
    NEXTOU_REQUIRE((N >= E && K >= E) || cdiv64(P, 64) * cdiv(N > K ? N : K, 64) < (1ll << 24),
                   "%s: too many rows of fewer than 16 bytes (P %lld, N %d, K %d)", who, (long long)P, N, K);
    NEXTOU_REQUIRE(dtype >= 0 && dtype <= 2, "%s: dtype %d", who, dtype);
    NEXTOU_REQUIRE(act >= 0 && act <= 4, "%s: activation %d", who, act);
    return 0;
}

}  // namespace
}  // namespace nextou

using namespace nextou;

extern "C" int nextou_linear_act_fwd(const void* x, const void* w, const void* bias, const void* residual, void* y, void* pre,
                                     int64_t P, int N, int K, int groups, int64_t ldx, int64_t ldr,
                                     int64_t ldy, int dtype, int bias_f32, int act, float slope, nextou_stream_t stream) {
    if (int e = check_sizes("linear_act_fwd", P, N, K, groups, dtype, act)) return e;
    NEXTOU_REQUIRE(x && w && y, "linear_act_fwd: null pointer");
    NEXTOU_REQUIRE(ldx >= 0 && ldr >= 0 && ldy >= (int64_t)groups * N, "linear_act_fwd: bad row strides %lld, %lld, %lld", (long long)ldx,
                   (long long)ldr, (long long)ldy);
    const Epilogue e{bias, bias_f32, residual, (long)ldr, pre, act, slope};
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case 0: return launch_fwd<float>((const float*)x, (const float*)w, (float*)y, P, N, K, groups, ldx, ldy, e, s);
        case 1: return launch_fwd<bf16_t>((const bf16_t*)x, (const bf16_t*)w, (bf16_t*)y, P, N, K, groups, ldx, ldy, e, s);
        default: return launch_fwd<f16_t>((const f16_t*)x, (const f16_t*)w, (f16_t*)y, P, N, K, groups, ldx, ldy, e, s);
    }
}

extern "C" int nextou_linear_act_bwd_workspace(int64_t P, int N, int K, int groups, int dtype, int act, int want_gx, int want_gw, int want_gb,
                                               size_t* bytes) {
    if (int e = check_sizes("linear_act_bwd_workspace", P, N, K, groups, dtype, act)) return e;
    NEXTOU_REQUIRE(bytes, "linear_act_bwd_workspace: null pointer");
    *bytes = plan_bwd(P, N, K, groups, dtype, act, want_gx != 0, want_gw != 0, want_gb != 0).total;
    return 0;
}

extern "C" int nextou_linear_act_bwd(const void* gy, const void* x, const void* w, const void* saved, int saved_kind, void* gx, void* gw,
                                     void* gb, void* workspace, size_t workspace_bytes, int64_t P, int N, int K, int groups, int64_t ldg,
                                     int64_t ldx, int dtype, int gb_f32, int act, float slope, nextou_stream_t stream) {
    if (int e = check_sizes("linear_act_bwd", P, N, K, groups, dtype, act)) return e;
    NEXTOU_REQUIRE(gy && x && w && (gx || gw || gb), "linear_act_bwd: null pointer");
    NEXTOU_REQUIRE(ldg >= 0 && ldx >= 0, "linear_act_bwd: bad row strides %lld, %lld", (long long)ldg, (long long)ldx);
    NEXTOU_REQUIRE((act == kActNone) == (saved_kind == 0) && saved_kind >= 0 && saved_kind <= 2 && (saved_kind == 0 || saved),
                   "linear_act_bwd: activation %d with saved tensor kind %d", act, saved_kind);
    NEXTOU_REQUIRE(saved_kind != 2 || act == kActRelu || (act == kActLeaky && slope >= 0.f),
                   "linear_act_bwd: activation %d (slope %g) cannot be undone from its output's sign", act, slope);
    size_t need = 0;
    nextou_linear_act_bwd_workspace(P, N, K, groups, dtype, act, gx != nullptr, gw != nullptr, gb != nullptr, &need);
    if (workspace_bytes < need || (need && !workspace))
        return fail(NEXTOU_ENOSPACE, "linear_act_bwd: workspace %zu < %zu bytes", workspace_bytes, need);
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case 0:
            return launch_bwd<float>((const float*)gy, (const float*)x, (const float*)w, saved, saved_kind, (float*)gx, (float*)gw, gb, gb_f32,
                                     (char*)workspace, P, N, K, groups, ldg, ldx, dtype, act, slope, s);
        case 1:
            return launch_bwd<bf16_t>((const bf16_t*)gy, (const bf16_t*)x, (const bf16_t*)w, saved, saved_kind, (bf16_t*)gx, (bf16_t*)gw, gb,
                                      gb_f32, (char*)workspace, P, N, K, groups, ldg, ldx, dtype, act, slope, s);
        default:
            return launch_bwd<f16_t>((const f16_t*)gy, (const f16_t*)x, (const f16_t*)w, saved, saved_kind, (f16_t*)gx, (f16_t*)gw, gb, gb_f32,
                                     (char*)workspace, P, N, K, groups, ldg, ldx, dtype, act, slope, s);
    }
}
