// K10 — point-wise products with their epilogue, forward and backward (gfx950): float32, bfloat16 and float16 rows of any width.
//
//   z[p, gN+n] = sum_k x[p, gK+k] w[gN+n, k] + b[gN+n]          y = act(z) + residual
//   dz = gy act'(z)     dx[p, gK+k] = sum_n dz[p, gN+n] w[gN+n, k]     dw[gN+n, k] = sum_p dz[p, gN+n] x[p, gK+k]     db = sum_p dz
//
// Sums are held in float32; y, dz (16-bit types only: the matrix units read 16-bit operands) and the gradients are rounded once each.
#include "common.h"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace nextou {
namespace {

using bf16_t = __bf16;
using f16_t = _Float16;

enum Act { kActNone = 0, kActRelu = 1, kActLeaky = 2, kActGelu = 3, kActHardswish = 4 };

constexpr float kInvSqrt2 = 0.70710678118654752f, kInvSqrt2Pi = 0.39894228040143268f;

__device__ __forceinline__ float act_value(float z, int act, float slope) {
    switch (act) {
        case kActRelu: return z <= 0.f ? 0.f : z;              // (NaN stays NaN)
        case kActLeaky: return z > 0.f ? z : z * slope;
        case kActGelu: return z * (0.5f * erfcf(-z * kInvSqrt2));
        case kActHardswish: return z * fminf(fmaxf(z + 3.f, 0.f), 6.f) / 6.f;
        default: return z;
    }
}

__device__ __forceinline__ float act_slope(float z, int act, float slope) {
    switch (act) {
        case kActRelu: return z <= 0.f ? 0.f : 1.f;
        case kActLeaky: return z > 0.f ? 1.f : slope;
        case kActGelu: {
            const float c = fminf(fmaxf(z, -40.f), 40.f);      // beyond that z phi(z) is 0 and must not become inf * 0
            return fmaf(c * kInvSqrt2Pi, expf(-0.5f * c * c), 0.5f * erfcf(-c * kInvSqrt2));
        }
        case kActHardswish: return z <= -3.f ? 0.f : (z >= 3.f ? 1.f : (2.f * z + 3.f) / 6.f);
        default: return 1.f;
    }
}

// What the backward needs of z: float32 for float32 rows, float16 for BOTH 16-bit types (the derivative saturates far inside float16's
// range, and float16's 11 bits keep the saved value's rounding out of the gradients).  A positive z never becomes zero: the sign decides.
__device__ __forceinline__ f16_t pre_half(float z) {
    const float c = z > 65504.f ? 65504.f : (z < -65504.f ? -65504.f : z);
    f16_t h = (f16_t)c;
    if (z > 0.f && h == (f16_t)0.f) h = __builtin_bit_cast(f16_t, (unsigned short)1);
    return h;
}
template <typename T> struct PreOf { using type = f16_t; };
template <> struct PreOf<float> { using type = float; };

template <typename T> __device__ __forceinline__ void store_pre(typename PreOf<T>::type* p, float z) { *p = pre_half(z); }
template <> __device__ __forceinline__ void store_pre<float>(float* p, float z) { *p = z; }

// ---- a plain tiled product, right for every shape and stride ------------------------------------------------------------------------
// C[m, n] = sum_k A[m am + k ak] B[n bn + k bk]
struct Epilogue {
    const void* bias;
    int bias_f32;
    const void* residual;
    long ldr;
    void* pre;             // dense rows of groups * N
    int act;
    float slope;
};

template <typename T>
__global__ __launch_bounds__(256) void plain_gemm_kernel(const T* __restrict__ A, const T* __restrict__ B, T* __restrict__ C, long M,
                                                         int N, long K, long am, long ak, long bn, long bk, long ldc, long ag, long bg,
                                                         long cg, Epilogue e) {
    __shared__ float As[16][65], Bs[16][65];
    const int g = blockIdx.z;
    const long m0 = (long)blockIdx.x * 64;
    const int n0 = blockIdx.y * 64;
    A += g * ag;
    B += g * bg;
    C += g * cg;
    float acc[4][4] = {};
    const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;
    for (long k0 = 0; k0 < K; k0 += 16) {
        for (int i = threadIdx.x; i < 1024; i += 256) {
            const int kk = i / 64, r = i % 64;
            As[kk][r] = (m0 + r < M && k0 + kk < K) ? (float)A[(m0 + r) * am + (k0 + kk) * ak] : 0.f;
            Bs[kk][r] = (n0 + r < N && k0 + kk < K) ? (float)B[(n0 + r) * bn + (k0 + kk) * bk] : 0.f;
        }
        __syncthreads();
        for (int kk = 0; kk < 16; ++kk)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(As[kk][tm * 4 + i], Bs[kk][tn * 4 + j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i) {
        const long m = m0 + tm * 4 + i;
        if (m >= M) continue;
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + tn * 4 + j;
            if (n >= N) continue;
            float z = acc[i][j];
            const long col = (long)g * N + n;
            if (e.bias) z += e.bias_f32 ? static_cast<const float*>(e.bias)[col] : (float)static_cast<const T*>(e.bias)[col];
            if (e.pre) store_pre<T>(static_cast<typename PreOf<T>::type*>(e.pre) + m * (long)(gridDim.z) * N + col, z);
            z = act_value(z, e.act, e.slope);
            if (e.residual) z += (float)static_cast<const T*>(e.residual)[m * e.ldr + col];
            C[m * ldc + n] = (T)z;
        }
    }
}

// dz = gy * act'(saved), dense rows; saved is z (kind 1) or, for the activations whose sign is z's, y itself (kind 2)
template <typename T>
__global__ __launch_bounds__(256) void act_grad_kernel(const T* __restrict__ gy, const void* __restrict__ saved, T* __restrict__ dz, long P,
                                                       long C, long ldg, int kind, int act, float slope) {
    const long total = P * C;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long p = i / C, c = i % C;
        const float s = kind == 2 ? (float)static_cast<const T*>(saved)[i] : (float)static_cast<const typename PreOf<T>::type*>(saved)[i];
        dz[i] = (T)((float)gy[p * ldg + c] * act_slope(s, act, slope));
    }
}

template <typename T>
__global__ __launch_bounds__(256) void column_sum_kernel(const T* __restrict__ gy, const void* __restrict__ saved, void* __restrict__ gb,
                                                         int gb_f32, long P, long C, long ldg, int kind, int act, float slope) {
    __shared__ float part[4][64];
    const long c = (long)blockIdx.x * 64 + (threadIdx.x & 63);
    const int w = threadIdx.x >> 6;
    float acc = 0.f;
    if (c < C)
        for (long p = w; p < P; p += 4) {
            float v = (float)gy[p * ldg + c];
            if (kind == 1) v *= act_slope((float)static_cast<const typename PreOf<T>::type*>(saved)[p * C + c], act, slope);
            if (kind == 2) v *= act_slope((float)static_cast<const T*>(saved)[p * C + c], act, slope);
            acc += v;
        }
    part[w][threadIdx.x & 63] = acc;
    __syncthreads();
    if (w == 0 && c < C) {
        const float t = (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
        if (gb_f32) static_cast<float*>(gb)[c] = t;
        else static_cast<T*>(gb)[c] = (T)t;
    }
}

size_t elem_bytes(int dtype) { return dtype == 0 ? 4 : 2; }

template <typename T>
int launch_fwd(const T* x, const T* w, T* y, int64_t P, int N, int K, int groups, int64_t ldx, int64_t ldy, const Epilogue& e,
               hipStream_t s) {
    const dim3 grid((unsigned)cdiv64(P, 64), (unsigned)cdiv(N, 64), (unsigned)groups);
    hipLaunchKernelGGL(plain_gemm_kernel<T>, grid, dim3(256), 0, s, x, w, y, (long)P, N, (long)K, (long)ldx, 1l, (long)K, 1l, (long)ldy,
                       (long)K, (long)N * K, (long)N, e);
    return check_launch("linear_act_fwd");
}

template <typename T>
int launch_bwd(const T* gy, const T* x, const T* w, const void* saved, int kind, T* gx, T* gw, void* gb, int gb_f32, T* dz, int64_t P,
               int N, int K, int groups, int64_t ldg, int64_t ldx, int act, float slope, hipStream_t s) {
    const long C = (long)groups * N;
    const Epilogue none{};
    if (gb)
        hipLaunchKernelGGL(column_sum_kernel<T>, dim3((unsigned)cdiv64(C, 64)), dim3(256), 0, s, gy, saved, gb, gb_f32, (long)P, C, (long)ldg,
                           kind, act, slope);
    if (kind && (gx || gw)) {
        const int64_t blocks = cdiv64(P * C, 256);
        hipLaunchKernelGGL(act_grad_kernel<T>, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, s, gy, saved, dz, (long)P, C,
                           (long)ldg, kind, act, slope);
        gy = dz;
        ldg = C;
    }
    if (gx)
        hipLaunchKernelGGL(plain_gemm_kernel<T>, dim3((unsigned)cdiv64(P, 64), (unsigned)cdiv(K, 64), (unsigned)groups), dim3(256), 0, s, gy,
                           w, gx, (long)P, K, (long)N, (long)ldg, 1l, 1l, (long)K, (long)groups * K, (long)N, (long)N * K, (long)K, none);
    if (gw)
        hipLaunchKernelGGL(plain_gemm_kernel<T>, dim3((unsigned)cdiv(N, 64), (unsigned)cdiv(K, 64), (unsigned)groups), dim3(256), 0, s, gy, x,
                           gw, (long)N, K, (long)P, 1l, (long)ldg, 1l, (long)ldx, (long)K, (long)N, (long)K, (long)N * K, none);
    return check_launch("linear_act_bwd");
}

int check_sizes(const char* who, int64_t P, int N, int K, int groups, int dtype, int act) {
    NEXTOU_REQUIRE(P > 0 && P <= (1ll << 36) && N > 0 && K > 0 && groups > 0 && groups <= 65535 && (int64_t)groups * N <= (1ll << 22) &&
                       (int64_t)groups * K <= (1ll << 22),
                   "%s: bad sizes (P %lld, N %d, K %d, groups %d)", who, (long long)P, N, K, groups);
    NEXTOU_REQUIRE(dtype >= 0 && dtype <= 2, "%s: dtype %d", who, dtype);
    NEXTOU_REQUIRE(act >= 0 && act <= 4, "%s: activation %d", who, act);
    return 0;
}

}  // namespace
}  // namespace nextou

using namespace nextou;

extern "C" int nextou_linear_act_fwd_workspace(int64_t P, int N, int K, int groups, int dtype, size_t* bytes) {
    if (int e = check_sizes("linear_act_fwd_workspace", P, N, K, groups, dtype, 0)) return e;
    NEXTOU_REQUIRE(bytes, "linear_act_fwd_workspace: null pointer");
    *bytes = 0;
    return 0;
}

extern "C" int nextou_linear_act_fwd(const void* x, const void* w, const void* bias, const void* residual, void* y, void* pre,
                                     void* workspace, size_t workspace_bytes, int64_t P, int N, int K, int groups, int64_t ldx, int64_t ldr,
                                     int64_t ldy, int dtype, int bias_f32, int act, float slope, nextou_stream_t stream) {
    if (int e = check_sizes("linear_act_fwd", P, N, K, groups, dtype, act)) return e;
    NEXTOU_REQUIRE(x && w && y, "linear_act_fwd: null pointer");
    NEXTOU_REQUIRE(ldx >= 0 && ldr >= 0 && ldy >= (int64_t)groups * N, "linear_act_fwd: bad row strides %lld, %lld, %lld", (long long)ldx,
                   (long long)ldr, (long long)ldy);
    size_t need = 0;
    nextou_linear_act_fwd_workspace(P, N, K, groups, dtype, &need);
    if (workspace_bytes < need) return fail(NEXTOU_ENOSPACE, "linear_act_fwd: workspace %zu < %zu bytes", workspace_bytes, need);
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
    *bytes = act != kActNone && (want_gx || want_gw) ? (size_t)P * groups * N * elem_bytes(dtype) : 0;
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
                                     (float*)workspace, P, N, K, groups, ldg, ldx, act, slope, s);
        case 1:
            return launch_bwd<bf16_t>((const bf16_t*)gy, (const bf16_t*)x, (const bf16_t*)w, saved, saved_kind, (bf16_t*)gx, (bf16_t*)gw, gb,
                                      gb_f32, (bf16_t*)workspace, P, N, K, groups, ldg, ldx, act, slope, s);
        default:
            return launch_bwd<f16_t>((const f16_t*)gy, (const f16_t*)x, (const f16_t*)w, saved, saved_kind, (f16_t*)gx, (f16_t*)gw, gb, gb_f32,
                                     (f16_t*)workspace, P, N, K, groups, ldg, ldx, act, slope, s);
    }
}
