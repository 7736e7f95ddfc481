// K11 — the global norm of a list of gradients, and the clip (gfx950).
//
//   norm = (sum |g|^p)^(1/p) over every element of every tensor, p = 1, 2, or max |g| (p = inf)
//   clip: c = min(1, max_norm / (norm + 1e-6)),  g <- c g  (rounded once to the tensor's type)
//
// The step's own clip (step_glue.hip) takes float32 gradients of one parameter group on its way into SGD; this one takes any mixture of
// float32 / bfloat16 / float16 tensors, for any optimizer.  HBM-bound: every gradient is read for the norm (4 or 2 bytes an element), and
// read and written again for the scale, since the factor depends on the last element.
//
// Two launches: partial sums (float64, a fixed order: bit-reproducible), then the scale, in which every workgroup sums the (at
// most kNormGroups) partials itself instead of waiting for a third launch.  The tensors are named by a table of 16-byte rows.  Up to
// kArgRows = 224 rows ride in the launch's arguments; a longer table is written to the workspace first, by one small launch (1.5 us) for every 224
// rows (arguments again, so that a captured graph holds no host pointer): 358 tensors take 4 launches, 610 take 5.
//
// Work is cut into kChunkBytes pieces of each tensor's 16-byte-aligned span; a workgroup takes a contiguous run of pieces.  A tensor may
// start at any multiple of its element size (views into a flat bucket): the first and last 16 bytes are taken element by element, the
// rest as 16-byte accesses.
//
// Measured: 358 float32 tensors of 30.7 M values, norm 35 us, with the scale 71 us (read, read and write: 368 MB, 5.2 TB/s, the second read partly out
// of the last cache); 610 tensors of 10^9 bfloat16 and float32 values 350 us and 1.2 ms (6 GB, 5.0 TB/s).  A copy reaches 4.9.  Where the norm is
// below the limit the scale's workgroups end after their look at the factor.
#include "common.h"
#include <algorithm>
#include <new>

namespace nextou {
namespace {

constexpr int kNormThreads = 256;
constexpr int kNormGroups = 2048;        // 8 workgroups on each of the 256 CUs
constexpr int kArgRows = 224;            // 3.5 KB of launch arguments
constexpr int kChunkBytes = 16384;

// dtype in the top 2 bits of `where`; elements in the low 36 bits of `size`, the row's first piece in the upper 28
struct NormRow {
    unsigned long long where, size;
};
struct NormRows {
    NormRow r[kArgRows];
};
constexpr unsigned long long kCountMask = (1ull << 36) - 1;

using uint4v = __attribute__((ext_vector_type(4))) unsigned;

// addresses come out of the table as integers: without the address space every access would be a flat one
#define NEXTOU_GLOBAL(T, at) reinterpret_cast<__attribute__((address_space(1))) T*>(at)

__device__ __forceinline__ int find_row(const NormRow* rows, int n, unsigned piece, int* found) {
    for (int i = threadIdx.x; i < n; i += kNormThreads) {
        const unsigned b = (unsigned)(rows[i].size >> 36), e = i + 1 < n ? (unsigned)(rows[i + 1].size >> 36) : 0xffffffffu;
        if (b <= piece && piece < e) *found = i;      // every row has at least one piece: exactly one i
    }
    __syncthreads();
    return *found;
}

__device__ __forceinline__ float bf16_of(unsigned short b) { return __builtin_bit_cast(float, (unsigned)b << 16); }
__device__ __forceinline__ float f16_of(unsigned short b) { return (float)__builtin_bit_cast(_Float16, b); }

// round to nearest even; NaN stays NaN
__device__ __forceinline__ unsigned short to_bf16(float f) { return __builtin_bit_cast(unsigned short, (__bf16)f); }
__device__ __forceinline__ unsigned short to_f16(float f) { return __builtin_bit_cast(unsigned short, (_Float16)f); }

// the norm's accumulator: float64 sums, or the largest |g| as its bit pattern (a NaN's is larger than infinity's, so it wins)
template <int P> struct Acc {
    double v = 0.0;
    __device__ __forceinline__ void add(float x) {
        if constexpr (P == 2) v = fma((double)x, (double)x, v);
        else v += (double)fabsf(x);
    }
    __device__ __forceinline__ void join(const Acc& o) { v += o.v; }
    __device__ __forceinline__ double get() const { return v; }
    __device__ __forceinline__ void set(double d) { v = d; }
};
template <> struct Acc<0> {
    unsigned v = 0;
    __device__ __forceinline__ void add(float x) { v = max(v, __builtin_bit_cast(unsigned, x) & 0x7fffffffu); }
    __device__ __forceinline__ void join(const Acc& o) { v = max(v, o.v); }
    __device__ __forceinline__ double get() const { return (double)__builtin_bit_cast(float, v); }
    __device__ __forceinline__ void set(double d) { v = __builtin_bit_cast(unsigned, (float)d) & 0x7fffffffu; }
};

template <int P>
__device__ __forceinline__ double group_total(Acc<P> a) {        // fixed tree; valid in thread 0
    __shared__ double wave_part[kNormThreads / 64];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        Acc<P> o;
        o.set(__shfl_down(a.get(), off, 64));
        a.join(o);
    }
    if ((threadIdx.x & 63) == 0) wave_part[threadIdx.x >> 6] = a.get();
    __syncthreads();
    Acc<P> t;
    t.set(wave_part[0]);
#pragma unroll
    for (int w = 1; w < kNormThreads / 64; ++w) {
        Acc<P> o;
        o.set(wave_part[w]);
        t.join(o);
    }
    return t.get();
}

template <int P, int D>
__device__ __forceinline__ void add_vec(Acc<P>& a, uint4v w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned u = w[i];        // (a bit cast of the vector's element itself takes the vector's first)
        if constexpr (D == 0) a.add(__builtin_bit_cast(float, u));
        if constexpr (D == 1) {
            a.add(__builtin_bit_cast(float, u << 16));
            a.add(__builtin_bit_cast(float, u & 0xffff0000u));
        }
        if constexpr (D == 2) {
            a.add(f16_of((unsigned short)u));
            a.add(f16_of((unsigned short)(u >> 16)));
        }
    }
}

template <int D>
__device__ __forceinline__ float load_one(unsigned long long at) {
    if constexpr (D == 0) return *NEXTOU_GLOBAL(const float, at);
    else if constexpr (D == 1) return bf16_of(*NEXTOU_GLOBAL(const unsigned short, at));
    else return f16_of(*NEXTOU_GLOBAL(const unsigned short, at));
}

template <int D>
__device__ __forceinline__ void store_one(unsigned long long at, float v) {
    if constexpr (D == 0) *NEXTOU_GLOBAL(float, at) = v;
    else if constexpr (D == 1) *NEXTOU_GLOBAL(unsigned short, at) = to_bf16(v);
    else *NEXTOU_GLOBAL(unsigned short, at) = to_f16(v);
}

// Calls vec(address) for every whole 16-byte vector of [lo, hi) and one(address) for the elements before and behind them.
template <int E, typename V, typename O>
__device__ __forceinline__ void walk(unsigned long long lo, unsigned long long hi, V vec, O one) {
    const unsigned long long a = (lo + 15) & ~15ull, b = hi & ~15ull;
    if (a >= b) {                                   // no whole vector: at most 30 bytes
        const unsigned long long at = lo + (unsigned long long)threadIdx.x * E;
        if (at < hi) one(at);
        return;
    }
#pragma unroll 4
    for (unsigned long long v = a + threadIdx.x * 16ull; v < b; v += kNormThreads * 16ull) vec(v);
    const int head = (int)((a - lo) / E), tail = (int)((hi - b) / E);       // at most 7 each
    if ((int)threadIdx.x < head) one(lo + threadIdx.x * (unsigned long long)E);
    else if ((int)threadIdx.x >= 64 && (int)threadIdx.x - 64 < tail) one(b + (threadIdx.x - 64) * (unsigned long long)E);
}

// f(dtype, lo, hi) for this workgroup's run of pieces
template <typename F>
__device__ __forceinline__ void for_pieces(const NormRow* rows, int n, unsigned pieces, F f) {
    __shared__ int found;
    const unsigned from = (unsigned)((unsigned long long)pieces * blockIdx.x / gridDim.x);
    const unsigned to = (unsigned)((unsigned long long)pieces * (blockIdx.x + 1) / gridDim.x);
    if (from >= to) return;
    int r = find_row(rows, n, from, &found);
    unsigned at = from;
    while (at < to) {
        const NormRow row = rows[r];
        const int dtype = (int)(row.where >> 62);
        const unsigned long long base = row.where & ~(3ull << 62), end = base + (row.size & kCountMask) * (dtype ? 2 : 4);
        const unsigned begin = (unsigned)(row.size >> 36);
        const unsigned stop = r + 1 < n ? (unsigned)(rows[r + 1].size >> 36) : pieces;
        const unsigned upto = min(stop, to);
        unsigned long long lo = (base & ~15ull) + (unsigned long long)(at - begin) * kChunkBytes;
        unsigned long long hi = (base & ~15ull) + (unsigned long long)(upto - begin) * kChunkBytes;
        f(dtype, lo < base ? base : lo, hi > end ? end : hi);
        at = upto;
        ++r;
    }
}

template <int P>
__global__ __launch_bounds__(kNormThreads) void norm_partial_kernel(const NormRow* __restrict__ table, NormRows args, int n, unsigned pieces,
                                                                    double* __restrict__ partial) {
    const NormRow* rows = table ? table : args.r;
    Acc<P> acc;
    for_pieces(rows, n, pieces, [&](int dtype, unsigned long long lo, unsigned long long hi) {
        if (dtype == 0)
            walk<4>(lo, hi, [&](unsigned long long p) { add_vec<P, 0>(acc, *NEXTOU_GLOBAL(const uint4v, p)); }, [&](unsigned long long p) { acc.add(load_one<0>(p)); });
        else if (dtype == 1)
            walk<2>(lo, hi, [&](unsigned long long p) { add_vec<P, 1>(acc, *NEXTOU_GLOBAL(const uint4v, p)); }, [&](unsigned long long p) { acc.add(load_one<1>(p)); });
        else
            walk<2>(lo, hi, [&](unsigned long long p) { add_vec<P, 2>(acc, *NEXTOU_GLOBAL(const uint4v, p)); }, [&](unsigned long long p) { acc.add(load_one<2>(p)); });
    });
    const double t = group_total<P>(acc);
    if (threadIdx.x == 0) partial[blockIdx.x] = t;
}

// (norm, factor) from the partials, in every thread of the workgroup
template <int P>
__device__ __forceinline__ float2 norm_and_factor(const double* __restrict__ partial, int n, float max_norm) {
    __shared__ float2 both;
    Acc<P> acc;
    for (int i = threadIdx.x; i < n; i += kNormThreads) {
        Acc<P> o;
        o.set(partial[i]);
        acc.join(o);
    }
    const double t = group_total<P>(acc);
    if (threadIdx.x == 0) {
        const float norm = (float)(P == 2 ? sqrt(t) : t);
        float c = max_norm / (norm + 1e-6f);
        if (c > 1.0f) c = 1.0f;              // (a NaN norm gives a NaN factor, as torch's clamp does)
        both = make_float2(norm, c);
    }
    __syncthreads();
    return both;
}

template <int P>
__global__ __launch_bounds__(kNormThreads) void norm_finish_kernel(const double* __restrict__ partial, int n, float max_norm,
                                                                   float* __restrict__ norm_coef) {
    const float2 r = norm_and_factor<P>(partial, n, max_norm);
    if (threadIdx.x == 0) {
        norm_coef[0] = r.x;
        norm_coef[1] = r.y;
    }
}

template <int D>
__device__ __forceinline__ void scale_vec(unsigned long long p, float c) {
    uint4v w = *NEXTOU_GLOBAL(const uint4v, p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned u = w[i];
        if constexpr (D == 0) w[i] = __builtin_bit_cast(unsigned, __builtin_bit_cast(float, u) * c);
        if constexpr (D == 1) w[i] = to_bf16(__builtin_bit_cast(float, u << 16) * c) | (unsigned)to_bf16(__builtin_bit_cast(float, u & 0xffff0000u) * c) << 16;
        if constexpr (D == 2) w[i] = to_f16(f16_of((unsigned short)u) * c) | (unsigned)to_f16(f16_of((unsigned short)(u >> 16)) * c) << 16;
    }
    *NEXTOU_GLOBAL(uint4v, p) = w;
}

template <int P>
__global__ __launch_bounds__(kNormThreads) void norm_scale_kernel(const NormRow* __restrict__ table, NormRows args, int n, unsigned pieces,
                                                                  const double* __restrict__ partial, int n_partial, float max_norm,
                                                                  float* __restrict__ norm_coef) {
    const NormRow* rows = table ? table : args.r;
    const float2 r = norm_and_factor<P>(partial, n_partial, max_norm);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        norm_coef[0] = r.x;
        norm_coef[1] = r.y;
    }
    const float c = r.y;
    if (c == 1.0f) return;                // below the limit: nothing changes (the same for every workgroup)
    for_pieces(rows, n, pieces, [&](int dtype, unsigned long long lo, unsigned long long hi) {
        if (dtype == 0) walk<4>(lo, hi, [&](unsigned long long p) { scale_vec<0>(p, c); }, [&](unsigned long long p) { store_one<0>(p, load_one<0>(p) * c); });
        else if (dtype == 1) walk<2>(lo, hi, [&](unsigned long long p) { scale_vec<1>(p, c); }, [&](unsigned long long p) { store_one<1>(p, load_one<1>(p) * c); });
        else walk<2>(lo, hi, [&](unsigned long long p) { scale_vec<2>(p, c); }, [&](unsigned long long p) { store_one<2>(p, load_one<2>(p) * c); });
    });
}

__global__ __launch_bounds__(256) void norm_table_kernel(NormRow* __restrict__ dst, NormRows args, int n) {
    if ((int)threadIdx.x < n) dst[threadIdx.x] = args.r[threadIdx.x];
}

struct Plan {
    NormRows args;             // the first kArgRows rows
    const NormRow* table;      // NULL: the rows are in args
    unsigned pieces;
    int groups;
};

size_t table_bytes(int n) { return n > kArgRows ? ((size_t)n * sizeof(NormRow) + 255) / 256 * 256 : 0; }

// No two tensors of a clip may share an element: two workgroups would scale it at once.
int check_apart(const char* who, const int64_t* table_host, int n) {
    struct Span {
        unsigned long long lo, hi;
    };
    Span* spans = new (std::nothrow) Span[n];
    if (!spans) return fail(NEXTOU_ENOSPACE, "%s: no host memory for %d tensors", who, n);
    for (int i = 0; i < n; ++i) {
        const unsigned long long at = (unsigned long long)table_host[3 * i];
        spans[i] = Span{at, at + (unsigned long long)table_host[3 * i + 1] * (table_host[3 * i + 2] == 0 ? 4 : 2)};
    }
    std::sort(spans, spans + n, [](const Span& a, const Span& b) { return a.lo < b.lo; });
    bool apart = true;
    for (int i = 1; i < n && apart; ++i) apart = spans[i].lo >= spans[i - 1].hi;
    delete[] spans;
    NEXTOU_REQUIRE(apart, "%s: two of the gradients overlap in memory (the same one listed twice?)", who);
    return 0;
}

// Checks the host table and brings a long one into the workspace.  ws: [partials][table]
int make_plan(const char* who, const int64_t* table_host, int n, int p_code, bool scale, void* workspace, size_t workspace_bytes, hipStream_t s,
              Plan* plan, double* bytes) {
    NEXTOU_REQUIRE(table_host && n > 0 && n <= (1 << 24), "%s: null table or %d tensors", who, n);
    NEXTOU_REQUIRE(p_code >= 0 && p_code <= 2, "%s: norm %d is none of 0 (max), 1, 2", who, p_code);
    const size_t need = kNormGroups * sizeof(double) + table_bytes(n);
    if (!workspace || workspace_bytes < need) return fail(NEXTOU_ENOSPACE, "%s: workspace %zu < %zu bytes", who, workspace_bytes, need);
    unsigned long long pieces = 0;
    *bytes = 0;
    for (int i = 0; i < n; ++i) {          // everything is checked before anything is launched
        const unsigned long long at = (unsigned long long)table_host[3 * i];
        const int64_t count = table_host[3 * i + 1], dtype = table_host[3 * i + 2];
        const int size = dtype == 0 ? 4 : 2;
        NEXTOU_REQUIRE(dtype >= 0 && dtype <= 2 && count > 0 && count <= (int64_t)kCountMask && at && at % size == 0 && !(at >> 62),
                       "%s: tensor %d: %lld elements of type %lld at %p", who, i, (long long)count, (long long)dtype, (void*)at);
        const unsigned long long span = at % 16 + (unsigned long long)count * size;
        pieces += (span + kChunkBytes - 1) / kChunkBytes;
        NEXTOU_REQUIRE(pieces < (1ull << 28), "%s: more than 4 TB of gradients", who);
        *bytes += (double)count * size;
    }
    if (scale)
        if (int e = check_apart(who, table_host, n)) return e;
    plan->pieces = (unsigned)pieces;
    plan->groups = (int)(pieces < kNormGroups ? pieces : kNormGroups);
    plan->table = n > kArgRows ? reinterpret_cast<const NormRow*>((char*)workspace + kNormGroups * sizeof(double)) : nullptr;
    pieces = 0;
    for (int i = 0; i < n; ++i) {
        const unsigned long long at = (unsigned long long)table_host[3 * i], count = (unsigned long long)table_host[3 * i + 1];
        const int dtype = (int)table_host[3 * i + 2];
        plan->args.r[i % kArgRows] = NormRow{at | (unsigned long long)dtype << 62, count | pieces << 36};
        pieces += (at % 16 + count * (dtype == 0 ? 4 : 2) + kChunkBytes - 1) / kChunkBytes;
        if (plan->table && (i % kArgRows == kArgRows - 1 || i == n - 1))
            hipLaunchKernelGGL(norm_table_kernel, dim3(1), dim3(256), 0, s, const_cast<NormRow*>(plan->table) + i / kArgRows * kArgRows,
                               plan->args, i % kArgRows + 1);
    }
    for (int i = n; i < kArgRows; ++i) plan->args.r[i] = NormRow{0, 0};
    return 0;
}

template <int P>
void launch_partials(const Plan& plan, int n, double* partial, double bytes, hipStream_t s) {
    ProfScope prof(s, kBoundHbm, bytes, "norm_partial_kernel[T%d]", n);
    hipLaunchKernelGGL(norm_partial_kernel<P>, dim3(plan.groups), dim3(kNormThreads), 0, s, plan.table, plan.args, n, plan.pieces, partial);
}

template <int P>
void launch_norm(const Plan& plan, int n, double* partial, double bytes, float max_norm, float* norm_coef, bool scale, hipStream_t s) {
    launch_partials<P>(plan, n, partial, bytes, s);
    if (scale) {
        ProfScope prof(s, kBoundHbm, 2 * bytes, "norm_scale_kernel[T%d]", n);
        hipLaunchKernelGGL(norm_scale_kernel<P>, dim3(plan.groups), dim3(kNormThreads), 0, s, plan.table, plan.args, n, plan.pieces, partial,
                           plan.groups, max_norm, norm_coef);
    } else {
        hipLaunchKernelGGL(norm_finish_kernel<P>, dim3(1), dim3(kNormThreads), 0, s, partial, plan.groups, max_norm, norm_coef);
    }
}

int multi(const char* who, const int64_t* table_host, int n, int p_code, float max_norm, void* workspace, size_t workspace_bytes,
          float* norm_coef, bool scale, nextou_stream_t stream) {
    NEXTOU_REQUIRE(norm_coef && max_norm >= 0.f, "%s: null pointer or max_norm %g", who, max_norm);
    hipStream_t s = (hipStream_t)stream;
    Plan plan;
    double bytes;
    if (int e = make_plan(who, table_host, n, p_code, scale, workspace, workspace_bytes, s, &plan, &bytes)) return e;
    double* partial = static_cast<double*>(workspace);
    if (p_code == 0) launch_norm<0>(plan, n, partial, bytes, max_norm, norm_coef, scale, s);
    else if (p_code == 1) launch_norm<1>(plan, n, partial, bytes, max_norm, norm_coef, scale, s);
    else launch_norm<2>(plan, n, partial, bytes, max_norm, norm_coef, scale, s);
    return check_launch(who);
}

}  // namespace
}  // namespace nextou

using namespace nextou;

extern "C" int nextou_multi_norm_workspace(int n_tensors, size_t* bytes) {
    NEXTOU_REQUIRE(bytes && n_tensors > 0 && n_tensors <= (1 << 24), "multi_norm_workspace: null pointer or %d tensors", n_tensors);
    *bytes = kNormGroups * sizeof(double) + table_bytes(n_tensors);
    return 0;
}

extern "C" int nextou_multi_norm(const int64_t* table_host, int n_tensors, int norm, float max_norm, void* workspace, size_t workspace_bytes,
                                 float* norm_coef, nextou_stream_t stream) {
    return multi("multi_norm", table_host, n_tensors, norm, max_norm, workspace, workspace_bytes, norm_coef, false, stream);
}

extern "C" int nextou_multi_clip(const int64_t* table_host, int n_tensors, int norm, float max_norm, void* workspace, size_t workspace_bytes,
                                 float* norm_coef, nextou_stream_t stream) {
    return multi("multi_clip", table_host, n_tensors, norm, max_norm, workspace, workspace_bytes, norm_coef, true, stream);
}
