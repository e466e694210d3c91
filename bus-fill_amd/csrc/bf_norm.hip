// Residual addition and root-mean-square norm of rows:
//   r = x + d,  y = r / sqrt(mean(r^2) + eps) (w + offset),
// r kept in x's type, y rounded once to fp16 (the next GEMM's A) and, or instead,
// quantized to int8 per 32 values (the integer-dot GEMM's Aq, as k_quantize_q8
// does of fp16 rows: dd = amax / 127, q = round(y / dd) half away from zero, from
// the unrounded fp32 y here).
//
// Bound by memory (x, d read, r, y written, once each): a row's values stay in
// registers (LDS where rows are not of whole 16-byte pieces) between the sum of
// squares and the product.  Sums are fp32 over at most 32 values of a thread (rows in
// LDS: up to four such sums), then across lanes; where squares leave fp32's range they
// are summed again in 64 bits.
//
// Measured, fp32 residual, fp16 addend, rows of 5120: 2000 rows 26.7 us for 123 MB
// (4.6 TB/s; a copy of 2 GiB reaches 4.9); 32 rows 4.0 us in the kernel and 4.8 to 5.0 a
// call from Python, 16 rows to int8 4.7 in the kernel: load, two barriers of a workgroup's
// sums, store, and the launch.  Codes: one division a block and a product a value
// (a division a value: 0.3 us more), with a division for those near half way.
#include <atomic>

#include "bf_device.h"
#include "bf_grid.h"
#include "bf_launch.h"

namespace bf {
namespace {

constexpr int kNormMaxK = 32768;

struct NormDev {
    NormArgs a;
    int8_t* q;                                     // the three regions of Aq (NULL: none)
    float* d;
    int* s;
};

template <class T> __device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
    for (int x = 32; x; x >>= 1) v += __shfl_xor(v, x);
    return v;
}

// The sum over a workgroup of up to 16 waves, for all threads.
template <class T> __device__ __forceinline__ T group_sum(T v, T* part) {
    v = wave_sum(v);
    const int waves = (blockDim.x + 63) >> 6, wave = threadIdx.x >> 6;
    if (waves == 1) return v;
    __syncthreads();                               // part may still be read
    if ((threadIdx.x & 63) == 0) part[wave] = v;
    __syncthreads();
    T s = 0;
    for (int w = 0; w < waves; w++) s += part[w];
    return s;
}

// Squares that left fp32's range: too large, or lost where eps does not cover them.
__device__ __forceinline__ bool out_of_range(float ss, float eps) { return ss > 3e38f || (ss < 0x1p-80f && eps < 0x1p-60f); }

// Factor of r: 1 / sqrt(mean + eps), in fp32, or in 64 bits where that is needed.
struct Factor {
    float f;
    double f64;
    bool wide;
    __device__ __forceinline__ float of(float r, float w) const { return wide ? (float)((double)r * f64 * (double)w) : r * f * w; }
};

template <class V>
__device__ __forceinline__ Factor factor(float ss, int K, float eps, V values, int n, double* part) {
    Factor f{0.f, 0.0, out_of_range(ss, eps)};     // (the same in all threads)
    if (f.wide) {
        double s = 0;
        for (int i = 0; i < n; i++) s += (double)values(i) * (double)values(i);
        f.f64 = 1.0 / __builtin_sqrt(group_sum(s, part) / K + (double)eps);
    } else {
        f.f = 1.f / __builtin_sqrtf(ss / K + eps);
    }
    return f;
}

// A value's code: its quotient by the block's scale (0: all zero; not finite: codes 0), rounded.
__device__ __forceinline__ float quotient(float y, float dd) { return dd > 0.f && dd < __builtin_inff() ? y / dd : 0.f; }
__device__ __forceinline__ int code(float v) {
    return (int)__builtin_fminf(__builtin_fmaxf(__builtin_roundf(v), -127.f), 127.f);
}
// Codes of a lane's eight values.  One division a block, and one a value where one of them is next to half way between two
// codes (its product with the reciprocal is within 2^-15 of the rounded quotient, whose code counts) or where dd or its
// reciprocal is not normal.
__device__ __forceinline__ void codes(int (&q)[8], const float (&y)[8], float dd) {
    const float inv = dd >= 0x1p-125f && dd < 0x1p125f ? 1.f / dd : 0.f;
    float v[8], near = 1.f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        v[e] = y[e] * inv;
        near = __builtin_fminf(near, __builtin_fabsf(__builtin_amdgcn_fractf(v[e]) - 0.5f));
    }
    if (near < 0x1p-14f || inv == 0.f)
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = quotient(y[e], dd);
#pragma unroll
    for (int e = 0; e < 8; e++) q[e] = code(v[e]);
}

__device__ __forceinline__ float load1(const void* p, int f16, int64_t i) {
    return f16 ? (float)((const _Float16*)p)[i] : ((const float*)p)[i];
}
__device__ __forceinline__ void load8(float* o, const void* p, int f16, int64_t i) {
    if (f16) {
        const h8 v = *(const h8*)((const _Float16*)p + i);
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = (float)v[e];
    } else {
        const f4 a = *(const f4*)((const float*)p + i), b = *(const f4*)((const float*)p + i + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            o[e] = a[e];
            o[4 + e] = b[e];
        }
    }
}

// A row a workgroup, eight values a thread and turn (C turns).
template <int C>
__global__ __launch_bounds__(1024) void k_rms_norm(NormDev p) {
    __shared__ float part[16];
    __shared__ double part64[16];
    const NormArgs& a = p.a;
    const int tid = threadIdx.x, n = blockDim.x, pieces = a.K >> 3;
    const int64_t row = blockIdx.x;
    float r[C][8], ss = 0.f;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int at = tid + c * n;
        if (at < pieces) {
            load8(r[c], a.X, a.x_f16, row * a.ldx + 8 * at);
            if (a.D) {
                float d[8];
                load8(d, a.D, a.d_f16, row * a.ldd + 8 * at);
#pragma unroll
                for (int e = 0; e < 8; e++) r[c][e] += d[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) r[c][e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; e++) ss = __builtin_fmaf(r[c][e], r[c][e], ss);
    }
    ss = group_sum(ss, part);
    const Factor f = factor(ss, a.K, a.eps, [&](int i) { return r[i >> 3][i & 7]; }, 8 * C, part64);
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int at = tid + c * n;
        const bool live = at < pieces;
        float w[8], y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = 1.f;
        if (live && a.W) load8(w, a.W, a.w_f16, 8 * at);
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = f.of(r[c][e], w[e] + a.offset);
        if (live && a.R) {
            if (a.x_f16) {
                *(u4*)((_Float16*)a.R + row * a.ldr + 8 * at) =
                    f32x8_to_f16(f4{r[c][0], r[c][1], r[c][2], r[c][3]}, f4{r[c][4], r[c][5], r[c][6], r[c][7]});
            } else {
                float* to = (float*)a.R + row * a.ldr + 8 * at;
                *(f4*)to = f4{r[c][0], r[c][1], r[c][2], r[c][3]};
                *(f4*)(to + 4) = f4{r[c][4], r[c][5], r[c][6], r[c][7]};
            }
        }
        if (live && a.H) *(u4*)(a.H + row * a.ldh + 8 * at) = f32x8_to_f16(f4{y[0], y[1], y[2], y[3]}, f4{y[4], y[5], y[6], y[7]});
        if (p.q) {                                 // four lanes a block of 32 (live or not together)
            float m = 0.f, bad = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                m = __builtin_fmaxf(m, __builtin_fabsf(y[e]));
                bad += y[e] * 0.f;                 // NaN from an infinity or NaN
            }
            m = __builtin_fmaxf(m, __shfl_xor(m, 1));
            m = __builtin_fmaxf(m, __shfl_xor(m, 2));
            bad += __shfl_xor(bad, 1);
            bad += __shfl_xor(bad, 2);
            const float dd = m / 127.0f + bad;
            int q[8], sum = 0;
            codes(q, y, dd);
#pragma unroll
            for (int e = 0; e < 8; e++) sum += q[e];
            sum += __shfl_xor(sum, 1);
            sum += __shfl_xor(sum, 2);
            if (live) {
                uint32_t lo = 0, hi = 0;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    lo |= ((uint32_t)q[e] & 0xFFu) << (8 * e);
                    hi |= ((uint32_t)q[4 + e] & 0xFFu) << (8 * e);
                }
                *(uint2*)(p.q + row * a.K + 8 * at) = uint2{lo, hi};
                if ((at & 3) == 0) {
                    p.d[row * (a.K >> 5) + (at >> 2)] = dd;
                    p.s[row * (a.K >> 5) + (at >> 2)] = sum;
                }
            }
        }
    }
}

// Rows of any length and alignment: an element a thread and turn, the row in LDS.
__global__ __launch_bounds__(256) void k_rms_norm_any(NormDev p) {
    extern __shared__ float r[];
    __shared__ float part[16];
    __shared__ double part64[16];
    const NormArgs& a = p.a;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    float ss = 0.f;
    int n = 0;
    for (int k0 = 0; k0 < a.K; k0 += 32 * 256) {
        float s = 0.f;
        for (int k = k0 + tid; k < min(a.K, k0 + 32 * 256); k += 256, n++) {
            float v = load1(a.X, a.x_f16, row * a.ldx + k);
            if (a.D) v += load1(a.D, a.d_f16, row * a.ldd + k);
            r[k] = v;
            s = __builtin_fmaf(v, v, s);
        }
        ss += s;
    }
    ss = group_sum(ss, part);
    const Factor f = factor(ss, a.K, a.eps, [&](int i) { return r[tid + 256 * i]; }, n, part64);
    for (int k0 = 0; k0 < a.K; k0 += 256) {
        const int k = k0 + tid;
        const bool live = k < a.K;                 // (with codes, K is a multiple of 32: blocks are live together)
        const float v = live ? r[k] : 0.f, y = f.of(v, (live && a.W ? load1(a.W, a.w_f16, k) : 1.f) + a.offset);
        if (live && a.R) {
            if (a.x_f16) ((_Float16*)a.R)[row * a.ldr + k] = (_Float16)v;
            else ((float*)a.R)[row * a.ldr + k] = v;
        }
        if (live && a.H) ((_Float16*)a.H)[row * a.ldh + k] = (_Float16)y;
        if (p.q) {
            float m = __builtin_fabsf(y), bad = y * 0.f;
#pragma unroll
            for (int x = 1; x < 32; x <<= 1) {
                m = __builtin_fmaxf(m, __shfl_xor(m, x));
                bad += __shfl_xor(bad, x);
            }
            const float dd = m / 127.0f + bad;
            const int q = code(quotient(y, dd));
            int sum = q;
#pragma unroll
            for (int x = 1; x < 32; x <<= 1) sum += __shfl_xor(sum, x);
            if (live) {
                p.q[row * a.K + k] = (int8_t)q;
                if ((k & 31) == 0) {
                    p.d[row * (a.K >> 5) + (k >> 5)] = dd;
                    p.s[row * (a.K >> 5) + (k >> 5)] = sum;
                }
            }
        }
    }
}

// Rows of whole 16-byte pieces: eight fp16 or four fp32 values (two pieces) a thread.
bool rows_fit(const void* p, int64_t ld, int f16) { return !p || (((uintptr_t)p & 15) == 0 && ld % (f16 ? 8 : 4) == 0); }

template <int C> void go(const NormDev& p, int threads, hipStream_t st) {
    hipLaunchKernelGGL(k_rms_norm<C>, dim3((unsigned)p.a.T), dim3(threads), 0, st, p);
}

}  // namespace

bool rms_norm_fits(int T, int K) { return K <= kNormMaxK && launch_fits(T, 1024); }

hipError_t rms_norm(const NormArgs& a, hipStream_t st) {
    NormDev p{a, (int8_t*)a.Aq, nullptr, nullptr};
    if (a.Aq) {
        p.d = (float*)(p.q + (int64_t)a.T * a.K);
        p.s = (int*)(p.d + (int64_t)a.T * (a.K / 32));
    }
    const bool wide = a.K % 8 == 0 && rows_fit(a.X, a.ldx, a.x_f16) && rows_fit(a.D, a.ldd, a.d_f16) &&
                      rows_fit(a.R, a.ldr, a.x_f16) && rows_fit(a.W, 0, a.w_f16) && rows_fit(a.H, a.ldh, 1);
    if (wide) {
        const int pieces = a.K / 8, turns = (pieces + 1023) / 1024;
        const int threads = ((pieces + turns - 1) / turns + 63) / 64 * 64;
        if (turns == 1) go<1>(p, threads, st);
        else if (turns == 2) go<2>(p, threads, st);
        else go<4>(p, threads, st);
    } else {
        static std::atomic<uint64_t> attr_set{0};  // one bit per device: LDS limit raised
        int dev = 0;
        hipError_t e = hipGetDevice(&dev);
        if (e != hipSuccess) return e;
        const uint64_t bit = 1ull << (dev & 63);
        if (!(attr_set.load(std::memory_order_acquire) & bit)) {
            e = hipFuncSetAttribute((const void*)k_rms_norm_any, hipFuncAttributeMaxDynamicSharedMemorySize, 4 * kNormMaxK);
            if (e != hipSuccess) return e;
            attr_set.fetch_or(bit, std::memory_order_acq_rel);
        }
        hipLaunchKernelGGL(k_rms_norm_any, dim3((unsigned)a.T), dim3(256), (size_t)4 * a.K, st, p);
    }
    return hipGetLastError();
}

}  // namespace bf
