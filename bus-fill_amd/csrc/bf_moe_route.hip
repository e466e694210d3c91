// Routing to experts: k_moe_route, one wave a token.
//
//   s = softmax(x) or sigmoid(x) over the E experts' logits;
//   chosen: the k experts of largest s + bias (equal ones: the lowest index);
//   with groups: E / groups consecutive experts each, a group's score the sum of
//   its two largest s + bias, the experts of the top_groups best groups only;
//   weights: s of the chosen (without the bias), over their sum if renorm, times
//   factor.
//
// Without a bias the order of s is that of the logits, which are compared
// themselves: nothing hangs on how exp rounds.  Lane l holds experts EPL l ..
// EPL l + EPL - 1, so among equal values the lowest lane's first one has the
// lowest index.  What is compared are integers in the order of the values, with a
// NaN below -inf and nothing (an expert that does not exist, is chosen already or
// is in a group that is not) below a NaN.  A NaN logit has score NaN and takes no
// part in the other experts' softmax; logits of +inf share all of it.
//
// Reads each logit once, from then on everything is in the wave's registers: k
// rounds of a maximum over the wave and the lane that holds it.  4096 rows of 256
// experts in eight groups, eight chosen: 7.2 us (4.5 MB; maxima of floats, without an
// order among NaN, -inf and the lowest value, 8.2), 32 rows of 64: 3.0 us, a launch.
#include <climits>

#include "bf_device.h"
#include "bf_grid.h"
#include "bf_moe_launch.h"

namespace bf {
namespace {

constexpr int kRtWaves = 4;

// In the order of the values: -0 equals 0, a NaN comes before -inf, kNone before that.
constexpr int kNone = INT_MIN;
__device__ __forceinline__ int order_of(float v) {
    const int b = __builtin_bit_cast(int, v + 0.f);
    return v == v ? b ^ ((b >> 31) & INT_MAX) : kNone + 1;
}

// The value of lane 63 after a step-wise reduction over the wave's rows of 16,
// then the rows; lanes without a source keep `none`.
template <typename V, typename F>
__device__ __forceinline__ V wave_reduce(V v, V none, F f) {
#define BF_DPP(ctrl, rows)                                                                                        \
    v = f(v, __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none),                     \
                                                               __builtin_bit_cast(int, v), ctrl, rows, 0xF, false)))
    BF_DPP(0x111, 0xF);        // row_shr:1, 2, 4, 8
    BF_DPP(0x112, 0xF);
    BF_DPP(0x114, 0xF);
    BF_DPP(0x118, 0xF);
    BF_DPP(0x142, 0xA);        // row_bcast:15 into rows 1 and 3
    BF_DPP(0x143, 0xC);        // row_bcast:31 into rows 2 and 3
#undef BF_DPP
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ int wave_max(int v) {
    return wave_reduce(v, kNone, [](int a, int b) { return max(a, b); });
}
__device__ __forceinline__ float wave_max(float v) {
    return wave_reduce(v, -__builtin_inff(), [](float a, float b) { return __builtin_fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float v) {
    return wave_reduce(v, 0.f, [](float a, float b) { return a + b; });
}

// The two largest of two pairs of largest ones.
__device__ __forceinline__ void top2(float& b1, float& b2, float o1, float o2) {
    b2 = __builtin_fmaxf(__builtin_fminf(b1, o1), __builtin_fmaxf(b2, o2));
    b1 = __builtin_fmaxf(b1, o1);
}

template <int EPL>
__global__ __launch_bounds__(64 * kRtWaves) void k_moe_route(RouteArgs a) {
    __shared__ float xs[kRtWaves][65 * EPL];       // of one wave each: a value per expert, one pad word per 64
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t t = blockIdx.x * (int64_t)kRtWaves + wave;
    if (t >= a.T) return;
    const int e0 = lane * EPL;
    const float ninf = -__builtin_inff();
    float x[EPL], s[EPL];
    int sel[EPL];
    const int64_t at = t * a.ldl + e0;
#pragma unroll
    for (int i = 0; i < EPL; i++)
        x[i] = e0 + i >= a.E ? ninf : a.f16 ? (float)((const _Float16*)a.logits)[at + i] : ((const float*)a.logits)[at + i];
    if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < EPL; i++) s[i] = __builtin_amdgcn_rcpf(1.f + expf(-x[i]));
    } else {
        float m = x[0];
#pragma unroll
        for (int i = 1; i < EPL; i++) m = __builtin_fmaxf(m, x[i]);
        m = wave_max(m);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            s[i] = x[i] != m ? expf(x[i] - m) : m == ninf ? 0.f : 1.f;  // (a row of -inf: all zero)
            if (e0 + i < a.E && x[i] == x[i]) sum += s[i];
        }
        sum = wave_sum(sum);
#pragma unroll
        for (int i = 0; i < EPL; i++) s[i] = sum == 0.f ? s[i] : s[i] * __builtin_amdgcn_rcpf(sum);
    }
    // what is compared, of groups and of experts
    float v[EPL];
#pragma unroll
    for (int i = 0; i < EPL; i++) {
        v[i] = a.bias ? s[i] + (e0 + i < a.E ? a.bias[e0 + i] : 0.f) : s[i];
        sel[i] = e0 + i < a.E ? order_of(a.bias ? v[i] : x[i]) : kNone;
    }
    if (a.groups > 1) {
        const int size = a.E / a.groups, lanes = size / EPL;
        float b1 = ninf, b2 = ninf;                                    // (a NaN as -inf)
#pragma unroll
        for (int i = 0; i < EPL; i++) v[i] = e0 + i < a.E ? __builtin_fmaxf(v[i], ninf) : ninf;
        if (lanes * EPL == size && (lanes & (lanes - 1)) == 0) {       // a power of two of lanes holds a group: they meet
#pragma unroll
            for (int i = 0; i < EPL; i++) top2(b1, b2, v[i], ninf);
            for (int d = 1; d < lanes; d *= 2) top2(b1, b2, __shfl_xor(b1, d), __shfl_xor(b2, d));
            const int from = min(lane * lanes, 63);
            b1 = __shfl(b1, from);
            b2 = __shfl(b2, from);
        } else {                                                       // lane g walks through group g
#pragma unroll
            for (int i = 0; i < EPL; i++) xs[wave][e0 + i + (e0 + i) / 64] = v[i];
            for (int i = 0; lane < a.groups && i < size; i++) {
                const int e = lane * size + i;
                top2(b1, b2, xs[wave][e + e / 64], ninf);
            }
        }
        int best = lane >= a.groups ? kNone : order_of(size > 1 ? b1 + b2 : b1);
        uint64_t keep = 0;
        for (int i = 0; i < a.top_groups; i++) {
            const int m = wave_max(best);
            const int l = __builtin_ctzll(__ballot(best == m));
            keep |= 1ull << l;
            if (lane == l) best = kNone;
        }
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            const int g = (e0 + i) / size;
            if (e0 + i < a.E && !((keep >> g) & 1)) sel[i] = kNone;
        }
    }
#pragma unroll
    for (int i = 0; i < EPL; i++) xs[wave][e0 + i + (e0 + i) / 64] = s[i];
    int id = 0;
    for (int j = 0; j < a.k; j++) {
        int b = sel[0];
        int bi = 0;
#pragma unroll
        for (int i = 1; i < EPL; i++)
            if (sel[i] > b) {
                b = sel[i];
                bi = i;
            }
        const int m = wave_max(b);
        const int l = __builtin_ctzll(__ballot(b == m));
        const int e = l * EPL + __builtin_amdgcn_readlane(bi, l);
        if (lane == j) id = e;
#pragma unroll
        for (int i = 0; i < EPL; i++)
            if (e0 + i == e) sel[i] = kNone;
    }
    float w = xs[wave][id + id / 64];
    if (a.renorm) {
        const float sum = wave_sum(lane < a.k ? w : 0.f);
        w = sum == 0.f ? 0.f : w / sum;
    }
    if (lane < a.k) {
        a.ids[t * a.k + lane] = id;
        a.w[t * a.k + lane] = w * a.factor;
    }
}

int64_t groups_of(int T) { return ((int64_t)T + kRtWaves - 1) / kRtWaves; }
}  // namespace

bool moe_route_fits(int T) { return launch_fits(groups_of(T), 64 * kRtWaves); }

hipError_t moe_route(const RouteArgs& a, hipStream_t st) {
    const int epl = (a.E + 63) / 64;
    auto k = epl <= 1 ? k_moe_route<1> : epl <= 2 ? k_moe_route<2> : epl <= 4 ? k_moe_route<4>
             : epl <= 8 ? k_moe_route<8> : k_moe_route<16>;
    hipLaunchKernelGGL(k, dim3((unsigned)groups_of(a.T)), dim3(64 * kRtWaves), 0, st, a);
    return hipGetLastError();
}

}  // namespace bf
