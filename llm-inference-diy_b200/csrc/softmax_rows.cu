// softmax_rows.cu — probabilities of rows of fp16 logits, with a temperature per row
// (include/llmdiy_tree.h).  No counterpart in the reference, whose engine takes the argmax only.
//
// One pass over memory: a cluster of C CTAs holds a row in registers (as fp16), slice c of it in CTA c.
// Each CTA finds its slice's maximum and its sum of exponentials relative to that maximum; one
// exchange of the C pairs through distributed shared memory gives the row's maximum M and sum
// S = sum_c s_c 2^{(m_c - M) k}, k = log2(e) / t, and every thread writes 2^{(x - M) k} / S from its
// registers.  x - M is exact in fp32 for fp16 x (but for far smaller x, whose share is 0), so the exponent carries
// two roundings (k and the product).  Reading 2 and writing 4 bytes an entry is the bound: the exponentials
// are taken twice (the second time for M) rather than kept, which would double the registers.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "llmdiy_tree.h"

using namespace llmdiy;

namespace {

constexpr int kSmThreads = 256;
constexpr int kSmVecs = 10;                              // eight entries each, per thread
constexpr int kSmSlice = kSmThreads * kSmVecs * 8;       // entries a CTA holds
constexpr int kSmMaxCluster = 8;

LLMDIY_DEV float sm_ex2(float x) {  // 2^x (2^-inf = 0)
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
LLMDIY_DEV uint32_t sm_pair(uint16_t lo, uint16_t hi) { return (uint32_t)lo | ((uint32_t)hi << 16); }
LLMDIY_DEV float2 sm_floats(uint32_t w) { return __half22float2(*reinterpret_cast<const half2*>(&w)); }

// VEC: rows of logits and probabilities are 16-byte aligned; a thread's entries are runs of eight (16-byte
// loads, two 16-byte stores).  Otherwise entry e of vector i is at (8 i + e) * threads + thread of
// the slice, so that a warp's 2-byte loads and 4-byte stores are consecutive.
template <bool VEC>
__global__ void __launch_bounds__(kSmThreads, 3)
    softmax_rows_k(const half* __restrict__ logits, int ldl, const float* __restrict__ temp, int V, int slice,
                   float* __restrict__ probs, int ldp) {
    namespace cg = cooperative_groups;
    constexpr uint32_t kNone = 0xFC00FC00u;  // a pair of -inf
    __shared__ float red_m[kSmThreads / 32], red_s[kSmThreads / 32];
    __shared__ float2 part[kSmMaxCluster];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const size_t r = blockIdx.x / C;
    if (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // "this CTA runs"
    const int v0 = min(V, rank * slice), n = min(V, v0 + slice) - v0;  // this CTA's entries
    const uint16_t* x = reinterpret_cast<const uint16_t*>(logits) + r * ldl + v0;
    float* y = probs + r * ldp + v0;
    const float t = temp ? temp[r] : 1.f;
    // entries past the registers' kSmSlice (rows of more than 8 x kSmSlice entries) are read again each time
    const int held = min(n, kSmSlice);
    uint32_t w[kSmVecs][4];
#pragma unroll
    for (int i = 0; i < kSmVecs; ++i) {
        if (VEC) {
            const int at = (i * kSmThreads + tid) * 8;
            if (at + 8 <= held) {
                const uint4 u = ld_stream_u4(x + at);
                w[i][0] = u.x; w[i][1] = u.y; w[i][2] = u.z; w[i][3] = u.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    w[i][e] = sm_pair(at + 2 * e < held ? x[at + 2 * e] : 0xFC00, at + 2 * e + 1 < held ? x[at + 2 * e + 1] : 0xFC00);
            }
        } else {
            if (i * 8 * kSmThreads >= held) {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[i][e] = kNone;
                continue;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int a0 = (i * 8 + 2 * e) * kSmThreads + tid, a1 = a0 + kSmThreads;
                w[i][e] = sm_pair(a0 < held ? __ldg(x + a0) : 0xFC00, a1 < held ? __ldg(x + a1) : 0xFC00);
            }
        }
    }
    // maximum of the slice (NaN is passed over here; it reaches the sum)
    half2 h = __half2half2(__ushort_as_half(0xFC00));
#pragma unroll
    for (int i = 0; i < kSmVecs; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) h = __hmax2(h, *reinterpret_cast<const half2*>(&w[i][e]));
    float m = fmaxf(__low2float(h), __high2float(h));
    for (int a = kSmSlice + tid; a < n; a += kSmThreads) m = fmaxf(m, h2f(__ushort_as_half(x[a])));
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) red_m[warp] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSmThreads / 32; ++k) m = fmaxf(m, red_m[k]);
    // greedy (t <= 0 or NaN): the exponent is 0 at the maximum and -inf elsewhere.  k is bounded so that
    // 0 * k is 0 at any t > 0.
    const bool greedy = !(t > 0.f);
    const float k = greedy ? 0.f : fminf(1.4426950408889634f / t, 1e30f);
    auto weight = [&](float v, float top) {
        return greedy ? (v == top ? 1.f : v != v ? v : 0.f) : sm_ex2((v - top) * k);
    };
    const float ref = m == -INFINITY ? 0.f : m;  // nothing above -inf: every weight 0
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kSmVecs; ++i) {
        float a = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = sm_floats(w[i][e]);
            a += weight(f.x, ref) + weight(f.y, ref);
        }
        s += a;
    }
    for (int a = kSmSlice + tid; a < n; a += kSmThreads) s += weight(h2f(__ushort_as_half(x[a])), ref);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) red_s[warp] = s;
    __syncthreads();
    float M = m, total = 0.f;
#pragma unroll
    for (int j = 0; j < kSmThreads / 32; ++j) total += red_s[j];
    if (C > 1) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        if (tid < C) *cluster.map_shared_rank(&part[rank], tid) = make_float2(m, total);
        cluster.sync();
        for (int c = 0; c < C; ++c) M = fmaxf(M, part[c].x);
        total = 0.f;
        for (int c = 0; c < C; ++c) {
            const float2 q = part[c];
            const float f = q.x == -INFINITY ? 1.f : q.x == M ? 1.f : greedy ? 0.f : sm_ex2((q.x - M) * k);
            total += q.y * f;  // (q.x = -inf: a sum of 0, or NaN)
        }
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const float top = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int i = 0; i < kSmVecs; ++i) {
        float o[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = sm_floats(w[i][e]);
            o[2 * e] = weight(f.x, top) * inv;
            o[2 * e + 1] = weight(f.y, top) * inv;
        }
        if (VEC) {
            const int at = (i * kSmThreads + tid) * 8;
            if (at + 8 <= held) {
                *reinterpret_cast<float4*>(y + at) = make_float4(o[0], o[1], o[2], o[3]);
                *reinterpret_cast<float4*>(y + at + 4) = make_float4(o[4], o[5], o[6], o[7]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (at + e < held) y[at + e] = o[e];
            }
        } else if (i * 8 * kSmThreads < held) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int at = (i * 8 + e) * kSmThreads + tid;
                if (at < held) y[at] = o[e];
            }
        }
    }
    for (int a = kSmSlice + tid; a < n; a += kSmThreads) y[a] = weight(h2f(__ushort_as_half(x[a])), top) * inv;
}

}  // namespace

extern "C" int llmdiy_softmax_rows(const uint16_t* logits, int ldl, const float* temp, int R, int V, float* probs,
                                   int ldp, void* stream) {
    if (!logits || !probs || R <= 0 || V <= 0 || ldl < V || ldp < V || (reinterpret_cast<uintptr_t>(logits) & 1) ||
        (reinterpret_cast<uintptr_t>(probs) & 3))
        return (int)cudaErrorInvalidValue;
    const bool vec = (reinterpret_cast<uintptr_t>(logits) & 15) == 0 && (reinterpret_cast<uintptr_t>(probs) & 15) == 0 &&
                     ldl % 8 == 0 && ldp % 4 == 0;
    // CTAs per row: enough to hold it, and more while they leave SMs idle and a slice stays above 4096 entries
    int C = 1;
    while (C < kSmMaxCluster && ((V + C - 1) / C > kSmSlice || ((long long)R * C < 74 && V / C >= 8192))) C *= 2;
    if ((long long)R * C > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    const int slice = (((V + C - 1) / C) + 7) / 8 * 8;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(R * C);
    lc.blockDim = dim3(kSmThreads);
    lc.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    lc.attrs = at;
    lc.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&lc, vec ? softmax_rows_k<true> : softmax_rows_k<false>,
                                   reinterpret_cast<const half*>(logits), ldl, temp, V, slice, probs, ldp);
}
