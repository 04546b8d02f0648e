// softmax_rows.cu — probabilities of rows of fp16 logits, with a temperature per row
// (include/llmdiy_tree.h).  No counterpart in the reference, whose engine takes the argmax only.
//
// One pass over memory, by persistent clusters of C CTAs: cluster c takes rows c, c + clusters, ..., slice k of
// a row in CTA k.  Bulk copies bring the next two rows' slices into shared memory while a row is
// worked on; its entries go to registers, which frees their stage for the copy after next.  Each CTA finds
// its slice's maximum m_c and its sum s_c of exponentials relative to it (kept in registers as
// fp32); one exchange of the C pairs through distributed shared memory (asynchronous stores that complete on the
// receiver's mbarrier: a cluster barrier would also wait for the last row's output to be written) gives
// the row's maximum M and sum S = sum_c s_c 2^{(m_c - M) k}, k = log2(e) / t, and every thread writes its share times
// 2^{(m_c - M) k} / S.  x - m is exact in fp32 for fp16 x (but for far smaller x, whose share is 0), so the
// exponent carries two roundings (k and the product).  Reading 2 and writing 4 bytes an entry is the bound.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "llmdiy_tree.h"

using namespace llmdiy;

namespace {

constexpr int kSmThreads = 512;
constexpr int kSmPairs = 20;                                  // pairs of entries a thread holds
constexpr int kSmSlice = kSmThreads * kSmPairs * 2 - 8;       // entries a CTA holds (pairs may start one entry early)
constexpr int kSmStages = 2;
// A stage: eight entries before the slice's first granule, the granules, and room for every thread's pairs
constexpr int kSmStageBytes = (16 + (kSmThreads * kSmPairs * 2 + 16) * 2 + 127) / 128 * 128;
constexpr int kSmMaxCluster = 8;
constexpr int kSmCtasPerSm = 2;

LLMDIY_DEV float sm_ex2(float x) {  // 2^x (2^-inf = 0)
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
LLMDIY_DEV uint32_t sm_pair(uint16_t lo, uint16_t hi) { return (uint32_t)lo | ((uint32_t)hi << 16); }
// Two fp32 values at once
LLMDIY_DEV uint64_t sm_f2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
LLMDIY_DEV float2 sm_split(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
LLMDIY_DEV uint64_t sm_add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
LLMDIY_DEV uint64_t sm_mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// Eight bytes into the shared memory of CTA `rank` of the cluster, counted by the mbarrier there.
LLMDIY_DEV void sm_send(float2* dst, uint64_t* bar, uint32_t rank, float a, float b) {
    uint32_t d, m;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(smem_u32(dst)), "r"(rank));
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(m) : "r"(smem_u32(bar)), "r"(rank));
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(d),
                 "f"(a), "f"(b), "r"(m)
                 : "memory");
}
LLMDIY_DEV float2 sm_floats(uint32_t w) { return __half22float2(*reinterpret_cast<const half2*>(&w)); }

// The 16-byte granules around entries [v0, v0 + n) of a row, cut at the ends of the whole buffer
// [first, last): what a bulk copy brings.  `lead`: where entry v0 lies in a stage, in entries.
struct SmWindow {
    uintptr_t from, to;
    int lead;
};
LLMDIY_DEV SmWindow sm_window(const uint16_t* x, int n, uintptr_t first, uintptr_t last) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = a + 2 * (uintptr_t)n;
    SmWindow w;
    w.lead = (int)(a & 15) / 2;
    w.from = a & ~(uintptr_t)15;
    w.to = (b + 15) & ~(uintptr_t)15;
    if (w.from < first) w.from += 16;
    if (w.to > last) w.to -= 16;
    if (w.to < w.from) w.to = w.from;
    return w;
}

__global__ void __launch_bounds__(kSmThreads, kSmCtasPerSm)
    softmax_rows_k(const half* logits, int ldl, const float* temp, int R, int V, int slice,
                   float* probs, int ldp) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(128) uint8_t stage[];  // [kSmStages][kSmStageBytes]
    __shared__ float red_m[kSmThreads / 32], red_s[kSmThreads / 32];
    __shared__ float2 part[2][kSmMaxCluster];  // (m_c, s_c) of the cluster's CTAs: odd and even rows
    __shared__ uint64_t full[kSmStages], got[2];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int r0 = blockIdx.x / C, step = gridDim.x / C;
    const int v0 = min(V, rank * slice), n = min(V, v0 + slice) - v0;  // this CTA's entries of every row
    const int held = min(n, kSmSlice);  // those past the registers (rows of more than 8 kSmSlice) are read again
    const uint16_t* base = reinterpret_cast<const uint16_t*>(logits);
    const uintptr_t first = reinterpret_cast<uintptr_t>(base), last = first + 2 * ((uintptr_t)(R - 1) * ldl + V);
    const uint64_t pol = l2_policy_evict_first();
    auto copy = [&](int r, int st) {  // (one thread)
        const SmWindow w = sm_window(base + (size_t)r * ldl + v0, held, first, last);
        const uint32_t bytes = (uint32_t)(w.to - w.from);
        mbar_arrive_expect_tx(&full[st], bytes);
        // (a stage begins with the granule that holds the slice's first entry)
        const uintptr_t g0 = reinterpret_cast<uintptr_t>(base + (size_t)r * ldl + v0) & ~(uintptr_t)15;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // after the plain stores to this stage
        if (bytes)
            bulk_g2s(stage + st * kSmStageBytes + 16 + (w.from - g0), reinterpret_cast<const void*>(w.from), bytes, &full[st],
                     pol);
    };
    if (tid == 0) {
        for (int i = 0; i < kSmStages; ++i) mbar_init(&full[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&got[i], 1);
        mbar_fence_init();
    }
    // what no copy writes is -inf for every row
    for (int i = tid; i < kSmStages * kSmStageBytes / 4; i += kSmThreads) reinterpret_cast<uint32_t*>(stage)[i] = 0xFC00FC00u;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    pdl_wait();  // nothing in global memory has been touched before this
    pdl_launch_dependents();
    if (tid == 0)
        for (int i = 0; i < kSmStages; ++i)
            if (r0 + (long long)i * step < R) copy(r0 + i * step, i);
    if (C > 1) cluster.sync();  // every CTA of the cluster runs: its shared memory may be written
    int it = 0;
    for (long long row = r0; row < R; row += step, ++it) {
        const size_t r = (size_t)row;
        const uint16_t* x = base + r * ldl + v0;
        float* y = probs + r * ldp + v0;
        const int st = it % kSmStages;
        const float t = temp ? temp[r] : 1.f;
        const SmWindow win = sm_window(x, held, first, last);
        uint16_t* sx = reinterpret_cast<uint16_t*>(stage + st * kSmStageBytes + 16) + win.lead;
        const bool ok = mbar_wait(&full[st], (it / kSmStages) & 1);
        // The copy's first and last granules hold up to seven entries of the rows beside this slice, and the
        // last row in this stage may have ended up to fourteen entries further on: -inf for those; and
        // where the whole buffer ends inside a granule, its entries come from global memory.
        if (tid < 40) {
            const uintptr_t xa = reinterpret_cast<uintptr_t>(x);
            const int c0 = win.from > xa ? (int)(win.from - xa) / 2 : 0;
            const int c1 = win.to > xa ? min(held, (int)((win.to - xa) / 2)) : 0;
            const int a = tid < 16 ? tid - 8 : max(held - 8, 8) + tid - 16;  // -8 .. 7 and held - 8 .. held + 15
            const bool in = a >= 0 && a < held;
            if (!in) sx[a] = 0xFC00;
            else if (a < c0 || a >= c1) sx[a] = x[a];
        }
        __syncthreads();
        // pairs begin where 8-byte stores of the output do
        const int odd = (int)(reinterpret_cast<uintptr_t>(y) >> 2) & 1;
        const uint16_t* mine = sx - odd + 2 * tid;
        uint32_t w[kSmPairs];
        if (((win.lead - odd) & 1) == 0) {
#pragma unroll
            for (int i = 0; i < kSmPairs; ++i) w[i] = *reinterpret_cast<const uint32_t*>(mine + 2 * i * kSmThreads);
        } else {
#pragma unroll
            for (int i = 0; i < kSmPairs; ++i)
                w[i] = sm_pair(mine[2 * i * kSmThreads], mine[2 * i * kSmThreads + 1]);
        }
        half2 h = __half2half2(__ushort_as_half(0xFC00));
#pragma unroll
        for (int i = 0; i < kSmPairs; ++i) h = __hmax2(h, *reinterpret_cast<const half2*>(&w[i]));  // (NaN reaches the sum)
        float m = fmaxf(__low2float(h), __high2float(h));
        for (int a = kSmSlice + tid; a < n; a += kSmThreads) m = fmaxf(m, h2f(__ushort_as_half(x[a])));
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (lane == 0) red_m[warp] = m;
        __syncthreads();  // the stage has been read
        if (tid == 0 && row + (long long)kSmStages * step < R) copy((int)row + kSmStages * step, st);
        m = red_m[lane & (kSmThreads / 32 - 1)];
#pragma unroll
        for (int o = kSmThreads / 64; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        // k is bounded so that 0 * k is 0 and -inf * k is -inf at any t > 0; greedy (t <= 0 or NaN) takes the upper
        // bound, where the smallest difference of two fp16 values gives 2^-inf
        const float k = t > 0.f ? fminf(fmaxf(1.4426950408889634f / t, 1e-30f), 1e30f) : 1e30f;
        auto weight = [&](float v, float top) { return sm_ex2((v - top) * k); };
        const float ref = m == -INFINITY ? 0.f : m;  // nothing above -inf: every weight 0
        uint64_t ex[kSmPairs], s2[2] = {0, 0};
        const uint64_t minus = sm_f2(-ref, -ref), k2 = sm_f2(k, k);
#pragma unroll
        for (int i = 0; i < kSmPairs; ++i) {
            const float2 f = sm_floats(w[i]);
            const float2 d = sm_split(sm_mul2(sm_add2(sm_f2(f.x, f.y), minus), k2));
            ex[i] = sm_f2(sm_ex2(d.x), sm_ex2(d.y));
            s2[i & 1] = sm_add2(s2[i & 1], ex[i]);
        }
        const float2 sp = sm_split(sm_add2(s2[0], s2[1]));
        float s = sp.x + sp.y;
        for (int a = kSmSlice + tid; a < n; a += kSmThreads) s += weight(h2f(__ushort_as_half(x[a])), ref);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) red_s[warp] = s;
        __syncthreads();
        float M = m, total = red_s[lane & (kSmThreads / 32 - 1)];
#pragma unroll
        for (int o = kSmThreads / 64; o >= 1; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        if (!ok) total = NAN;  // a copy that never landed shows in its row
        if (C > 1) {
            // Two tables take turns: a CTA sends row i + 2's pair only after every CTA's pair of row i + 1 has come,
            // which each sends after it has read row i's table.
            float2* tab = part[it & 1];
            if (tid == 0) mbar_arrive_expect_tx(&got[it & 1], C * 8);
            if (tid < C) sm_send(&tab[rank], &got[it & 1], tid, m, total);
            const bool all = mbar_wait(&got[it & 1], (it >> 1) & 1);
            const float2 q = tab[lane & (C - 1)];
            M = q.x;
            for (int o = C / 2; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
            total = q.y * (q.x == -INFINITY ? 1.f : weight(q.x, M));  // (q.x = -inf: a sum of 0, or NaN)
            for (int o = C / 2; o >= 1; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
            if (!all) total = NAN;
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;
        const float top = M == -INFINITY ? 0.f : M;
        const float scale = inv * (m == -INFINITY ? 1.f : weight(m, top));
        float2* out = reinterpret_cast<float2*>(y - odd) + tid;
        const int room = held + odd - 2 * tid;           // entries from this thread's first on
        const int whole = (held + odd) / (2 * kSmThreads);  // runs that lie inside the slice as a whole
        const bool head = odd && tid == 0;               // the pair that begins one entry early
        const uint64_t scale2 = sm_f2(scale, scale);
#pragma unroll
        for (int i = 0; i < kSmPairs; ++i) {
            const float2 o = sm_split(sm_mul2(ex[i], scale2));
            if (i == 0 && head) {
                if (held > 0) y[0] = o.y;
            } else if (i < whole || 2 * i * kSmThreads + 1 < room) {
                out[i * kSmThreads] = o;
            } else if (2 * i * kSmThreads + 1 == room) {
                out[i * kSmThreads].x = o.x;
            }
        }
        for (int a = kSmSlice + tid; a < n; a += kSmThreads) y[a] = weight(h2f(__ushort_as_half(x[a])), top) * inv;
    }
}

// Clusters of C CTAs that run at once on the current device.
int sm_clusters(int C) {
    static std::atomic<int> known[64][4];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
    const int slot = C == 1 ? 0 : C == 2 ? 1 : C == 4 ? 2 : 3;
    int n = known[dev][slot];
    if (n) return n;
    cudaFuncSetAttribute(softmax_rows_k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmStages * kSmStageBytes);
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(C);
    lc.blockDim = dim3(kSmThreads);
    lc.dynamicSmemBytes = kSmStages * kSmStageBytes;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    lc.attrs = at;
    lc.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, softmax_rows_k, &lc) != cudaSuccess || n < 1) n = 1;
    known[dev][slot] = n;
    return n;
}

}  // namespace

extern "C" int llmdiy_softmax_rows(const uint16_t* logits, int ldl, const float* temp, int R, int V, float* probs,
                                   int ldp, void* stream) {
    if (!logits || !probs || R <= 0 || V <= 0 || V > (1 << 30) || ldl < V || ldp < V ||
        (reinterpret_cast<uintptr_t>(logits) & 1) || !words_aligned(probs, temp))
        return (int)cudaErrorInvalidValue;
    // CTAs per row: enough to hold it, and more while they leave SMs idle and a slice stays above 4096 entries
    int C = 1;
    while (C < kSmMaxCluster && ((V + C - 1) / C > kSmSlice || ((long long)R * C < 74 && V / C >= 8192))) C *= 2;
    const int slice = (((V + C - 1) / C) + 7) / 8 * 8;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(std::min(R, sm_clusters(C)) * C);
    lc.blockDim = dim3(kSmThreads);
    lc.dynamicSmemBytes = kSmStages * kSmStageBytes;
    lc.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at;
    lc.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&lc, softmax_rows_k, reinterpret_cast<const half*>(logits), ldl, temp, R, V, slice,
                                   probs, ldp);
}
