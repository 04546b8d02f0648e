// softmax_rows.cu — probabilities of rows of fp16 logits, with a temperature per row
// (include/llmdiy_tree.h).  No counterpart in the reference, whose engine takes the argmax only.
//
// One pass over memory, by persistent clusters of C CTAs: cluster c takes rows c, c + clusters, ..., slice k of
// a row in CTA k, each warp a run of it.  A bulk copy brings the next row's slice into shared memory while a row, whose
// entries are in registers, is worked on, and its results leave the same way.  Each warp finds its run's maximum m_w and its sum s_w of exponentials
// relative to it (kept in registers as fp32) and sends the pair to every CTA of the cluster by asynchronous stores
// that complete on the receiver's mbarrier; with all the pairs it forms the row's maximum M and sum
// S = sum_w s_w 2^{(m_w - M) k}, k = log2(e) / t, and writes its run times 2^{(m_w - M) k} / S.  With C > 1 no barrier stands in the
// loop.  x - m is exact in fp32 for fp16 x (but for far smaller x, whose share is 0), so
// the exponent carries two roundings (k and the product).
//
// Reading 2 and writing 4 bytes an entry is the bound: 768 rows of 151936 entries take 125 us, 5.6 TB/s of the 6.5 of
// a copy.  What a cluster of nine cannot hold, entries past 156600 (9 kSmSlice) of a row, is read three times, two bytes at a
// time: 400 rows of 151936 take 67 us (5.5 TB/s), of 200000 180 (2.7 TB/s), of 262144 230.  A row is in work for about
// 5 us (shared-memory loads, 16 warps' exponentials, the exchange of the cluster's
// pairs), with 30 clusters of 9 resident.  Rejected: the whole CTA's maximum and sum by barriers and plain stores (clusters
// of 8, 141.7 us; an SM writes 32 bytes a cycle, and the warps wait for that), plain stores without barriers (139.7), one or
// two of a thread's pairs in plain stores for clusters of 8 (137 to 142), clusters of 10 (138.6), rows fetched into L2 two
// ahead (139.0), fp16 entries held and their exponentials taken twice (188).  The last row's results are stored
// plainly (5 rows in all took 5.5 us so and 6.0 by bulk copies when first tried; now 5.3).
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "llmdiy_tree.h"

using namespace llmdiy;

namespace {

constexpr int kSmThreads = 512;
constexpr int kSmPairs = 17;                                  // pairs of entries a thread holds
constexpr int kSmSlice = kSmThreads * kSmPairs * 2 - 8;       // entries a CTA holds (pairs may start one entry early)
constexpr int kSmWarps = kSmThreads / 32;
constexpr int kSmRun = kSmPairs * 64;                         // a warp's run of entries
// The stage: eight entries before the slice's first granule, the granules, and room for every thread's pairs
constexpr int kSmStageBytes = (16 + (kSmThreads * kSmPairs * 2 + 16) * 2 + 127) / 128 * 128;
// Results on their way out: a warp's run, at either 8-byte offset within 16 bytes
constexpr int kSmOutBytes = kSmRun * 4 + 16;
constexpr int kSmBytes = kSmStageBytes + kSmWarps * kSmOutBytes;
constexpr int kSmMaxCluster = 9;
constexpr int kSmTable = (kSmMaxCluster * kSmWarps + 31) / 32;  // pairs of a row that a lane reads
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
LLMDIY_DEV void sm_bulk_out(void* dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\ncp.async.bulk.commit_group;" ::"l"(dst),
                 "r"(smem_u32(src)), "r"(bytes)
                 : "memory");
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
// x + c for both fp16 halves x of w, in fp32 (one instruction each, without a conversion)
LLMDIY_DEV float2 sm_add_halves(uint32_t w, float c) {
    float2 r;
    asm("{\n .reg .f16 a, b;\n mov.b32 {a, b}, %2;\n add.f32.f16 %0, a, %3;\n add.f32.f16 %1, b, %3;\n}"
        : "=f"(r.x), "=f"(r.y)
        : "r"(w), "f"(c));
    return r;
}

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
    extern __shared__ __align__(128) uint8_t stage[];  // kSmStageBytes, then the warps' results
    __shared__ float2 part[2][kSmMaxCluster * kSmWarps];  // (m_w, s_w) of the cluster's warps: odd and even rows
    __shared__ uint64_t full, empty, got[2];
    __shared__ int copied;  // copies issued (the thread that issues them writes and reads it)
    cg::cluster_group cluster = cg::this_cluster();
    // whether some copy begins or ends inside a granule
    const bool edges = (reinterpret_cast<uintptr_t>(logits) & 15) || (ldl & 7) || (V & 7);
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int r0 = blockIdx.x / C, step = gridDim.x / C;
    const int v0 = min(V, rank * slice), n = min(V, v0 + slice) - v0;  // this CTA's entries of every row
    const int held = min(n, kSmSlice);  // those past the registers (rows of more than kSmMaxCluster kSmSlice) are read again
    const uint16_t* base = reinterpret_cast<const uint16_t*>(logits);
    const uintptr_t first = reinterpret_cast<uintptr_t>(base), last = first + 2 * ((uintptr_t)(R - 1) * ldl + V);
    const uint64_t pol = l2_policy_evict_first();
    auto copy = [&](int r) {  // (one thread)
        const SmWindow w = sm_window(base + (size_t)r * ldl + v0, held, first, last);
        const uint32_t bytes = (uint32_t)(w.to - w.from);
        ++copied;
        mbar_arrive_expect_tx(&full, bytes);
        // (the stage begins with the granule that holds the slice's first entry)
        const uintptr_t g0 = reinterpret_cast<uintptr_t>(base + (size_t)r * ldl + v0) & ~(uintptr_t)15;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // after the plain stores to this stage
        if (bytes)
            bulk_g2s(stage + 16 + (w.from - g0), reinterpret_cast<const void*>(w.from), bytes, &full, pol);
    };
    if (tid == 0) {
        copied = 0;
        mbar_init(&full, 1);
        mbar_init(&empty, kSmWarps);
        for (int i = 0; i < 2; ++i) mbar_init(&got[i], 1);
        mbar_fence_init();
    }
    // what no copy writes is -inf for every row
    for (int i = tid; i < kSmStageBytes / 4; i += kSmThreads) reinterpret_cast<uint32_t*>(stage)[i] = 0xFC00FC00u;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    pdl_wait();  // nothing in global memory has been touched before this
    pdl_launch_dependents();
    if (tid == 0 && r0 < R) copy(r0);
    if (C > 1) cluster.sync();  // every CTA of the cluster runs: its shared memory may be written
    int it = 0;
    bool lost = false;  // a wait of this warp has expired (of this CTA where it is a cluster)
    long long row = r0;
    for (; row < R && !lost; row += step, ++it) {
        const size_t r = (size_t)row;
        const uint16_t* x = base + r * ldl + v0;
        float* y = probs + r * ldp + v0;
        const float t = temp ? temp[r] : 1.f;
        const SmWindow win = sm_window(x, held, first, last);
        uint16_t* sx = reinterpret_cast<uint16_t*>(stage + 16) + win.lead;
        // pairs begin where 8-byte stores of the output do
        const int odd = (int)(reinterpret_cast<uintptr_t>(y) >> 2) & 1;
        const int run0 = warp * kSmRun - odd;  // this warp's entries: [run0, run0 + kSmRun) of the slice
        bool ok = mbar_wait(&full, it & 1);
        // The copy's first and last granules hold up to seven entries of the rows beside this slice, and the
        // last row in this stage may have ended up to fourteen entries further on: -inf for those; and
        // where the whole buffer ends inside a granule, its entries come from global memory.  Each warp sees to its own run.
        if (edges) {
            const uintptr_t xa = reinterpret_cast<uintptr_t>(x);
            const int c0 = win.from > xa ? (int)(win.from - xa) / 2 : 0;
            const int c1 = win.to > xa ? min(held, (int)((win.to - xa) / 2)) : 0;
            for (int i = lane; i < 40; i += 32) {
                const int a = i < 16 ? i - 8 : max(held - 8, 8) + i - 16;  // -8 .. 7 and held - 8 .. held + 15
                if (a < run0 || a >= run0 + kSmRun) continue;
                const bool in = a >= 0 && a < held;
                if (!in) sx[a] = 0xFC00;
                else if (a < c0 || a >= c1) sx[a] = x[a];
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // a later copy writes there too
            __syncwarp();
        }
        const uint16_t* mine = sx + run0 + 2 * lane;
        uint32_t w[kSmPairs];
        if (((win.lead - odd) & 1) == 0) {
#pragma unroll
            for (int i = 0; i < kSmPairs; ++i) w[i] = *reinterpret_cast<const uint32_t*>(mine + 64 * i);
        } else {
#pragma unroll
            for (int i = 0; i < kSmPairs; ++i)
                w[i] = sm_pair(mine[64 * i], mine[64 * i + 1]);
        }
        half2 h = __half2half2(__ushort_as_half(0xFC00));
#pragma unroll
        for (int i = 0; i < kSmPairs; ++i) h = __hmax2(h, *reinterpret_cast<const half2*>(&w[i]));  // (NaN reaches the sum)
        float m = fmaxf(__low2float(h), __high2float(h));
        for (int a = kSmSlice + tid; a < n; a += kSmThreads) m = fmaxf(m, h2f(__ushort_as_half(x[a])));
        m = redux_max(m);
        const bool more = row + step < R;
        if (lane == 0) mbar_arrive(&empty);  // this warp has read the stage
        // k is bounded so that 0 * k is 0 and -inf * k is -inf at any t > 0; greedy (t <= 0 or NaN) takes the upper
        // bound, where the smallest difference of two fp16 values gives 2^-inf
        const float k = t > 0.f ? fminf(fmaxf(1.4426950408889634f / t, 1e-30f), 1e30f) : 1e30f;
        auto weight = [&](float v, float top) { return sm_ex2((v - top) * k); };
        const float ref = m == -INFINITY ? 0.f : m;  // nothing above -inf: every weight 0
        uint64_t ex[kSmPairs], s2[2] = {0, 0};
        const uint64_t k2 = sm_f2(k, k);
#pragma unroll
        for (int i = 0; i < kSmPairs; ++i) {
            const float2 f = sm_add_halves(w[i], -ref);
            const float2 d = sm_split(sm_mul2(sm_f2(f.x, f.y), k2));
            ex[i] = sm_f2(sm_ex2(d.x), sm_ex2(d.y));
            s2[i & 1] = sm_add2(s2[i & 1], ex[i]);
        }
        const float2 sp = sm_split(sm_add2(s2[0], s2[1]));
        float s = sp.x + sp.y;
        for (int a = kSmSlice + tid; a < n; a += kSmThreads) s += weight(h2f(__ushort_as_half(x[a])), ref);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (!ok) s = NAN;  // a copy that never landed shows in its row
        // Two tables take turns: a warp sends row i + 2's pair only after every warp's pair of row i + 1 has come,
        // which each sends after it has read row i's table.
        float2* tab = part[it & 1];
        if (tid == 0 && more) {
            if (mbar_wait(&empty, it & 1)) copy((int)row + step);
            else ok = false;
        }
        if (C > 1) {
            if (tid == 0) mbar_arrive_expect_tx(&got[it & 1], C * kSmWarps * 8);
            if (lane < C) sm_send(&tab[rank * kSmWarps + warp], &got[it & 1], lane, m, s);
            ok = mbar_wait(&got[it & 1], (it >> 1) & 1) && ok;
            lost = __any_sync(0xffffffffu, !ok);
        } else {  // (a barrier is quicker within one CTA: a row of 8192 entries 3.7 us against 4.4)
            if (lane == 0) tab[warp] = make_float2(m, s);
            lost = __syncthreads_or(!ok);
        }
        float2 q[kSmTable];
        float M = -INFINITY, total = 0.f;
#pragma unroll
        for (int j = 0; j < kSmTable; ++j) {
            const int at = lane + 32 * j;
            q[j] = at < C * kSmWarps ? tab[at] : make_float2(-INFINITY, 0.f);
            M = fmaxf(M, q[j].x);
        }
        M = redux_max(M);
#pragma unroll
        for (int j = 0; j < kSmTable; ++j)  // (q.x = -inf: a sum of 0, or NaN)
            total += q[j].y * (q[j].x == -INFINITY ? 1.f : weight(q[j].x, M));
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        if (lost) total = NAN;
        const float inv = total == 0.f ? 0.f : 1.f / total;
        const float top = M == -INFINITY ? 0.f : M;
        const float scale = inv * (m == -INFINITY ? 1.f : weight(m, top));
        if (more && run0 < held && !lost) {
            // The next row's entries are taken up while these leave as one bulk copy of each warp: entries c of its run
            // (c = 0: entry run0 of the slice) from [lo, hi), of which [b0, b1) lies between 16-byte boundaries.
            float* to = y + run0;
            const int lo = run0 < 0, end = min(held - run0, kSmRun);
            const int turn = (int)(reinterpret_cast<uintptr_t>(to) >> 2) & 3;  // 0 or 2
            const int b0 = turn ? 2 : 4 * lo, b1 = ((end + turn) & ~3) - turn;
            float* mo = reinterpret_cast<float*>(stage + kSmStageBytes + warp * kSmOutBytes) + turn;
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the last row's have left
            __syncwarp();
            const uint64_t scale2 = sm_f2(scale, scale);
#pragma unroll
            for (int i = 0; i < kSmPairs; ++i)
                *reinterpret_cast<float2*>(mo + 2 * lane + 64 * i) = sm_split(sm_mul2(ex[i], scale2));
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0 && b1 > b0) sm_bulk_out(to + b0, mo + b0, (b1 - b0) * 4);
            const int c = lane < 4 ? lo + lane : max(b1, min(b0, end)) + lane - 4;  // up to three before and behind it
            if (lane < 8 && c < (lane < 4 ? min(b0, end) : end)) to[c] = mo[c];
            for (int a = kSmSlice + tid; a < n; a += kSmThreads) y[a] = weight(h2f(__ushort_as_half(x[a])), top) * inv;
            continue;
        }
        float* out = y + run0 + 2 * lane;
        const int room = held - run0 - 2 * lane;  // entries from this thread's first on
        const int whole = (held - run0) / 64;     // pairs' runs that lie inside the slice as a whole
        const bool head = odd && tid == 0;        // the pair that begins one entry early
        const uint64_t scale2 = sm_f2(scale, scale);
#pragma unroll
        for (int i = 0; i < kSmPairs; ++i) {
            const float2 o = sm_split(sm_mul2(ex[i], scale2));
            if (i == 0 && head) {
                if (held > 0) y[0] = o.y;
            } else if (i < whole || 64 * i + 1 < room) {
                *reinterpret_cast<float2*>(out + 64 * i) = o;
            } else if (64 * i + 1 == room) {
                out[64 * i] = o.x;
            }
        }
        for (int a = kSmSlice + tid; a < n; a += kSmThreads) y[a] = weight(h2f(__ushort_as_half(x[a])), top) * inv;
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    if (lost) {  // this warp's part of the rows that are left is NaN too
        for (; row < R; row += step) {
            float* y = probs + (size_t)row * ldp + v0;
            const int run0 = warp * kSmRun - ((int)(reinterpret_cast<uintptr_t>(y) >> 2) & 1);
            for (int a = max(run0, 0) + lane; a < min(held, run0 + kSmRun); a += 32) y[a] = NAN;
            for (int a = kSmSlice + tid; a < n; a += kSmThreads) y[a] = NAN;
        }
        if (tid == 0 && copied) mbar_drain(&full, (copied - 1) & 1);
        if (C > 1) cluster_drain();
    }
}

// Clusters of C CTAs that run at once on the current device.
int sm_clusters(int C) {
    static std::atomic<int> known[64][kSmMaxCluster + 1];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
    int n = known[dev][C];
    if (n) return n;
    cudaFuncSetAttribute(softmax_rows_k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmBytes);
    cudaFuncSetAttribute(softmax_rows_k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(C);
    lc.blockDim = dim3(kSmThreads);
    lc.dynamicSmemBytes = kSmBytes;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    lc.attrs = at;
    lc.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, softmax_rows_k, &lc) != cudaSuccess || n < 1) n = 1;
    known[dev][C] = n;
    return n;
}

}  // namespace

extern "C" int llmdiy_softmax_rows(const uint16_t* logits, int ldl, const float* temp, int R, int V, float* probs,
                                   int ldp, void* stream) {
    if (!logits || !probs || R <= 0 || V <= 0 || V > (1 << 30) || ldl < V || ldp < V ||
        (reinterpret_cast<uintptr_t>(logits) & 1) || !words_aligned(probs, temp))
        return (int)cudaErrorInvalidValue;
    // CTAs per row: as many as hold it.  (Twice as many gained 0.2 us of 4.9 at 32000 entries up to 16 rows and lost
    // from 32 on, 5.7 against 5.0; at 8192 entries they cost 0.9 of 3.6.)
    const int C = std::min(kSmMaxCluster, (V + kSmSlice - 1) / kSmSlice);
    const int slice = (((V + C - 1) / C) + 7) / 8 * 8;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(std::min(R, sm_clusters(C)) * C);
    lc.blockDim = dim3(kSmThreads);
    lc.dynamicSmemBytes = kSmBytes;
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
