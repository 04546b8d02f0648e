// tree_attn_few.cuh — tree attention of units of one to four query rows (a single token, a short chain), on the CUDA
// cores (include/llmdiy_tree.h; included by tree_attn.cu).
//
// A cluster of C CTAs per (sequence, kv head), each with an equal run of the cache rows; the first also takes the
// tree's.  Sixteen lanes hold a key, eight dims each: its score is eight products a lane and a sum over the lanes by
// shuffles, and the same lanes add p times their eight dims of V.  U keys a half warp are in flight at once (their K
// and V rows, 32 U bytes a lane), with one rescaling (online softmax in base 2, fp32 throughout) for all of them.
// Warps join through shared memory, CTAs by asynchronous stores that complete on an mbarrier of the row's owner, so
// that no cluster barrier follows the loads; every join is in a fixed order.
//
// Launch, two dependent loads (lengths, rows) and the joins' latency bound it: one row of 16 heads over 1023 cache rows takes
// 5.0 us in a graph (the tensor-core kernel 8.8), over 300 4.5.  Tried: the next keys loaded ahead (one row 5.9 us, four rows
// 9.1 against 8.8), a shuffle sum and an exponential of its own for every key of a lane (5.7 and 8.8; now 8.1).
#pragma once

constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewRows = 4;     // most query rows of a unit
constexpr int kFewCluster = 8;  // most CTAs of a unit

LLMDIY_DEV void few_send4(float4* dst, uint64_t* bar, uint32_t rank, const float4& v) {
    uint32_t d, m;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(smem_u32(dst)), "r"(rank));
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(m) : "r"(smem_u32(bar)), "r"(rank));
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(d),
                 "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(m)
                 : "memory");
}
LLMDIY_DEV void few_send2(float2* dst, uint64_t* bar, uint32_t rank, const float2& v) {
    uint32_t d, m;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(smem_u32(dst)), "r"(rank));
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(m) : "r"(smem_u32(bar)), "r"(rank));
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(d),
                 "f"(v.x), "f"(v.y), "r"(m)
                 : "memory");
}
// Joins up to 32 parts of a row in order, part k's (m, l) in lane k (-inf, 0 past the last), o(k) its dims of this lane.
template <class O>
LLMDIY_DEV float2 few_join(const float2& w, int parts, O o, float4& acc) {
    const float M = redux_max(w.x);
    const float f = ta_ex2(w.x - (M == -INFINITY ? 0.f : M));  // nothing seen: 0 (its l is 0, or NaN, which stays)
    float L = w.y * f;
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) L += __shfl_xor_sync(0xffffffffu, L, d);
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int k = 0; k < parts; ++k) {
        const float fk = __shfl_sync(0xffffffffu, f, k);
        const float4 y = o(k);
        acc.x = __fmaf_rn(fk, y.x, acc.x);
        acc.y = __fmaf_rn(fk, y.y, acc.y);
        acc.z = __fmaf_rn(fk, y.z, acc.z);
        acc.w = __fmaf_rn(fk, y.w, acc.w);
    }
    return make_float2(M, L);
}

LLMDIY_DEV void few_unpack(const uint4& v, uint64_t* x) {  // eight halves as four pairs of floats
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 f = __half22float2(*reinterpret_cast<const half2*>(&w[e]));
        x[e] = ta_f2(f.x, f.y);
    }
}

template <int R, int U>
__global__ void __launch_bounds__(kFewThreads, 2)
    tree_attn_few_k(const __grid_constant__ TaArgs a, const half* K, const half* V, int stride, int* err) {
    __shared__ float4 wo[kFewWarps][R][32], po[R][kFewCluster][32];  // the warps' and the CTAs' parts of each row
    __shared__ float2 wml[kFewWarps][R], pml[R][kFewCluster];
    __shared__ uint64_t got[R];
    const int C = gridDim.x, rank = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int hw = tid >> 4, dim0 = (tid & 15) * 8, G = a.H / a.KV;
    if (tid < R) mbar_init(&got[tid], 1);
    if (tid < 32) mbar_fence_init();
    __syncwarp();
    pdl_wait();  // nothing in global memory has been touched before this
    pdl_launch_dependents();
    const int n = ta_nodes(a, b);
    if (n == 0) return;  // the whole cluster
    if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    const int L = ta_len(a, b);
    uint64_t q[R][4], acc[R][4];  // pairs of dims
    float m[R], l[R];             // (l: of this lane's own keys)
    bool live[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int node = r / G;
        live[r] = r < a.rows && node < n;
        const uint4 y = live[r] ? ld_once_u4(a.Q + ((size_t)b * a.N + node) * a.ldq + (kvh * G + r - node * G) * kTaDim + dim0)
                                : make_uint4(0u, 0u, 0u, 0u);
        few_unpack(y, q[r]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[r][e] = 0;
        m[r] = -INFINITY;
        l[r] = 0.f;
    }
    auto dot = [&](const uint64_t* x, int r) {  // this lane's eight dims
        uint64_t s = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) s = ta_fma2(q[r][e], x[e], s);
        float s0, s1;
        ta_split(s, s0, s1);
        return s0 + s1;
    };
    auto add = [&](int r, float p, const uint64_t* x) {
        const uint64_t pp = ta_f2(p, p);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[r][e] = ta_fma2(pp, x[e], acc[r][e]);
    };
    auto rescale = [&](int r, float top) {  // returns the reference point, the warp's
        const float to = fmaxf(m[r], top), nm = to == -INFINITY ? 0.f : to, f = ta_ex2(m[r] - nm);
        const uint64_t ff = ta_f2(f, f);
        m[r] = to;
        l[r] *= f;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[r][e] = ta_fma2(ff, acc[r][e], 0);
        return nm;
    };
    // A half warp's U scores are summed over its lanes all at once: at each step a lane passes on half of those it
    // has and keeps the others, so that key u's ends up in the 16 / U lanes from u * 16 / U on.
    constexpr int kOwn = 16 / U;
    const int own = (lane & 15) / kOwn;
    const int k1 = (int)((long long)L * (rank + 1) / C);
    int k0 = (int)((long long)L * rank / C) + hw;
    const size_t at = ((size_t)(L ? ta_slot(a, b) : 0) * a.slot_rows + k0) * stride + kvh * kTaDim + dim0;
    const half *kp = K + at, *vp = V + at;
    const size_t jump = (size_t)(2 * kFewWarps) * stride;
    for (; k0 - hw < k1; k0 += 2 * kFewWarps * U, kp += U * jump, vp += U * jump) {
        uint4 kk[U], vv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            kk[u] = vv[u] = make_uint4(0u, 0u, 0u, 0u);
            if (k0 + u * 2 * kFewWarps < k1) {
                kk[u] = ld_once_u4(kp + u * jump);
                vv[u] = ld_once_u4(vp + u * jump);
            }
        }
        float s[R][U], p[R];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint64_t x[4];
            few_unpack(kk[u], x);
#pragma unroll
            for (int r = 0; r < R; ++r) s[r][u] = dot(x, r);
        }
        const bool mine = k0 + own * 2 * kFewWarps < k1;
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int d = 8, h = U / 2; d >= 1; d >>= 1, h >>= 1) {
                if (h == 0) {
                    s[r][0] += __shfl_xor_sync(0xffffffffu, s[r][0], d);
                } else {
#pragma unroll
                    for (int i = 0; i < h; ++i) {
                        const float give = lane & d ? s[r][i] : s[r][i + h], keep = lane & d ? s[r][i + h] : s[r][i];
                        s[r][i] = keep + __shfl_xor_sync(0xffffffffu, give, d);
                    }
                }
            }
            const float x = mine ? s[r][0] * kTaScaleLog2 : -INFINITY;
            const float nm = rescale(r, redux_max(x));
            p[r] = ta_ex2(x - nm);
            l[r] += p[r];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint64_t x[4];
            few_unpack(vv[u], x);
#pragma unroll
            for (int r = 0; r < R; ++r) add(r, __shfl_sync(0xffffffffu, p[r], (lane & 16) + u * kOwn), x);
        }
    }
    if (rank == 0 && 2 * warp < n) {  // the tree's rows, one to a half warp; what a row does not see adds nothing, be it NaN
        const size_t row = (((size_t)b * a.N + min(hw, n - 1)) * a.KV + kvh) * kTaDim + dim0;
        const uint4 kt = ld_once_u4(a.TK + row), vt = ld_once_u4(a.TV + row);
        uint64_t xk[4], xv[4];
        few_unpack(kt, xk);
        few_unpack(vt, xv);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint64_t word = live[r] ? a.mask[(size_t)b * a.N + r / G] : 0;
            const bool sees = hw < n && (word >> hw & 1);
            float x = dot(xk, r);
#pragma unroll
            for (int d = 8; d >= 1; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
            x *= kTaScaleLog2;
            const float nm = rescale(r, redux_max(sees ? x : -INFINITY));
            if (sees) {
                const float p = ta_ex2(x - nm);
                if (own == 0) l[r] += p;  // (one key: in the first one's lanes)
                add(r, p, xv);
            }
        }
    }
    // ---------------- the warp's two halves, the CTA's warps, the cluster's CTAs
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int d = 16; d >= kOwn; d >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], d);
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) ta_split(acc[r][e], x[2 * e], x[2 * e + 1]);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] += __shfl_xor_sync(0xffffffffu, x[e], 16);
        if (lane < 16) {
            wo[warp][r][2 * lane] = make_float4(x[0], x[1], x[2], x[3]);
            wo[warp][r][2 * lane + 1] = make_float4(x[4], x[5], x[6], x[7]);
        }
        if (lane == 0) wml[warp][r] = make_float2(m[r], l[r]);
    }
    if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA's mbarriers are set up
    __syncthreads();
    const int r = warp, node = r / G;
    if (r >= R || r >= a.rows || node >= n) return;
    const float2 none = make_float2(-INFINITY, 0.f);
    float4 o;
    float2 ml = few_join(lane < kFewWarps ? wml[lane][r] : none, kFewWarps, [&](int k) { return wo[k][r][lane]; }, o);
    if (C > 1) {
        const int owner = r % C;
        if (rank == owner && lane == 0) mbar_arrive_expect_tx(&got[r], C * (kTaDim * 4 + 8));
        few_send4(&po[r][rank][lane], &got[r], owner, o);
        if (lane == 0) few_send2(&pml[r][rank], &got[r], owner, ml);
        if (rank != owner) return;
        const bool ok = mbar_wait(&got[r], 0);
        if (!__all_sync(0xffffffffu, ok)) {
            if (lane == 0) atomicExch(err, 1);
            cluster_drain();
        }
        ml = few_join(lane < C ? pml[r][lane] : none, C, [&](int k) { return po[r][k][lane]; }, o);
    }
    ta_store4(a.O + ((size_t)b * a.N + node) * a.ldo + (kvh * G + r - node * G) * kTaDim + lane * 4, o,
              ml.y == 0.f ? 0.f : 1.f / ml.y);
}

template <int R, int U>
int few_launch(const TaArgs& a, const half* K, const half* V, int stride, int* err, int cluster, cudaStream_t st) {
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(cluster, a.KV, a.B);
    lc.blockDim = dim3(kFewThreads);
    lc.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at;
    lc.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&lc, tree_attn_few_k<R, U>, a, K, V, stride, err);
}
