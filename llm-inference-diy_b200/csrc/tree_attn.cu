// tree_attn.cu — attention of a tree of drafted tokens over the cache (include/llmdiy_tree.h).
// No counterpart in the reference, which attends one query token per step.
#include "llmdiy_tree.h"
#include "ops.cuh"

using namespace llmdiy;

namespace {

constexpr int kTaDim = 128;
constexpr int kTaThreads = 128;

// One CTA per (head, node, sequence): half-warp q takes keys q, q + 8, ... of the cache rows and then of the
// tree's, each lane holding 8 of the 128 dims, with an online softmax per half-warp.
__global__ void __launch_bounds__(kTaThreads)
    tree_attn_k(const half* __restrict__ Q, int ldq, const half* __restrict__ K, const half* __restrict__ V, int stride,
                int slot_rows, int num_slots, const int* __restrict__ slot, const int* __restrict__ len, int max_len,
                const half* __restrict__ TK, const half* __restrict__ TV, const uint64_t* __restrict__ mask,
                const int* __restrict__ tree_len, int N, int H, int KV, half* __restrict__ O, int ldo) {
    __shared__ float so[4][kTaDim], sm[4], sl[4];
    const int h = blockIdx.x, i = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const int n = tree_len ? min(max(tree_len[b], 0), N) : N;
    if (i >= n) return;
    const int warp = tid >> 5, lane = tid & 31, hw = lane >> 4, dl = (lane & 15) * 8, hq = warp * 2 + hw;
    const int kvh = h / (H / KV);
    const int at = slot ? slot[b] : b;
    const int L = at >= 0 && at < num_slots ? min(max(len[b], 0), max_len) : 0;
    const size_t row = (size_t)b * N + i;
    const uint64_t* mw = mask + row * ((N + 63) / 64);
    const half* Kb = K + (size_t)max(at, 0) * slot_rows * stride + kvh * kTaDim + dl;
    const half* Vb = V + (size_t)max(at, 0) * slot_rows * stride + kvh * kTaDim + dl;
    const half* Tk = TK + ((size_t)b * N * KV + kvh) * kTaDim + dl;
    const half* Tv = TV + ((size_t)b * N * KV + kvh) * kTaDim + dl;
    float q8[8], o8[8], m = -INFINITY, l = 0.f;
    unpack8(*reinterpret_cast<const uint4*>(Q + row * ldq + h * kTaDim + dl), q8);
#pragma unroll
    for (int e = 0; e < 8; ++e) o8[e] = 0.f;
    const float scale = 0.08838834764831845f;
    for (int k0 = 0; k0 < L + n; k0 += 8) {  // the same bound for every lane: the sums shuffle
        const int k = k0 + hq, j = k - L;
        const bool seen = k < L || (j < n && ((mw[j >> 6] >> (j & 63)) & 1));
        const half* kp = k < L ? Kb + (size_t)k * stride : Tk + (size_t)j * KV * kTaDim;
        const half* vp = k < L ? Vb + (size_t)k * stride : Tv + (size_t)j * KV * kTaDim;
        float kf[8], vf[8], d = 0.f;
        if (seen) {
            unpack8(*reinterpret_cast<const uint4*>(kp), kf);
            unpack8(*reinterpret_cast<const uint4*>(vp), vf);
#pragma unroll
            for (int e = 0; e < 8; ++e) d = __fmaf_rn(q8[e], kf[e], d);
        }
#pragma unroll
        for (int mk = 8; mk >= 1; mk >>= 1) d += __shfl_xor_sync(0xffffffffu, d, mk);
        if (!seen) continue;
        const float s = d * scale, mx = fmaxf(m, s);
        if (mx == -INFINITY) continue;
        const float corr = __expf(m - mx), p = __expf(s - mx);
        l = l * corr + p;
#pragma unroll
        for (int e = 0; e < 8; ++e) o8[e] = __fmaf_rn(p, vf[e], o8[e] * corr);
        m = mx;
    }
    combine_halfwarps(m, l, o8);
    if (lane < 16)
#pragma unroll
        for (int e = 0; e < 8; ++e) so[warp][dl + e] = o8[e];
    if (lane == 0) { sm[warp] = m; sl[warp] = l; }
    __syncthreads();
    float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), Ls = 0.f, acc = 0.f;
    for (int w = 0; w < 4; ++w) {
        if (sm[w] == -INFINITY) continue;
        const float f = __expf(sm[w] - M);
        Ls += sl[w] * f;
        acc = __fmaf_rn(f, so[w][tid], acc);
    }
    O[row * ldo + h * kTaDim + tid] = f2h(Ls == 0.f ? 0.f : acc / Ls);
}

}  // namespace

extern "C" {

size_t llmdiy_tree_attn_work_bytes(int B, int N, int num_heads, int num_kv_heads, int max_len) {
    if (B <= 0 || N <= 0 || N > LLMDIY_TREE_MAX_NODES || num_kv_heads <= 0 || num_heads <= 0 ||
        num_heads % num_kv_heads || max_len < 0)
        return 0;
    return 16;
}

int llmdiy_tree_attn(const uint16_t* Q, int ldq, const uint16_t* K, const uint16_t* V, int stride, int slot_rows,
                     int num_slots, const int* slot, const int* len, int max_len, const uint16_t* TK,
                     const uint16_t* TV, const uint64_t* mask, const int* tree_len, int B, int N, int num_heads,
                     int num_kv_heads, uint16_t* O, int ldo, float* work, size_t work_bytes, void* stream) {
    auto a16 = [](const void* p) { return p && (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    const size_t need = llmdiy_tree_attn_work_bytes(B, N, num_heads, num_kv_heads, max_len);
    if (!need || B > 65535 || !a16(Q) || !a16(K) || !a16(V) || !a16(TK) || !a16(TV) || !a16(O) || !len || !mask ||
        num_heads > 1024 || ldq < num_heads * kTaDim || (ldq & 7) || ldo < num_heads * kTaDim || (ldo & 7) ||
        stride < num_kv_heads * kTaDim || (stride & 7) || slot_rows <= 0 || num_slots <= 0 || max_len > slot_rows ||
        (long long)num_slots * slot_rows > 0x7fffffffLL || !a16(work) || work_bytes < need)
        return (int)cudaErrorInvalidValue;
    tree_attn_k<<<dim3(num_heads, N, B), kTaThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
        reinterpret_cast<const half*>(Q), ldq, reinterpret_cast<const half*>(K), reinterpret_cast<const half*>(V), stride,
        slot_rows, num_slots, slot, len, max_len, reinterpret_cast<const half*>(TK), reinterpret_cast<const half*>(TV),
        mask, tree_len, N, num_heads, num_kv_heads, reinterpret_cast<half*>(O), ldo);
    return (int)cudaGetLastError();
}

int llmdiy_tree_attn_status(const float* work) {
    if (!work) return (int)cudaErrorInvalidValue;
    int h = 0;
    int* word = reinterpret_cast<int*>(const_cast<float*>(work));
    cudaError_t e = cudaMemcpy(&h, word, sizeof(int), cudaMemcpyDeviceToHost);
    if (e != cudaSuccess) return (int)e;
    if (h) cudaMemset(word, 0, sizeof(int));
    return h ? -5 : 0;
}

}  // extern "C"
