// softmax_rows.cu — probabilities of rows of fp16 logits, with a temperature per row
// (include/llmdiy_tree.h).  No counterpart in the reference, whose engine takes the argmax only.
#include "common.cuh"
#include "llmdiy_tree.h"

using namespace llmdiy;

namespace {

constexpr int kSmThreads = 512;

// One CTA per row, three passes over it: maximum, sum, probabilities.
__global__ void __launch_bounds__(kSmThreads)
    softmax_rows_k(const half* __restrict__ logits, int ldl, const float* __restrict__ temp, int V,
                   float* __restrict__ probs, int ldp) {
    __shared__ float red[kSmThreads / 32];
    const int r = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const half* x = logits + (size_t)r * ldl;
    float* y = probs + (size_t)r * ldp;
    const float t = temp ? temp[r] : 1.f;
    const bool greedy = !(t > 0.f);
    const float it = greedy ? 0.f : 1.f / t;
    float mx = -INFINITY;
    for (int i = tid; i < V; i += kSmThreads) mx = fmaxf(mx, h2f(x[i]));
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) red[warp] = mx;
    __syncthreads();
    for (int w = 0; w < kSmThreads / 32; ++w) mx = fmaxf(mx, red[w]);
    __syncthreads();
    // -inf stays below every finite substitute: e = 0 where nothing is above it
    const float m = mx == -INFINITY ? 0.f : mx;
    auto e_of = [&](float v) { return greedy ? (v == m ? 1.f : 0.f) : expf((v - m) * it); };
    float s = 0.f;
    for (int i = tid; i < V; i += kSmThreads) s += e_of(h2f(x[i]));
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) red[warp] = s;
    __syncthreads();
    s = 0.f;
    for (int w = 0; w < kSmThreads / 32; ++w) s += red[w];
    const float inv = s == 0.f ? 0.f : 1.f / s;
    for (int i = tid; i < V; i += kSmThreads) y[i] = e_of(h2f(x[i])) * inv;
}

}  // namespace

extern "C" int llmdiy_softmax_rows(const uint16_t* logits, int ldl, const float* temp, int R, int V, float* probs,
                                   int ldp, void* stream) {
    if (!logits || !probs || R <= 0 || V <= 0 || ldl < V || ldp < V || (reinterpret_cast<uintptr_t>(logits) & 1) ||
        (reinterpret_cast<uintptr_t>(probs) & 3))
        return (int)cudaErrorInvalidValue;
    softmax_rows_k<<<R, kSmThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
        reinterpret_cast<const half*>(logits), ldl, temp, V, probs, ldp);
    return (int)cudaGetLastError();
}
