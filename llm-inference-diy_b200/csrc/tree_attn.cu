// tree_attn.cu — attention of a tree of drafted tokens over the cache (include/llmdiy_tree.h), on the
// tcgen05 tensor cores.  No counterpart in the reference, which attends one query token per step.
//
// (Units of one to four query rows with short caches have a kernel of their own on the CUDA cores, tree_attn_few.cuh: a
// CTA's setup of TMEM, tensor maps and MMAs costs more there than the products.)
//
// Work.  A unit is (sequence, kv head, M tile): the query rows m = node * G + g of the G heads that share the kv
// head, at most 128 rows (the MMA's M) of whole nodes.  A unit's keys are 64-row tiles: the cache
// rows [0, len), then the tree's own rows.  Two ways to share them out (ta_plan):
//
// Direct: a cluster of C <= 16 CTAs per unit, its tiles in C equal runs; the CTAs' parts (o unnormalised, m, l) are
// joined through distributed shared memory, each CTA finishing a share of the rows.  One launch, no global
// scratch.
//
// Flat: all units' tiles in a row, each unit with kTaUnitCost tiles more for its beginning and end, dealt to a
// grid of two CTAs per SM in equal contiguous ranges cut anywhere, so that ragged batches keep every SM
// busy to the end.  Whole units write their output, cut ones an fp32 partial, which tree_merge_k joins
// in order (both ways join in a fixed order: the same bits every time).
//
// CTA.  Warp 4 streams Q (once per unit) and the K and V tiles by TMA through rings that run on
// across units; warps 5 and 6 issue the MMAs:
//   S(j)  = Q K(j)^T          128 x 64,  K = 128 dims      -> TMEM, two buffers
//   O    += P(j) V(j)         128 x 128, K = 2 x 64 keys   -> TMEM (P from TMEM, in the place of S(j))
// S(j+1) is computed while the rows are at S(j), S(j+2) when the product that reads P(j) is complete.  Warps 0-3 own the
// rows (thread = row = TMEM lane): mask, online softmax in base 2; O is rescaled only when a row's maximum grows by more
// than 2^7 (P stays within fp16, and O / l does not depend on the reference point).
//
// P goes to the tensor cores as the sum of two fp16 terms, p = hi + lo, for rows of every call alike: half a step of one
// term is 2^-11 of each probability, whose scatter in the output is as large as the output's own rounding (2.9e-4 of the
// norm together on normal inputs, 2.1e-4 with two terms, as fp32 probabilities give), and shows as it is where values
// cancel.  Two terms leave 2^-22 of each, or 2^-32 of the row's largest (kTaRaise); l sums the unrounded fp32 values.  They cost 1.1 us of 11.3
// per call (26 nodes over 2047 rows), 8 of 71 (16 ragged trees) and 32 of 183 (2 x 48 nodes over 65536 rows, grouped): 28 of
// these the second product, the others its conversions.  With one S buffer, and P beside it, the rows wait for the last
// product before they can store P: 12.1, 85 and 226 us for these.
//
// What a row does not see must not reach it even as NaN * 0: masked scores are replaced by -inf
// (K may hold anything there), and V rows past the end, as well as tree rows with an Inf or NaN, are zeroed in
// shared memory before PV; the few rows that do see such a tree row add p * v themselves at the end.
//
// Bounds and what was measured (in a graph, where not said otherwise).  Short caches: launch, barriers, TMEM and first
// instructions (about 7 us) and 0.9 us a tile; 26 nodes x 16 heads over 2047 rows take 11.8 us (5 tiles a CTA), 12.4 per call.
// Long ones: HBM for few rows (64 nodes over 131072 rows of 16 heads 188 us, 5.7 TB/s of the 6.5 of a copy), for many the
// chain S, softmax, P, PV of a tile, with the tensor pipe at 67% (2 x 48 nodes, 32 heads on 8, over 65536 rows 176 us, 555
// TFLOP/s of S and one P; 215 per call, where it runs for long enough to meet the power limit: 1.58 GHz and less).  Ragged
// batches: 16 trees of 64 nodes, 16 heads, over up to 4160 rows 67 us, 79 per call, about 10 of them joining.
// Rejected, measured with P in one fp16 term (66.5 us that batch): two threads a row (94), unrolling the tile loop (78),
// fetching K and V into L2 a tile further ahead (131072 rows 211 us against 182), rows repeated over the lanes of small
// units, other joins (4 or 8 warps a block).
//
// Every wait is bounded; on expiry the CTA records an error in *err, waits (bounded) for its copies and
// MMAs in flight, frees its TMEM and returns.
#include <cuda.h>

#include <algorithm>
#include <cmath>
#include <atomic>
#include <mutex>

#include "gemm_tc_host.h"
#include "llmdiy_tree.h"
#include "ops.cuh"
#include "tc.cuh"

using namespace llmdiy;

namespace {

constexpr int kTaDim = 128;
constexpr int kTaKeys = 64;      // keys per tile
constexpr int kTaRows = 128;     // query rows of a unit at most (MMA M)
constexpr int kTaThreads = 224;  // warps 0-3: rows; warp 4: TMA; warps 5 and 6: the MMAs of S and of O
constexpr int kTaCtasPerSm = 2;
constexpr int kTaTileBytes = kTaKeys * kTaDim * 2;  // one K or V tile
constexpr uint32_t kTaCols = 256;                   // TMEM: two buffers of S, then P over it (64 columns each) | O (128)
constexpr int kTaDirectTiles = 48;  // (see ta_plan)
constexpr int kTaMaxGroup = 128;                    // query heads per kv head at most
constexpr int kTaCluster = 8;     // CTAs per unit (direct); long caches of few units take 12 or 16 (see ta_plan)
// a unit's beginning and end in tiles (16 ragged trees, P in one term: 1 70.9 us, 2 67.9, 4 67.2, 6 66.8, 10 68.4)
constexpr int kTaUnitCost = 4;

// Two layouts of the same kernel: units of up to 64 rows need only 16 KB for Q and get a third V
// stage; the MMA still reads 128 rows, so rows 64-127 of its A operand are whatever lies behind
// (rows do not mix, and nothing is read out of those).
template <int QR, int KS, int VS>
struct TaSmem {
    half q[2][QR * 64];           // dims 0-63 | 64-127: K-major, 128-byte swizzle
    half k[KS][2][kTaKeys * 64];  // per stage, dims 0-63 | 64-127, K-major (8 KB each)
    half v[VS][2][kTaKeys * 64];  // per stage, dims 0-63 | 64-127, MN-major (8 KB each)
    uint64_t q_full, q_empty, k_full[KS], k_empty[KS], v_full[VS], v_empty[VS];
    uint64_t s_full[2], p_full[2], o_done[2], drain[2];
    // tree rows with a non-finite V, by tree tile and quarter (a warp's 16 rows); two units' worth
    alignas(8) uint16_t bad[2][4][4];
    uint32_t tmem_base;
    int fail;
};

struct TaArgs {
    const int* slot;
    const int* len;
    const int* tree_len;
    const uint64_t* mask;
    const half *Q, *TK, *TV;  // for the rare rows that see a non-finite V
    half* O;
    float* part;  // [W][2][rows][128] fp32, then [W][2][rows][2]
    int B, N, H, KV, ldq, ldo, slot_rows, num_slots, max_len;
    int rows;  // rows of a partial: G * nodes_per_tile
    int npt;   // nodes per M tile
    int mt;    // M tiles of a kv head (of the longest tree)
    int W;     // flat: most CTAs that share the tiles of one M tile
    int evict_first;
};

LLMDIY_DEV int ta_nodes(const TaArgs& a, int b) {
    return a.tree_len ? min(max(a.tree_len[b], 0), a.N) : a.N;
}
LLMDIY_DEV int ta_slot(const TaArgs& a, int b) { return a.slot ? a.slot[b] : b; }
LLMDIY_DEV int ta_len(const TaArgs& a, int b) {
    const int s = ta_slot(a, b);
    return s >= 0 && s < a.num_slots ? min(max(a.len[b], 0), a.max_len) : 0;
}
// Tiles of a unit of sequence b, and its units of one M tile (its kv heads).
LLMDIY_DEV void ta_shape(const TaArgs& a, int b, int& n, int& L, int& tiles, int& units) {
    n = ta_nodes(a, b);
    L = n ? ta_len(a, b) : 0;
    tiles = (L + kTaKeys - 1) / kTaKeys + (n + kTaKeys - 1) / kTaKeys;
    units = n ? a.KV : 0;
}

// Flat positions: a unit takes kTaUnitCost + tiles of them, the first kTaUnitCost without a tile.  W CTAs:
// CTA w has [ta_start_of(w), ta_start_of(w + 1)).
struct TaDeal {
    int total, W, base, rem;
    LLMDIY_DEV TaDeal(int total_, int most) : total(total_), W(min(most, total_)) {
        base = W ? total / W : 0;
        rem = total - base * W;
    }
    LLMDIY_DEV int start(int w) const { return base * w + min(w, rem); }
    LLMDIY_DEV int owner(int f) const {
        const int big = (base + 1) * rem;  // the first rem CTAs have one position more
        return f < big ? f / (base + 1) : rem + (f - big) / base;
    }
};

// A unit, and what is left of a CTA's range from position `at` of it on.
struct TaCursor {
    int b, n, L, tiles, units;  // sequence and its shape
    int unit;                   // within the sequence: kv head
    int at;                     // flat position within the unit
    int left;                   // positions left of this CTA's range
    int row0;                   // first cache row of the sequence's slot (set by the producer)
    // the range's tiles of this unit: [t0, t0 + result)
    LLMDIY_DEV int seg(int& t0) const {
        t0 = max(at - kTaUnitCost, 0);
        return max(min(at + left, tiles + kTaUnitCost) - kTaUnitCost, 0) - t0;
    }
    LLMDIY_DEV void next(const TaArgs& a) {  // to the next unit
        left -= tiles + kTaUnitCost - at;
        at = 0;
        if (left <= 0) {
            left = 0;
            return;
        }
        if (++unit < units) return;
        unit = 0;
        do {
            if (++b >= a.B) {  // (not reached while left > 0, unless the lengths change under the kernel)
                left = 0;
                return;
            }
            ta_shape(a, b, n, L, tiles, units);
        } while (units == 0);
    }
};

// The unit at position f of the flat order, c.at = f within it; returns that unit's first position
// (f < total; a whole warp calls it together).
LLMDIY_DEV int ta_locate(const TaArgs& a, int f, int lane, TaCursor& c) {
    int before = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {  // 32 sequences at a time, inclusive sums
        int n = 0, L = 0, tiles = 0, units = 0;
        if (b0 + lane < a.B) ta_shape(a, b0 + lane, n, L, tiles, units);
        const int own = (tiles + kTaUnitCost) * units;
        int inc = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += o;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + inc > f);
        if (hit) {
            const int l = __ffs(hit) - 1;
            c.b = b0 + l;
            c.n = __shfl_sync(0xffffffffu, n, l);
            c.L = __shfl_sync(0xffffffffu, L, l);
            c.tiles = __shfl_sync(0xffffffffu, tiles, l);
            c.units = __shfl_sync(0xffffffffu, units, l);
            const int rest = f - before - __shfl_sync(0xffffffffu, inc - own, l);
            c.unit = rest / (c.tiles + kTaUnitCost);
            c.at = rest - c.unit * (c.tiles + kTaUnitCost);
            return f - c.at;
        }
        before += __shfl_sync(0xffffffffu, inc, 31);
    }
    c.left = 0;  // (not reached: the position lies in some sequence)
    return 0;
}
LLMDIY_DEV int ta_total(const TaArgs& a, int lane) {
    int t = 0;
    for (int i = lane; i < a.B; i += 32) {
        int n, L, tiles, units;
        ta_shape(a, i, n, L, tiles, units);
        t += (tiles + kTaUnitCost) * units;
    }
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) t += __shfl_xor_sync(0xffffffffu, t, m);
    return t;
}

LLMDIY_DEV void named_bar_arrive(int id, int nthreads) {
    asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(nthreads) : "memory");
}
LLMDIY_DEV void tma_load_3d(void* dst, const void* tmap, int32_t x, int32_t y, int32_t z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_u32(dst)), "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}
// Loads from the shared memory of CTA `rank` of the cluster (addr: the same variable's address here).
LLMDIY_DEV float2 ta_peer_f2(uint32_t addr, uint32_t rank) {
    float2 v;
    asm volatile("{\n .reg .b32 p;\n mapa.shared::cluster.u32 p, %2, %3;\n ld.shared::cluster.v2.f32 {%0, %1}, [p];\n}"
                 : "=f"(v.x), "=f"(v.y)
                 : "r"(addr), "r"(rank)
                 : "memory");
    return v;
}
LLMDIY_DEV float4 ta_peer_f4(uint32_t addr, uint32_t rank) {
    float4 v;
    asm volatile(
        "{\n .reg .b32 p;\n mapa.shared::cluster.u32 p, %4, %5;\n ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [p];\n}"
        : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
        : "r"(addr), "r"(rank)
        : "memory");
    return v;
}
LLMDIY_DEV void ta_store4(half* dst, const float4& v, float scale) {
    const half2 y0 = __floats2half2_rn(v.x * scale, v.y * scale), y1 = __floats2half2_rn(v.z * scale, v.w * scale);
    uint2 u;
    u.x = *reinterpret_cast<const uint32_t*>(&y0);
    u.y = *reinterpret_cast<const uint32_t*>(&y1);
    *reinterpret_cast<uint2*>(dst) = u;
}
LLMDIY_DEV void ta_store8(float* dst, const float* v) {  // 32 bytes, a whole sector
    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                 "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                 : "memory");
}
LLMDIY_DEV bool elect_one() {  // one lane of a converged warp
    uint32_t p;
    asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}" : "=r"(p));
    return p != 0;
}
LLMDIY_DEV void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
LLMDIY_DEV uint32_t ta_pack(float lo, float hi) {
    const half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
LLMDIY_DEV float ta_ex2(float x) {  // 2^x (2^-inf = 0)
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The slow part of a wait, out of line: the loops that wait for every tile have to stay short, since each CTA's
// few warps run their code straight through once a tile and instruction fetch sets their pace.
__device__ __noinline__ bool ta_wait_slow(uint64_t* bar, uint32_t parity, const volatile int* fail) {
    return mbar_wait(bar, parity, fail);
}
LLMDIY_DEV bool ta_wait(uint64_t* bar, uint32_t parity, const volatile int* fail) {
    return (kSpinLimit && mbar_try_wait(bar, parity)) || ta_wait_slow(bar, parity, fail);
}
// Two fp32 values at once
LLMDIY_DEV uint64_t ta_f2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
LLMDIY_DEV void ta_split(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
LLMDIY_DEV uint64_t ta_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
LLMDIY_DEV uint64_t ta_add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
LLMDIY_DEV uint64_t ta_sub2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
LLMDIY_DEV float ta_max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
LLMDIY_DEV float ta_ex2v(float x) {  // as ta_ex2, issued where it stands
    float y;
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kTaScaleLog2 = 1.4426950408889634f * 0.08838834764831845f;  // log2(e) / sqrt(128)
// Probabilities are formed as 2^(x - m + kTaRaise), o and l alike, which divides out. A row's reference m stays within
// 2^kTaGrow of its maximum, so they reach 2^15 at most (7 - m may round to 8 - m), and of fp16's range below 1 as much as
// can be is left to the small ones: beside a key that takes nearly all the weight but has a small value, the output is
// made of those. Relative to the largest the rounding is 2^-32, where it was 2^-25 without (keys at 2^-24.6 of it were
// 52% off).
// The exponent is a rounded product, as m is one, and then a sum, and what m is compared by is a difference: both are exact
// near the maximum whatever the scores' size (in one fused operation the product's rounding error is left over, which
// passes fp16 from scores of 2^24 doublings on; a packed product and sum are made into one, a packed fma and a sum are not).
constexpr float kTaRaise = 7.f, kTaGrow = 7.f;

// add[e] += p v[dim0 + e] of the tree rows base + bit that `hit` names, for one query row (out of line: rare).
__device__ __noinline__ void ta_add_bad(const TaArgs& a, uint64_t hit, int b, int node, int base, int kvh, int h,
                                        int dim0, float nm, float* add) {
    for (; hit; hit &= hit - 1) {
        const int kn = base + __ffsll((long long)hit) - 1;
        const half* kr = a.TK + (((size_t)b * a.N + kn) * a.KV + kvh) * kTaDim;
        const half* vr = a.TV + (((size_t)b * a.N + kn) * a.KV + kvh) * kTaDim;
        const half* qr = a.Q + ((size_t)b * a.N + node) * a.ldq + h * kTaDim;
        float d = 0.f;
        for (int e = 0; e < kTaDim; ++e) d = __fmaf_rn(h2f(qr[e]), h2f(kr[e]), d);
        const float p = ta_ex2(__fadd_rn(__fmul_rn(d, kTaScaleLog2), nm));
        for (int e = 0; e < 32; ++e) add[e] = __fmaf_rn(p, h2f(vr[dim0 + e]), add[e]);
    }
}

template <int QR, int KS, int VS, bool DIRECT>
__global__ void __launch_bounds__(kTaThreads, kTaCtasPerSm)
    tree_attn_k(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap ttk,
                const __grid_constant__ CUtensorMap ttv, const __grid_constant__ TaArgs a, int* err) {
    using Smem = TaSmem<QR, KS, VS>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Smem& s = *reinterpret_cast<Smem*>(smem_raw);
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // (uniform for the compiler)
    const int G = a.H / a.KV;
    if (warp == 4 && lane == 0) {  // the thread that issues the copies: it need not wait for the others
        prefetch_tmap(&tq);
        prefetch_tmap(&tk);
        prefetch_tmap(&tv);
        prefetch_tmap(&ttk);
        prefetch_tmap(&ttv);
        mbar_init(&s.q_full, 1);
        mbar_init(&s.q_empty, 1);
        for (int i = 0; i < KS; ++i) {
            mbar_init(&s.k_full[i], 1);
            mbar_init(&s.k_empty[i], 1);
        }
        for (int i = 0; i < VS; ++i) {
            mbar_init(&s.v_full[i], 1);
            mbar_init(&s.v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s.s_full[i], 1);
            mbar_init(&s.p_full[i], 4);
            mbar_init(&s.o_done[i], 1);
        }
        mbar_init(&s.drain[0], 1);
        mbar_init(&s.drain[1], 1);
        s.fail = 0;
        mbar_fence_init();
        fence_async_smem();
    }
    if (warp == 0) {
        tmem_alloc(&s.tmem_base, kTaCols);
        tmem_relinquish();
    }
    pdl_wait();  // nothing in global memory has been touched before this
    pdl_launch_dependents();
    TaCursor c;
    c.left = 0;
    const int C = DIRECT ? (int)gridDim.x : 1, rank = DIRECT ? (int)blockIdx.x : 0;  // the unit's cluster
    // Flat: the M tiles of a kv head go to neighbouring CTAs at the same tiles, so that the second one to read a K/V
    // tile finds it in L2.
    const int mtile = DIRECT ? (int)blockIdx.y % a.mt : (int)blockIdx.x % a.mt, m0 = mtile * a.npt;
    if (DIRECT) {
        c.b = blockIdx.z;
        c.unit = blockIdx.y / a.mt;
        ta_shape(a, c.b, c.n, c.L, c.tiles, c.units);
        if (m0 < c.n) {
            // The unit's last tiles (the cache's tail, the tree) take up to two tiles longer: the last CTAs get that many
            // fewer where the others have as many.  16 x 17 tiles: 11.0 us with equal shares, 9.8 so; with 2 or 5
            // tiles in all equal shares are better (6.9 and 8.2 us against 7.0 and 8.4).
            const int span = c.tiles + min(2, (c.tiles - 1) / C);
            const int t0 = min(span * rank / C, c.tiles), t1 = min(span * (rank + 1) / C, c.tiles);
            c.at = kTaUnitCost + t0;
            c.left = t1 - t0;
        }
    } else {
        const TaDeal deal(ta_total(a, lane), a.W);
        const int w = blockIdx.x / a.mt;
        if (w < deal.W) {
            const int f = deal.start(w);
            c.left = deal.start(w + 1) - f;
            (void)ta_locate(a, f, lane, c);
        }
    }
    const bool work = c.left > 0;
    auto seg = [&](int& t0) { return m0 < c.n ? c.seg(t0) : 0; };  // (a tree may end before this M tile)
    auto warp_wait = [&](uint64_t* bar, uint32_t parity) -> bool {  // one answer for the warp
        return __all_sync(0xffffffffu, ta_wait(bar, parity, &s.fail));
    };
    if (warp != 4) {  // (the producer comes later)
        tc_fence_before();
        named_bar_sync(1, kTaThreads);
        tc_fence_after();
    } else {
        __syncwarp();
        named_bar_arrive(1, kTaThreads);
    }
    // S(j) at tmem + 64 * (j & 1); P(j) takes its place, the low terms 32 columns behind the high ones
    const uint32_t tmem = warp != 4 ? s.tmem_base : 0, tO = tmem + 128;

    if (warp == 4 && work) {
        if (lane == 0) {
            // ---------------- producer: tile j's K into stage j % KS, its V into stage j % VS
            const uint64_t pol = l2_policy_evict_first();
            uint32_t kn = 0, vn = 0, unit_no = 0;  // K tiles, V tiles and units' queries issued
            bool ok = true;
            auto load = [&](half (*dst)[kTaKeys * 64], const CUtensorMap* cache, const CUtensorMap* tree, int kvh, int t,
                            int tc, int row0, uint64_t* bar) {
                mbar_arrive_expect_tx(bar, kTaTileBytes);
                if (t < tc) {
                    const int y = row0 + t * kTaKeys;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (a.evict_first) tma_load_2d_hint(dst[x], cache, kvh * kTaDim + 64 * x, y, bar, pol);
                        else tma_load_2d(dst[x], cache, kvh * kTaDim + 64 * x, y, bar);
                    }
                } else {
                    const int y = c.b * a.N + (t - tc) * kTaKeys;
#pragma unroll
                    for (int x = 0; x < 2; ++x) tma_load_2d(dst[x], tree, kvh * kTaDim + 64 * x, y, bar);
                }
            };
            while (ok && c.left > 0) {
                const int kvh = c.unit;
                int t0;
                const int tc = (c.L + kTaKeys - 1) / kTaKeys, cnt = seg(t0);
                if (!DIRECT && cnt <= 0) {
                    c.next(a);
                    continue;
                }
                const int row0 = c.L ? ta_slot(a, c.b) * a.slot_rows : 0;
                auto load_q = [&]() -> bool {
                    if (unit_no && !ta_wait(&s.q_empty, (unit_no - 1) & 1, &s.fail)) return false;
                    mbar_arrive_expect_tx(&s.q_full, (uint32_t)(a.rows * kTaDim * 2));
                    tma_load_3d(s.q[0], &tq, 0, kvh * G, c.b * a.N + m0, &s.q_full);
                    tma_load_3d(s.q[1], &tq, 64, kvh * G, c.b * a.N + m0, &s.q_full);
                    ++unit_no;
                    return true;
                };
                const bool first_unit = unit_no == 0;
                if (first_unit) (void)load_q();
                for (int t = t0; t < t0 + cnt; ++t) {
                    if (kn >= KS && !ta_wait(&s.k_empty[kn % KS], (kn / KS - 1) & 1, &s.fail)) { ok = false; break; }
                    load(s.k[kn % KS], &tk, &ttk, kvh, t, tc, row0, &s.k_full[kn % KS]);
                    ++kn;
                    if (vn >= VS && !ta_wait(&s.v_empty[vn % VS], (vn / VS - 1) & 1, &s.fail)) { ok = false; break; }
                    load(s.v[vn % VS], &tv, &ttv, kvh, t, tc, row0, &s.v_full[vn % VS]);
                    ++vn;
                    // a later unit's queries take the place of the last one's when its S are done: its first
                    // tile is under way by then
                    if (t == t0 && !first_unit && !load_q()) { ok = false; break; }
                }
                if (DIRECT) break;
                if (ok) c.next(a);
            }
            // the last copies land in this CTA's shared memory: they have before it exits, whatever happens
            for (uint32_t i = kn > KS ? kn - KS : 0; i < kn; ++i) mbar_drain(&s.k_full[i % KS], (i / KS) & 1);
            for (uint32_t i = vn > VS ? vn - VS : 0; i < vn; ++i) mbar_drain(&s.v_full[i % VS], (i / VS) & 1);
            if (unit_no) mbar_drain(&s.q_full, (unit_no - 1) & 1);
            if (!ok) s.fail = 1;
        }
        __syncwarp();
    } else if (warp == 5 && work) {
        // ---------------- S(j) = Q K(j)^T, then release K(j)'s stage (and Q after a unit's last tile)
        constexpr uint32_t idS = umma_idesc_f16_f32(kTaRows, kTaKeys, false);
        // descriptors of the first stages; the start address field counts 16 bytes
        const uint64_t qd = umma_desc_sw128(smem_u32(s.q[0])), kd = umma_desc_sw128(smem_u32(s.k[0][0]));
        const bool lead = elect_one();
        uint32_t j = 0, st = 0, ph = 0, unit_no = 0;
        bool ok = true;
        while (ok && c.left > 0) {
            int t0;
            const int cnt = seg(t0);
            for (int i = 0; i < cnt; ++i, ++j) {
                if (i == 0 && !warp_wait(&s.q_full, unit_no++ & 1)) { ok = false; break; }
                // S(j) takes the place of P(j-2) when the product that reads it is complete
                if (j >= 2 && !warp_wait(&s.o_done[j & 1], ((j - 2) >> 1) & 1)) { ok = false; break; }
                if (!warp_wait(&s.k_full[st], ph)) { ok = false; break; }
                tc_fence_after();
                const uint64_t kj = kd + st * (kTaTileBytes / 16);
                if (lead) {
#pragma unroll
                    for (int kk = 0; kk < kTaDim / 16; ++kk)
                        umma_f16(tmem + 64 * (j & 1), qd + ((kk >> 2) * (QR * 128) + 32 * (kk & 3)) / 16,
                                 kj + ((kk >> 2) * 8192 + 32 * (kk & 3)) / 16, idS, kk != 0 ? 1u : 0u);
                    umma_commit(&s.s_full[j & 1]);
                    umma_commit(&s.k_empty[st]);
                    if (i + 1 == cnt) umma_commit(&s.q_empty);
                }
                __syncwarp();
                if (++st == KS) {
                    st = 0;
                    ph ^= 1;
                }
            }
            if (DIRECT) break;
            c.next(a);
        }
        if (!ok) s.fail = 1;
        __syncwarp();
    } else if (warp == 6 && work) {
        // ---------------- O (+)= P(j) V(j), then release V(j)'s stage
        constexpr uint32_t idO = umma_idesc_f16_f32(kTaRows, kTaDim, true);
        const uint64_t vd = umma_desc_sw128_mn(smem_u32(s.v[0][0]), 8192, 1024);
        const bool lead = elect_one();
        uint32_t j = 0, st = 0, ph = 0;
        bool ok = true;
        while (ok && c.left > 0) {
            int t0;
            const int cnt = seg(t0);
            for (int i = 0; i < cnt; ++i, ++j) {
                if (!warp_wait(&s.v_full[st], ph)) { ok = false; break; }
                if (!warp_wait(&s.p_full[j & 1], (j >> 1) & 1)) { ok = false; break; }
                tc_fence_after();
                const uint64_t vj = vd + st * (kTaTileBytes / 16);
                if (lead) {
#pragma unroll
                    for (int kk = 0; kk < kTaKeys / 8; ++kk)  // both terms against the same V
                        umma_f16_tmem_a(tO, tmem + 64 * (j & 1) + 8 * kk, vj + 2048 * (kk & 3) / 16, idO, i == 0 && kk == 0 ? 0u : 1u);
                    umma_commit(&s.v_empty[st]);
                    umma_commit(&s.o_done[j & 1]);  // last: the rows end the CTA when they have seen it
                }
                __syncwarp();
                if (++st == VS) {
                    st = 0;
                    ph ^= 1;
                }
            }
            if (DIRECT) break;
            c.next(a);
        }
        if (!ok) s.fail = 1;
        __syncwarp();
    } else if (warp < 4 && work) {
        // ---------------- rows
        const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
        const int r = tid, words = (a.N + 63) / 64;
        uint32_t j = 0;
        int slot_no = 0, tree_units = 0;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        while (ok && c.left > 0) {
            const int kvh = c.unit;
            int t0;
            const int tc = (c.L + kTaKeys - 1) / kTaKeys, cnt = seg(t0);
            if (!DIRECT && cnt <= 0) {
                c.next(a);
                slot_no = 1;
                continue;
            }
            const int node = m0 + r / G, g = r - (r / G) * G;
            const bool live = r < a.rows && node < c.n;
            const bool warp_live = warp * 32 < min(a.rows, (c.n - m0) * G);
            const uint64_t* mrow = a.mask + ((size_t)c.b * a.N + (live ? node : 0)) * words;
            const int tt0 = max(t0 - tc, 0);  // first tree tile of this segment, if any
            const int plain = c.L / kTaKeys;  // the tiles before this one are full cache tiles
            uint64_t word = live && t0 + cnt > tc ? mrow[tt0] : 0;
            m = -INFINITY;
            l = 0.f;
            for (int t = t0; t < t0 + cnt; ++t, ++j) {
                uint64_t seen = ~0ull;
                if (__builtin_expect(t >= plain, 0)) {
                    const bool tree = t >= tc;
                    const int tt = t - tc;
                    const int nv = tree ? min(kTaKeys, c.n - tt * kTaKeys) : min(kTaKeys, c.L - t * kTaKeys);
                    if (nv < kTaKeys) seen = (1ull << nv) - 1;
                    if (tree) {
                        seen &= word;
                        if (live && t + 1 < t0 + cnt) word = mrow[tt + 1];
                    }
                    // V rows that must not enter the product: past the end, or (tree) not finite
                    if (!warp_wait(&s.v_full[j % VS], (j / VS) & 1)) { ok = false; break; }
                    // (this warp's 16 rows; a row is two runs of eight 16-byte pieces)
                    uint32_t bad16 = 0;
#pragma unroll
                    for (int it = 0; it < 8; ++it) {
                        const int row = warp * 16 + it * 2 + (lane >> 4);
                        uint4* piece = reinterpret_cast<uint4*>(s.v[j % VS][(lane >> 3) & 1]) + row * 8 + (lane & 7);
                        const uint4 y = *piece;
                        auto odd = [](uint32_t w) { return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u; };
                        const bool out = row >= nv;
                        const unsigned hit = __ballot_sync(
                            0xffffffffu, tree && !out && (odd(y.x) || odd(y.y) || odd(y.z) || odd(y.w)));
                        const bool mine = hit & (lane < 16 ? 0xffffu : 0xffff0000u);
                        if (out || mine) *piece = make_uint4(0u, 0u, 0u, 0u);
                        bad16 |= (uint32_t)((hit & 0xffffu) != 0) << (2 * it) | (uint32_t)((hit >> 16) != 0) << (2 * it + 1);
                    }
                    if (tree && lane == 0) s.bad[tree_units & 1][tt][warp] = (uint16_t)bad16;
                    fence_async_smem();
                }
                if (!warp_wait(&s.s_full[j & 1], (j >> 1) & 1)) { ok = false; break; }
                if (warp_live) {
                    tc_fence_after();
                    const uint32_t pt = tmem + 64 * (j & 1) + lane_off;  // S(j), then P(j)
                    float x[kTaKeys];
#pragma unroll
                    for (int q = 0; q < kTaKeys; q += 16)
                        tmem_ld16(pt + q, reinterpret_cast<uint32_t*>(x + q));
                    tmem_ld_wait();
                    if (__builtin_expect(t >= plain, 0)) {
                        const uint32_t lo = (uint32_t)seen, hi = (uint32_t)(seen >> 32);
#pragma unroll
                        for (int q = 0; q < kTaKeys; ++q)
                            x[q] = ((q < 32 ? lo : hi) & (1u << (q & 31))) ? x[q] : -INFINITY;
                    }
                    float mx[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = ta_max3(x[3 * e], x[3 * e + 1], x[3 * e + 2]);
#pragma unroll
                    for (int q = 12; q < 60; q += 2) mx[(q >> 1) & 3] = ta_max3(mx[(q >> 1) & 3], x[q], x[q + 1]);
                    const float top = ta_max3(ta_max3(mx[0], x[60], x[61]), ta_max3(mx[1], x[62], x[63]),
                                              fmaxf(mx[2], mx[3])) * kTaScaleLog2;
                    const bool grow = live && top - m > kTaGrow;  // (m = -inf at first; a NaN maximum leaves m)
                    if (__builtin_expect(t != t0 && __any_sync(0xffffffffu, grow), 0)) {
                        // rescale O, complete through PV(j-1) (the whole warp: TMEM moves 32 rows at a time)
                        if (!warp_wait(&s.o_done[(j - 1) & 1], ((j - 1) >> 1) & 1)) { ok = false; break; }
                        tc_fence_after();
                        const float f = grow ? exp2f(m - top) : 1.f;  // m = -inf: 0
#pragma unroll 1
                        for (int q = 0; q < kTaDim; q += 16) {
                            uint32_t o[16];
                            tmem_ld16(tO + lane_off + q, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st16(tO + lane_off + q, o);
                        }
                        tmem_st_wait();
                        l *= f;
                    }
                    if (grow) m = top;
                    const float nm = m == -INFINITY ? 0.f : kTaRaise - m;  // nothing seen yet: every p is 2^-inf = 0
                    const uint64_t scale2 = ta_f2(kTaScaleLog2, kTaScaleLog2), nm2 = ta_f2(nm, nm);
                    uint64_t ls[2] = {0, 0};
                    // Sixteen keys at a time, the exponentials of one group ahead of the sums and the rounding of the
                    // last (in this order: a sum right behind its exponentials waits for them)
                    float e[2][16];
                    uint32_t pk[16];
                    auto exps = [&](int q0) {
                        float* to = e[(q0 >> 4) & 1];
#pragma unroll
                        for (int q = 0; q < 16; q += 2) {
                            float a0, a1;
                            ta_split(ta_add2(ta_fma2(ta_f2(x[q0 + q], x[q0 + q + 1]), scale2, 0), nm2), a0, a1);
                            to[q] = ta_ex2v(a0);
                            to[q + 1] = ta_ex2v(a1);
                        }
                    };
                    auto take = [&](int q0) {
                        const float* from = e[(q0 >> 4) & 1];
#pragma unroll
                        for (int q = 0; q < 16; q += 2) {
                            ls[(q >> 1) & 1] = ta_add2(ls[(q >> 1) & 1], ta_f2(from[q], from[q + 1]));
                            const uint32_t hi = ta_pack(from[q], from[q + 1]);
                            const float2 h = __half22float2(*reinterpret_cast<const half2*>(&hi));
                            float l0, l1;
                            ta_split(ta_sub2(ta_f2(from[q], from[q + 1]), ta_f2(h.x, h.y)), l0, l1);
                            pk[q / 2] = hi;
                            pk[8 + q / 2] = ta_pack(l0, l1);
                        }
                        tmem_st8(pt + q0 / 2, pk);
                        tmem_st8(pt + 32 + q0 / 2, pk + 8);
                    };
                    exps(0);
                    exps(16);
                    take(0);
                    exps(32);
                    take(16);
                    exps(48);
                    take(32);
                    take(48);
                    float l0, l1;
                    ta_split(ta_add2(ls[0], ls[1]), l0, l1);
                    l += l0 + l1;
                    tmem_st_wait();
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&s.p_full[j & 1]);
            }
            if (!ok) break;
            // ---------------- the unit's (or its part's) output
            if (!warp_wait(&s.o_done[(j - 1) & 1], ((j - 1) >> 1) & 1)) { ok = false; break; }
            tc_fence_after();
            const bool whole = cnt == c.tiles && C == 1;
            // a part of a unit goes to the workspace, or (direct) to shared memory: Q, K and V are done with
            float* own = reinterpret_cast<float*>(s.k[0][0]) + tid * kTaDim;
            const bool any_tree = t0 + cnt > tc;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const size_t at = (size_t)(blockIdx.x * 2 + slot_no) * a.rows + r;
            half* dst = a.O + ((size_t)c.b * a.N + node) * a.ldo + (kvh * G + g) * kTaDim;
            float* pdst = a.part + at * kTaDim;
            if (warp_live) {
                // non-finite V rows that this part's rows left out of PV (rare)
                bool any_bad = false;
                if (any_tree)
                    for (int tt = tt0; tt < t0 + cnt - tc; ++tt)
                        any_bad |= *reinterpret_cast<volatile uint64_t*>(s.bad[tree_units & 1][tt]) != 0;
#pragma unroll 1
                for (int q = 0; q < kTaDim; q += 32) {
                    float v[32];
                    __syncwarp();
                    tmem_ld16(tO + lane_off + q, reinterpret_cast<uint32_t*>(v));
                    tmem_ld16(tO + lane_off + q + 16, reinterpret_cast<uint32_t*>(v + 16));
                    tmem_ld_wait();
                    if (__builtin_expect(any_bad && live, 0)) {
                        float add[32];
                        for (int e = 0; e < 32; ++e) add[e] = 0.f;
                        for (int tt = tt0; tt < t0 + cnt - tc; ++tt)
                            ta_add_bad(a, *reinterpret_cast<volatile uint64_t*>(s.bad[tree_units & 1][tt]) & mrow[tt], c.b, node,
                                       tt * 64, kvh, kvh * G + g, q, m == -INFINITY ? 0.f : kTaRaise - m, add);
                        for (int e = 0; e < 32; ++e) v[e] += add[e];
                    }
                    if (!live) continue;
                    if (whole) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] *= inv;
#pragma unroll
                        for (int e = 0; e < 32; e += 8) *reinterpret_cast<uint4*>(dst + q + e) = pack8(v + e);
                    } else if (DIRECT) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            // (16-byte pieces of a row turned by the row: 32 rows' stores meet different banks)
                            float* to = own + (((q + e) / 4) ^ lane) * 4;
                            *reinterpret_cast<float4*>(to) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) ta_store8(pdst + q + e, v + e);
                    }
                }
                if (live && !whole && !DIRECT)
                    *reinterpret_cast<float2*>(a.part + (size_t)a.W * a.mt * 2 * a.rows * kTaDim + at * 2) = make_float2(m, l);
            }
            tc_fence_before();  // O has been read: the next unit's first PV may overwrite it
            if (any_tree) ++tree_units;
            slot_no = 1;
            if (DIRECT) break;
            c.next(a);
        }
        if (!ok) s.fail = 1;
        if (DIRECT && C > 1) reinterpret_cast<float2*>(s.q[0])[tid] = make_float2(m, l);
    } else if (warp < 4 && DIRECT && C > 1) {
        reinterpret_cast<float2*>(s.q[0])[tid] = make_float2(-INFINITY, 0.f);  // no tile for this CTA
    }
    if (DIRECT && C > 1) {
        // ---------------- the cluster's parts of the unit joined, each CTA a share of the rows
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (m0 < c.n) {
            const int kvh = c.unit;
            const int live = min(a.rows, (c.n - m0) * G), r1 = live * (rank + 1) / C;
            const uint32_t ml = smem_u32(s.q[0]), oo = smem_u32(s.k[0][0]);
            // two rows to a warp, half a warp each (C <= 16)
            const int gl = lane & 15;
            for (int r0 = live * rank / C + 2 * warp; r0 < r1; r0 += 2 * (kTaThreads / 32)) {
                const int r = min(r0 + (lane >> 4), r1 - 1);  // (the last row twice where they are odd)
                const float2 w = gl < C ? ta_peer_f2(ml + r * 8, gl) : make_float2(-INFINITY, 0.f);
                float M = w.x;
#pragma unroll
                for (int o = 8; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
                const unsigned parts = __ballot_sync(0xffffffffu, w.x != -INFINITY || w.y != w.y) >> (lane & 16);
                // nothing seen by a part: weight 0 (its l is 0, or NaN, which stays)
                const float f = w.x == -INFINITY ? (w.y == w.y ? 0.f : 1.f) : exp2f(w.x - M);
                float L = w.y * f;
#pragma unroll
                for (int o = 8; o >= 1; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
                float4 acc[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                for (int k = 0; k < C; ++k) {
                    const float fk = __shfl_sync(0xffffffffu, f, k, 16);
                    if ((parts >> k) & 1) {  // (a part that saw nothing has no o)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float4 y = ta_peer_f4(oo + r * (kTaDim * 4) + (((gl + 16 * e) ^ (r & 31)) * 16), k);
                            acc[e].x = __fmaf_rn(fk, y.x, acc[e].x);
                            acc[e].y = __fmaf_rn(fk, y.y, acc[e].y);
                            acc[e].z = __fmaf_rn(fk, y.z, acc[e].z);
                            acc[e].w = __fmaf_rn(fk, y.w, acc[e].w);
                        }
                    }
                }
                const int node = m0 + r / G, h = kvh * G + r - (r / G) * G;
                half* dst = a.O + ((size_t)c.b * a.N + node) * a.ldo + h * kTaDim + gl * 4;
                if (r0 + (lane >> 4) < r1)
#pragma unroll
                    for (int e = 0; e < 2; ++e) ta_store4(dst + 64 * e, acc[e], L == 0.f ? 0.f : 1.f / L);
            }
        }
        // The peers have read this CTA's part (relaxed: nothing written has to be seen).
        asm volatile("barrier.cluster.arrive.relaxed.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    if (__builtin_expect(*reinterpret_cast<volatile int*>(&s.fail), 0)) {
        if (tid == 0) atomicExch(err, 1);
        // whichever warp gave up: every MMA issued completes before the TMEM is freed and the CTA exits
        if (work && (warp == 5 || warp == 6)) {
            if (elect_one()) umma_commit(&s.drain[warp - 5]);
            mbar_drain(&s.drain[warp - 5], 0);
            __syncwarp();
        }
        __syncthreads();
    }
    if (warp == 0) tmem_dealloc(tmem, kTaCols);
}

// Flat: joins the partials of the units that were cut.  Block w - 1 looks at the cut before CTA w: if it
// parts a unit's tiles, the blocks of that unit's cuts share its rows, two rows to a warp and eight partials' loads
// in flight (with a warp per row, one row after the other, joining 64-row units took 20 us): of a row's sixteen
// lanes, lane i weighs partials i, i + 16, .., then each sums 8 dims over the partials in order.
constexpr int kTaMergeWarps = 16;

__global__ void __launch_bounds__(kTaMergeWarps * 32) tree_merge_k(const __grid_constant__ TaArgs a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w = blockIdx.x / a.mt + 1, m0 = blockIdx.x % a.mt * a.npt;
    // Every thread waits for the attention kernel, also where there is nothing to join: this grid must not be
    // over before that one is.  (That one triggers this launch only when it has itself seen the kernels before it
    // complete, so the lengths may be read ahead of the wait.)
    const TaDeal deal(ta_total(a, lane), a.W);
    TaCursor c;
    int f0 = 0;
    const bool cut = w < deal.W;
    if (cut) f0 = ta_locate(a, deal.start(w), lane, c);
    pdl_wait();
    pdl_launch_dependents();
    if (!cut || c.at <= kTaUnitCost || m0 >= c.n) return;  // no tile of the unit before the cut
    const int w0 = deal.owner(f0 + kTaUnitCost), w1 = deal.owner(f0 + kTaUnitCost + c.tiles - 1);
    // the first CTA's part of this unit is its first segment only when its range does not start before the unit
    const int mtile = blockIdx.x % a.mt;
    const int later = deal.start(w0) < f0 ? 1 : 0;
    auto part = [&](int k) { return (k * a.mt + mtile) * 2 + (k == w0 ? later : 0); };  // of CTA (k, mtile)
    const int G = a.H / a.KV, kvh = c.unit;
    const int live = min(a.rows, (c.n - m0) * G), share = w - w0 - 1, shares = w1 - w0;
    const int r1 = live * (share + 1) / shares;
    const float2* ml = reinterpret_cast<const float2*>(a.part + (size_t)a.W * a.mt * 2 * a.rows * kTaDim);
    const int gl = lane & 15;
    for (int q = live * share / shares + warp * 2; q < r1; q += kTaMergeWarps * 2) {
        const int r = min(q + (lane >> 4), r1 - 1);  // (lanes past the share repeat its last row)
        float M = -INFINITY;
        for (int k = w0 + gl; k <= w1; k += 16) M = fmaxf(M, ld_l2_f2(ml + (size_t)part(k) * a.rows + r).x);
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        float Ls = 0.f;
        float4 acc[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c0 = w0; c0 <= w1; c0 += 16) {
            float f = 0.f;
            if (c0 + gl <= w1) {
                const float2 y = ld_l2_f2(ml + (size_t)part(c0 + gl) * a.rows + r);
                // nothing seen by a part: weight 0 (its l is 0, or NaN, which stays)
                f = y.x == -INFINITY ? (y.y == y.y ? 0.f : 1.f) : exp2f(y.x - M);
                Ls += y.y * f;
            }
            const int cnt = min(16, w1 - c0 + 1);
#pragma unroll 8
            for (int i = 0; i < cnt; ++i) {
                const float fk = __shfl_sync(0xffffffffu, f, i, 16);
                const float4* src = reinterpret_cast<const float4*>(a.part + ((size_t)part(c0 + i) * a.rows + r) * kTaDim) + gl;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float4 y = ld_l2_f4(src + 16 * e);
                    acc[e].x = __fmaf_rn(fk, y.x, acc[e].x);
                    acc[e].y = __fmaf_rn(fk, y.y, acc[e].y);
                    acc[e].z = __fmaf_rn(fk, y.z, acc[e].z);
                    acc[e].w = __fmaf_rn(fk, y.w, acc[e].w);
                }
            }
        }
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) Ls += __shfl_xor_sync(0xffffffffu, Ls, o);
        const int node = m0 + r / G, h = kvh * G + r - (r / G) * G;
        half* dst = a.O + ((size_t)c.b * a.N + node) * a.ldo + h * kTaDim + gl * 4;
        if (q + (lane >> 4) < r1)
#pragma unroll
            for (int e = 0; e < 2; ++e) ta_store4(dst + 64 * e, acc[e], Ls == 0.f ? 0.f : 1.f / Ls);
    }
}

#include "tree_attn_few.cuh"

// ------------------------------------------------------------------ host
int ta_sms() {
    static std::atomic<int> known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    int n = known[dev];
    if (!n) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
        known[dev] = n;
    }
    return n;
}

struct TaPlan {
    int G, npt, rows, mt, W;  // W: flat CTAs per M tile
    int cluster;  // direct: CTAs per unit (0: flat)
    int few;      // CTAs per unit of the kernel for few rows (0: not that one)
    bool ok;
    size_t floats;  // of the flat partials
};

// The grid and the partials' size; the latter is never smaller for a larger B, N or max_len (same heads), so a
// workspace sized for the largest call serves the others.
TaPlan ta_plan(int B, int N, int H, int KV, int max_len) {
    TaPlan p = {};
    p.ok = B > 0 && B <= 65535 && N > 0 && N <= LLMDIY_TREE_MAX_NODES && KV > 0 && H >= KV && H <= 1024 && H % KV == 0 &&
           H / KV <= kTaMaxGroup && max_len >= 0;
    if (!p.ok) return p;
    p.G = H / KV;
    p.npt = std::min(kTaRows / p.G, N);
    p.rows = p.G * p.npt;
    p.mt = (N + p.npt - 1) / p.npt;
    const long long tiles = ((long long)max_len + kTaKeys - 1) / kTaKeys + (N + kTaKeys - 1) / kTaKeys;
    const long long units = (long long)B * KV * p.mt;
    p.ok = units * (tiles + kTaUnitCost) <= 0x7fffffffLL;
    const int slots = std::max(kTaCtasPerSm * ta_sms(), p.mt);
    // Flat CTAs have four tiles or more, and a unit is cut into sqrt(2 tiles) parts at most: joining costs about half as much
    // a part as the products a tile.  1 unit of 1025 tiles, 128 rows: 49.4 us with sqrt(tiles) parts, 45.6 so,
    // 47.3 with sqrt(5 tiles), 106 with 296.
    const double parts = std::sqrt(2.0 * (double)tiles);
    p.W = (int)std::max<long long>(
        1, std::min<long long>({slots / p.mt, units / p.mt * tiles / 4, (long long)((double)(units / p.mt) * parts)}));
    p.floats = (size_t)std::min<long long>(slots, units * tiles) * 2 * p.rows * (kTaDim + 2);
    // Units of up to four rows whose CTAs' shares are short go to the kernel for those: the products of a CTA, rows x
    // cache rows, decide.  Measured (this kernel / the one for few rows): 16 units of 1 row over 1023 8.8 / 4.9, over 8192
    // (1024 a CTA) 19.3 / 18.8, over 131072 179 / 240; 2 rows over 4096 (512 a CTA) 13.8 / 13.1, over 8192 19.4 / 22.3; 4 over
    // 1023 9.2 / 7.4, over 4000 (500 a CTA) 13.6 / 19.2; 32 units of 4 over 2048 (256 a CTA) 12.9 / 13.3; 1024 units of 1
    // over up to 300 37.6 / 24.1, over up to 1000 61.7 / 50.1.
    if (p.rows <= kFewRows) {
        const int c = (int)std::max<long long>(1, std::min<long long>({kFewCluster, slots / units, (max_len + 63) / 64}));
        if ((long long)p.rows * ((max_len + c - 1) / c) <= (p.rows <= 2 ? 1024 : 768)) p.few = c;
    }
    // Direct or flat, by what both would take if every sequence were max_len long, in us.  A CTA that runs its chain of
    // products undisturbed needs 0.75 a tile (1.0 with more than 32 rows), and all slots together 1.46 a tile and slot from
    // HBM; a flat call pays for its second launch and for joining W / units partials a row.  Of sequences
    // of different lengths direct waits for the longest, and its clusters do not fill the GPU evenly, so calls with more than
    // kTaDirectTiles tiles a CTA go flat.  Measured (direct / flat), 16 rows: 16 units of 17 tiles 9.3 / 14.5, 2 of 126 12.2 /
    // 18.9, 1024 of up to 33 110 / 118, 256 of up to 66 75 / 59; 8 rows: 16 units of 513 53 / 57, 769 77 / 78, 1025 102 / 96,
    // 2049 201 / 180, 8 of 513 41 / 41, 1025 74 / 62; 64 rows: 16 of 513 58 / 59, 769 85 / 80, 2049 218 / 190; 128 rows: 16 of
    // 514 64 / 66, 1026 120 / 110.
    // CTAs per unit (direct): the tiles of one, the cluster's barriers and its join (rows by 14 a time) against one another, in
    // us.  Clusters of more than two leave gaps: 7/8 of the slots are counted, and where 8 GPCs' SMs do not take all clusters one CTA to an
    // SM, units of many rows slow each other.  Measured with 1 / 2 / 4 / 8 CTAs: 12 units of 3 tiles and 115 rows 9.8 / 11.3 / 9.4 / 9.9;
    // 96 of 4 and 83 rows 10.5 / 12.9 / 19.2 / 30.2; 64 of 6 and 8 rows 10.0 / 9.8 / 8.5 / 16.1; 16 of 33 and 26 rows 29.9 / 19.1 /
    // 12.8 / 11.6; 20 of 28 and 125 rows 32.0 / 22.4 / 15.6 / 16.8 (14.4 with 5).
    int c = 1;
    double best = 1e30;
    for (int k = 1; k <= std::min<long long>(kTaCluster, tiles); ++k) {
        if (units * k > slots || (k > 2 && units * k * 8 > slots * 7LL)) break;
        const bool lone = units <= 8 * (slots / kTaCtasPerSm / 8 / k);
        const double us = std::max(1.0, (double)tiles / k) * (lone || p.rows <= 32 ? 0.75 : 1.1) +
                          (k > 1 ? 0.6 + 0.1 * k + 0.6 * ((p.rows + 14 * k - 1) / (14 * k)) : 0.0);
        if (us < best) {
            best = us;
            c = k;
        }
    }
    // Clusters of 12 or 16 for many tiles, where the units' all run at once: such clusters leave gaps, 21 and 14 of them fit
    // on 148 SMs (16 x 16 CTAs do not, and take 18.3 us against 11.5), so three quarters of the slots are counted.
    // Measured (8 / 16 CTAs), 8 units of 34 tiles 9.7 / 10.2, 2 of 65 12.2 / 9.8, 8 of 129 18.7 / 16.8; (8 / 12), 16
    // of 34 11.4 / 10.4, of 129 24.0 / 19.8.
    if (tiles > 6 * kTaCluster && c == kTaCluster)
        c = units * 16 * 4 <= slots * 3 ? 16 : units * 12 * 4 <= slots * 3 ? 12 : c;
    const double t = (double)((tiles + c - 1) / c), chain = p.rows > 32 ? 1.0 : 0.75, hbm = 1.46 / slots;
    const double flat_ctas = (double)p.W * p.mt;
    const double direct_us = 9.0 + t * std::max(chain, hbm * std::min<double>(slots, units * c));
    const double flat_us = 20.0 + units * tiles / flat_ctas * std::max(chain, hbm * flat_ctas) + 0.12 * flat_ctas / units;
    if (direct_us < flat_us && t <= kTaDirectTiles) p.cluster = c;
    return p;
}

// Query rows as [B * N][H][128] (pitch ldq): box of 64 dims x G heads x npt nodes, 128-byte swizzle.
bool make_query_map(CUtensorMap* m, const void* base, int nodes, int H, int ldq, int G, int npt) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static Encode fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<Encode>(p);
    });
    if (!fn) return false;
    cuuint64_t dims[3] = {(cuuint64_t)kTaDim, (cuuint64_t)H, (cuuint64_t)nodes};
    cuuint64_t strides[2] = {(cuuint64_t)kTaDim * 2, (cuuint64_t)ldq * 2};
    cuuint32_t box[3] = {64u, (cuuint32_t)G, (cuuint32_t)npt};
    cuuint32_t estr[3] = {1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr size_t kTaCtl = 8;  // floats before the partials, which begin on 32 bytes: word 0 is the error word
size_t ta_work_bytes(const TaPlan& p) { return (kTaCtl + p.floats) * sizeof(float); }

template <int QR, int KS, int VS, bool DIRECT>
int ta_launch(const CUtensorMap* m, const TaArgs& a, int* err, dim3 grid, int cluster, cudaStream_t st) {
    auto kern = tree_attn_k<QR, KS, VS, DIRECT>;
    constexpr int bytes = (int)sizeof(TaSmem<QR, KS, VS>);
    static_assert(bytes <= 115712, "two CTAs share an SM");
    static_assert((KS + VS) * kTaTileBytes >= QR * kTaDim * 4, "a part's rows fit over K and V");
    static std::atomic<bool> set[64];  // per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev < 0 || dev >= 64 || !set[dev])) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess && dev >= 0 && dev < 64) set[dev] = true;
    }
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = grid;
    lc.blockDim = dim3(kTaThreads);
    lc.dynamicSmemBytes = bytes;
    lc.stream = st;
    // programmatic serialization: the CTAs set up their barriers and TMEM while the stream's previous kernel ends
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at;
    lc.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&lc, kern, m[0], m[1], m[2], m[3], m[4], a, err);
}

}  // namespace

extern "C" {

size_t llmdiy_tree_attn_work_bytes(int B, int N, int num_heads, int num_kv_heads, int max_len) {
    const TaPlan p = ta_plan(B, N, num_heads, num_kv_heads, max_len);
    return p.ok ? ta_work_bytes(p) : 0;
}

int llmdiy_tree_attn_path(int B, int N, int num_heads, int num_kv_heads, int max_len) {
    const TaPlan p = ta_plan(B, N, num_heads, num_kv_heads, max_len);
    return !p.ok ? -1 : p.few ? 2 : p.cluster ? 1 : 0;
}

int llmdiy_tree_attn(const uint16_t* Q, int ldq, const uint16_t* K, const uint16_t* V, int stride, int slot_rows,
                     int num_slots, const int* slot, const int* len, int max_len, const uint16_t* TK,
                     const uint16_t* TV, const uint64_t* mask, const int* tree_len, int B, int N, int num_heads,
                     int num_kv_heads, uint16_t* O, int ldo, float* work, size_t work_bytes, void* stream) {
    auto a16 = [](const void* p) { return p && (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    const TaPlan p = ta_plan(B, N, num_heads, num_kv_heads, max_len);
    if (!p.ok || !a16(Q) || !a16(K) || !a16(V) || !a16(TK) || !a16(TV) || !a16(O) || !len || !mask ||
        (reinterpret_cast<uintptr_t>(mask) & 7) || !words_aligned(slot, len, tree_len) || ldq < num_heads * kTaDim || (ldq & 7) || ldo < num_heads * kTaDim ||
        (ldo & 7) || stride < num_kv_heads * kTaDim || (stride & 7) || slot_rows <= 0 || num_slots <= 0 ||
        max_len > slot_rows || (long long)num_slots * slot_rows > 0x7fffffffLL || !a16(work) ||
        work_bytes < ta_work_bytes(p))
        return (int)cudaErrorInvalidValue;
    TaArgs a = {};
    a.slot = slot;
    a.len = len;
    a.tree_len = tree_len;
    a.mask = mask;
    a.Q = reinterpret_cast<const half*>(Q);
    a.TK = reinterpret_cast<const half*>(TK);
    a.TV = reinterpret_cast<const half*>(TV);
    a.O = reinterpret_cast<half*>(O);
    a.part = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(work) & ~(uintptr_t)31) + kTaCtl * 4);
    a.B = B;
    a.N = N;
    a.H = num_heads;
    a.KV = num_kv_heads;
    a.ldq = ldq;
    a.ldo = ldo;
    a.slot_rows = slot_rows;
    a.num_slots = num_slots;
    a.max_len = max_len;
    a.rows = p.rows;
    a.npt = p.npt;
    a.mt = p.mt;
    a.W = p.W;
    a.evict_first = p.npt >= N;  // one M tile: every K/V row is read once
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    int* err = reinterpret_cast<int*>(work);
    if (p.few) {
        const half *hk = reinterpret_cast<const half*>(K), *hv = reinterpret_cast<const half*>(V);
        return p.rows == 1   ? few_launch<1, 8>(a, hk, hv, stride, err, p.few, st)
               : p.rows == 2 ? few_launch<2, 8>(a, hk, hv, stride, err, p.few, st)
                             : few_launch<4, 4>(a, hk, hv, stride, err, p.few, st);
    }
    CUtensorMap m[5];
    const int cols = num_kv_heads * kTaDim;
    if (!make_query_map(&m[0], Q, B * N, num_heads, ldq, p.G, p.npt) ||
        !make_kmajor_map(&m[1], K, num_slots * slot_rows, cols, stride, kTaKeys) ||
        !make_kmajor_map(&m[2], V, num_slots * slot_rows, cols, stride, kTaKeys) ||
        !make_kmajor_map(&m[3], TK, B * N, cols, cols, kTaKeys) || !make_kmajor_map(&m[4], TV, B * N, cols, cols, kTaKeys))
        return (int)cudaErrorInvalidValue;
    const bool direct = p.cluster > 0;
    const dim3 grid = direct ? dim3(p.cluster, num_kv_heads * p.mt, B) : dim3(p.W * p.mt);
    const int cluster = std::max(1, p.cluster);
    int rc;
    if (p.rows <= 64)
        rc = direct ? ta_launch<64, 3, 3, true>(m, a, err, grid, cluster, st)
                    : ta_launch<64, 3, 3, false>(m, a, err, grid, cluster, st);
    else
        rc = direct ? ta_launch<128, 3, 2, true>(m, a, err, grid, cluster, st)
                    : ta_launch<128, 3, 2, false>(m, a, err, grid, cluster, st);
    if (rc || direct || p.W < 2) return rc;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((p.W - 1) * p.mt);
    lc.blockDim = dim3(kTaMergeWarps * 32);
    lc.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at;
    lc.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&lc, tree_merge_k, a);
}

int llmdiy_tree_attn_status(const float* work) {
    if (!work) return (int)cudaErrorInvalidValue;
    int h = 0;
    int* word = reinterpret_cast<int*>(const_cast<float*>(work));
    cudaError_t e = cudaMemcpy(&h, word, sizeof(int), cudaMemcpyDeviceToHost);
    if (e != cudaSuccess) return (int)e;
    if (h) cudaMemset(word, 0, sizeof(int));  // the kernels only ever set it
    return h ? -5 : 0;
}

}  // extern "C"
