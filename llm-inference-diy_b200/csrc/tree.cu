// tree.cu — the speculative-decoding operators around the tree attention (include/llmdiy_tree.h):
// bias + rotary positions of a tree's rows, verification of the drafts, and the commit of the
// accepted K/V rows.  No counterpart in the reference, which decodes one token per step.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "llmdiy_tree.h"

using namespace llmdiy;

namespace {

constexpr int kDim = 128;  // head dimension
constexpr int kMaxNodes = LLMDIY_TREE_MAX_NODES;

inline cudaStream_t S(void* s) { return reinterpret_cast<cudaStream_t>(s); }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// (Pointers here carry no __restrict__: a load that the compiler may take for invariant could move ahead of pdl_wait.)
// Launches with programmatic stream serialization: the kernel is set up while the stream's previous one ends, and
// waits (pdl_wait) before it touches global memory.
template <class... P, class... A>
int launch_pdl(void (*kern)(P...), dim3 grid, int threads, cudaStream_t st, A... args) {
    cudaLaunchConfig_t lc = {};
    lc.gridDim = grid;
    lc.blockDim = dim3(threads);
    lc.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at;
    lc.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&lc, kern, static_cast<P>(args)...);
}

LLMDIY_DEV int nodes_of(const int* tree_len, int b, int N) {
    return tree_len ? min(max(tree_len[b], 0), N) : N;
}

// ---------------------------------------------------------------- bias + RoPE
// One CTA per node, bound by the latency of its loads (1536 nodes of 48 heads' rows 7.5 us, 4.2 TB/s of the 6.5 of a copy, in
// one wave and a third: 64 registers let 8 CTAs on an SM, 1184 of those nodes at once).  (y_t, y_{t+64}) turns by
// a = pos * base^(-t/64): the angle is formed and reduced to [-pi, pi] in 64 bits (a position of 10^5 leaves fp32 angles only 2 digits after the point), its sine
// and cosine are then taken in fp32 (absolute error < 2^-21 to angles of 2^24: 2^-23 of the reduced angle's rounding, two
// units of the last place of sine or cosine, 2^-25 of the 64-bit product; the fp16 outputs are rounded by 2^-11).  The 64
// frequencies come as a kernel argument, and the first rows' loads are under way while the angles are computed.
struct RopeFreqs {
    double f[kDim / 2];
};
constexpr int kRopeThreads = 128;  // (1536 nodes: 8.3 us with 256, 7.7 with 128)

__global__ void __launch_bounds__(kRopeThreads)
    tree_rope_k(const half* qkv, const half* bias, const int* depth,
                const int* len, const int* tree_len, int N, int H, int KV,
                const __grid_constant__ RopeFreqs freqs, half* Q, half* TK,
                half* TV) {
    __shared__ float cs[kDim / 2], sn[kDim / 2];
    const int b = blockIdx.y, i = blockIdx.x, tid = threadIdx.x;
    const size_t row = (size_t)b * N + i;
    const half* src = qkv + row * (H + 2 * KV) * kDim;
    // units: 8 threads per rotated head, each 8 pairs (two 16-byte loads), then 8 per value head (the same two loads)
    const int units = (H + 2 * KV) * 8, turned = (H + KV) * 8;
    uint4 a1, a2, c1 = make_uint4(0u, 0u, 0u, 0u), c2 = c1;
    auto fetch = [&](int u) {
        const int at = (u >> 3) * kDim + (u & 7) * 8;
        a1 = ld_once_u4(src + at);
        a2 = ld_once_u4(src + at + 64);
        if (bias) {
            c1 = ld_once_u4(bias + at);
            c2 = ld_once_u4(bias + at + 64);
        }
    };
    pdl_wait();
    pdl_launch_dependents();
    if (tid < units) fetch(tid);
    if (i >= nodes_of(tree_len, b, N)) return;
    if (tid < kDim / 2) {
        const double a = ((double)len[b] + depth[row]) * freqs.f[tid];
        constexpr double kTurn = 6.283185307179586476925;
        const float r = (float)(a - kTurn * rint(a * (1.0 / kTurn)));
        sincosf(r, &sn[tid], &cs[tid]);
    }
    __syncthreads();
    for (int u = tid; u < units;) {
        const int h = u >> 3, t0 = (u & 7) * 8;
        float x1[8], x2[8], b1[8], b2[8];
        unpack8(a1, x1);
        unpack8(a2, x2);
        unpack8(c1, b1);
        unpack8(c2, b2);
        const int next = u + kRopeThreads;
        if (next < units) fetch(next);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x1[e] += b1[e];
            x2[e] += b2[e];
        }
        half* dst = h < H ? Q + (row * H + h) * kDim : (u < turned ? TK : TV) + (row * KV + (h - H) % KV) * kDim;
        if (u < turned) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float c = cs[t0 + e], s = sn[t0 + e], y1 = x1[e], y2 = x2[e];
                x1[e] = y1 * c - y2 * s;
                x2[e] = y2 * c + y1 * s;
            }
        }
        *reinterpret_cast<uint4*>(dst + t0) = pack8(x1);
        *reinterpret_cast<uint4*>(dst + t0 + 64) = pack8(x2);
        u = next;
    }
}

// ---------------------------------------------------------------- verification
// A cluster of C CTAs per sequence.  Every thread walks the tree from shared memory (the tested
// entries p(x_i), q(x_i) of all nodes are fetched at the start, in one round trip); a refused
// child needs the sum of max(0, p - T q) over the row, and the end of the walk its running sum.  The row is cut
// into blocks of 128 entries, dealt contiguously to the cluster's warps (warp k of K: blocks
// [k U / K, (k + 1) U / K)), so the warps' totals in order are a running sum over the row.
//
// What bounds it is the walk: a refusal needs the sum over two rows before the next child can be tried.  V = 151936, in a
// graph: one sequence without a refusal 6.4 us, the first refusal 2.0 more (the draft's row), each further one at the same node 2.5
// to 3, at a new node 4.3 (its rows' loads); with 24 sequences 10.3, 6.9, 6.0 and 9 to 10.  There a round at the same
// node is the 64-bit arithmetic and its conversions on two CTAs' shares an SM, and a fifth of the rows (what does not fit
// kVerHeld) read again.  A chain of 4 takes 7.7 us (one round), 24 trees of 32 nodes 33 (up to five rounds at up to
// two nodes, 29 to 39 MB read).  Tried: blocks held in registers (two fit; 8.8 and 36.5 us), the root's rows fetched into L2 while
// the tree is read (24 trees 38.9 us against 35.5), the weights as two fp32 terms in place of fp64 (37.5 against 36.3).
constexpr int kVerThreads = 512;
constexpr int kVerWarps = kVerThreads / 32;
constexpr int kVerMaxCluster = 14;
constexpr int kVerCtasPerSm = 2;
constexpr int kVerHeld = 6;  // blocks of a warp's share kept in shared memory between rounds (two CTAs share an SM)
constexpr int kVerHeldBytes = kVerWarps * kVerHeld * 2 * 512;

LLMDIY_DEV double positive(double x) { return x > 0.0 ? x : 0.0; }  // NaN counts as 0

// Entries v0 .. v0 + 3 of a row (0 past V); vec: the rows are 16-byte aligned.
LLMDIY_DEV float4 ver_load(const float* row, int v0, int V, bool vec) {
    if (vec && v0 + 3 < V) return *reinterpret_cast<const float4*>(row + v0);
    float4 a;
    a.x = v0 < V ? row[v0] : 0.f;
    a.y = v0 + 1 < V ? row[v0 + 1] : 0.f;
    a.z = v0 + 2 < V ? row[v0 + 2] : 0.f;
    a.w = v0 + 3 < V ? row[v0 + 3] : 0.f;
    return a;
}

// max(0, p - T q) of four entries (T = 0: p, whatever q holds)
LLMDIY_DEV void ver_weights(const float4& p, const float4& q, double T, double* w) {
    w[0] = positive(p.x);
    w[1] = positive(p.y);
    w[2] = positive(p.z);
    w[3] = positive(p.w);
    if (T != 0.0) {
        w[0] = positive(w[0] - T * positive(q.x));
        w[1] = positive(w[1] - T * positive(q.y));
        w[2] = positive(w[2] - T * positive(q.z));
        w[3] = positive(w[3] - T * positive(q.w));
    }
}

// The same into this thread's place in shared memory, without waiting where it can.
LLMDIY_DEV void ver_hold(float4* dst, const float* row, int v0, int V, bool vec) {
    if (vec && v0 + 3 < V)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(row + v0) : "memory");
    else
        *dst = ver_load(row, v0, V, vec);
}

// Eight bytes into the shared memory of CTA `rank` of the cluster, counted by the mbarrier there.
LLMDIY_DEV void ver_send(double* dst, uint64_t* bar, uint32_t rank, double v) {
    uint32_t d, m;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(smem_u32(dst)), "r"(rank));
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(m) : "r"(smem_u32(bar)), "r"(rank));
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(d),
                 "l"(__double_as_longlong(v)), "r"(m)
                 : "memory");
}

LLMDIY_DEV double warp_sum(double x) {
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
    return x;
}

struct VerSmem {
    int parent[kMaxNodes], token[kMaxNodes], child[kMaxNodes], sibling[kMaxNodes];
    double p[kMaxNodes], q[kMaxNodes], u[kMaxNodes];
    double part[2][kVerMaxCluster * kVerWarps];  // the cluster's warp totals, in order (two rounds)
    uint64_t got[2];                             // counts their bytes
    int dead[kMaxNodes];                         // refused tokens of the current node (no draft distribution)
};

__global__ void __launch_bounds__(kVerThreads, kVerCtasPerSm)
    tree_verify_k(const float* target, int ldt, const float* draft, int ldd,
                  const int* token, const int* parent, const int* tree_len,
                  const float* uniform, int N, int V, int vec, int* path,
                  int* accepted, int* next) {
    namespace cg = cooperative_groups;
    __shared__ VerSmem s;
    extern __shared__ __align__(16) uint8_t ver_rows[];  // [warp][block][target, draft][lane] float4
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int b = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const size_t row0 = (size_t)b * N;
    const int U = (V + 127) / 128, K = C * kVerWarps, k = rank * kVerWarps + warp;
    const int u0 = (int)((long long)U * k / K), u1 = (int)((long long)U * (k + 1) / K);
    if (tid == 0) {
        mbar_init(&s.got[0], 1);
        mbar_init(&s.got[1], 1);
        mbar_fence_init();
    }
    cluster.sync();  // every CTA of the cluster runs and has set up its barriers: its shared memory may be written
    pdl_wait();      // nothing in global memory has been touched before this
    pdl_launch_dependents();
    int par = -1, tok = -1;
    if (tid > 0 && tid < N) {  // (in flight together with the tree's size)
        par = parent[row0 + tid];
        tok = token[row0 + tid];
    }
    const int n = nodes_of(tree_len, b, N);
    if (rank == 0)
        for (int i = tid; i < N; i += kVerThreads) path[row0 + i] = -1;
    if (n == 0) {
        if (rank == 0 && tid == 0) { accepted[b] = -1; next[b] = -1; }
        return;  // the whole cluster
    }
    if (tid < n) {
        const bool ok = par >= 0 && par < tid && tok >= 0 && tok < V;
        s.parent[tid] = ok ? par : -1;
        s.token[tid] = tok;
        s.u[tid] = uniform[row0 + tid];
        s.p[tid] = ok ? positive(target[(row0 + par) * ldt + tok]) : 0.0;
        s.q[tid] = ok ? (draft ? positive(draft[(row0 + par) * ldd + tok]) : 1.0) : 0.0;
    }
    __syncthreads();
    if (tid < n) {  // first child and next sibling in index order
        int child = -1, sib = -1;
        for (int j = n - 1; j > tid; --j) {
            if (s.parent[j] == tid) child = j;
            if (s.parent[j] == s.parent[tid]) sib = j;
        }
        s.child[tid] = child;
        s.sibling[tid] = s.parent[tid] >= 0 ? sib : -1;
    }
    __syncthreads();

    const float *prow = target, *qrow = draft;  // the current node's rows
    double T = 0.0;                             // weight of entry v: max(0, p - T q)
    int round = 0, dead0 = 0, ndead = 0;  // the current node's refused tokens: s.dead[dead0 .. dead0 + ndead)
    // The first kVerHeld blocks of the warp's share stay in shared memory while the walk is at a node (each lane reads what
    // it has copied itself); rows too long for that read the others again in every round.
    float4* held = reinterpret_cast<float4*>(ver_rows) + warp * kVerHeld * 64 + lane;
    const int uh = min(u1, u0 + kVerHeld);
    int held_node = -1;
    int cur = 0, cand = -1, count = 0;
    double Sj = 1.0;
    // this lane's four entries of a block
    auto weigh = [&](int u, const float4& p, const float4& q, double* w) {
        ver_weights(p, q, T, w);
        const int v0 = u * 128 + lane * 4;
        for (int j = 0; j < ndead; ++j) {  // without the refused tokens
            const int x = s.dead[dead0 + j] - v0;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = x == e ? 0.0 : w[e];
        }
    };
    auto fetch = [&](int u, float4& p, float4& q) {
        const int v0 = u * 128 + lane * 4;
        p = ver_load(prow, v0, V, vec);
        q = draft && T != 0.0 ? ver_load(qrow, v0, V, vec) : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    // This warp's total goes into every CTA's table by asynchronous stores that complete on the receiver's mbarrier (a
    // cluster barrier a round took as long as the row's pass itself); returns the table once it is complete, or sets
    // `lost` if that does not happen (bounded).  Two tables take turns: a warp sends round r + 2's total only after every warp's
    // of round r + 1 has come, which each sends after it has read round r's table.
    bool lost = false;  // a wait of this warp has expired
    auto totals = [&]() -> const double* {
        if (held_node != cur) {
            held_node = cur;
            for (int u = u0; u < uh; ++u) {
                ver_hold(held + (u - u0) * 64, prow, u * 128 + lane * 4, V, vec);
                if (draft && T != 0.0) ver_hold(held + (u - u0) * 64 + 32, qrow, u * 128 + lane * 4, V, vec);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
        double t = 0.0;
#pragma unroll 2
        for (int u = u0; u < uh; ++u) {
            double w[4];
            weigh(u, held[(u - u0) * 64], held[(u - u0) * 64 + 32], w);
            t += (w[0] + w[1]) + (w[2] + w[3]);
        }
#pragma unroll 2
        for (int u = uh; u < u1; ++u) {
            float4 p, q;
            double w[4];
            fetch(u, p, q);
            weigh(u, p, q, w);
            t += (w[0] + w[1]) + (w[2] + w[3]);
        }
        t = warp_sum(t);
        double* mine = s.part[round & 1];
        uint64_t* bar = &s.got[round & 1];
        if (tid == 0) mbar_arrive_expect_tx(bar, K * (uint32_t)sizeof(double));
        if (lane < C) ver_send(mine + k, bar, lane, t);
        const bool ok = mbar_wait(bar, (round >> 1) & 1);
        ++round;
        lost = !__all_sync(0xffffffffu, ok);
        return mine;
    };
    // lane l's share of the table: entries [l K / 32, (l + 1) K / 32)
    const int j0 = K * lane / 32, j1 = K * (lane + 1) / 32;
    auto lane_sum = [&](const double* tab) {
        double t = 0.0;
        for (int j = j0; j < j1; ++j) t += tab[j];
        return t;
    };

    auto at_node = [&](int c) {
        cur = c;
        cand = s.child[c];
        prow = target + (row0 + c) * ldt;
        qrow = draft + (draft ? (row0 + c) * ldd : 0);
        T = 0.0;
        Sj = 1.0;
        dead0 += ndead;  // every node is refused once at most: the list never overflows
        ndead = 0;
    };
    at_node(0);
    while (cand >= 0) {  // every thread of the cluster takes the same steps
        double w = positive(s.p[cand] - T * s.q[cand]);
        for (int j = 0; j < ndead; ++j)
            if (s.dead[dead0 + j] == s.token[cand]) w = 0.0;
        if (s.u[cand] * Sj * s.q[cand] < w) {
            if (rank == 0 && tid == 0) path[row0 + count] = cand;
            ++count;
            at_node(cand);
            continue;
        }
        if (!draft) {
            s.dead[dead0 + ndead] = s.token[cand];  // (the same value from every thread)
            ++ndead;
            Sj -= w;
        } else {
            T += Sj;
            if (s.sibling[cand] >= 0) Sj = warp_sum(lane_sum(totals()));
            if (lost) break;
        }
        cand = s.sibling[cand];
    }

    // the last token: first entry whose running sum of weights exceeds u_0 * their sum
    const double* tab = nullptr;
    double t, inc, total;
    for (int attempt = 0;; ++attempt) {
        if (!lost) tab = totals();
        if (lost) {  // this sequence has no result (the walk's steps are no longer the same everywhere)
            cluster_drain();
            if (lane == 0) {
                accepted[b] = -2;
                next[b] = -1;
            }
            return;
        }
        t = lane_sum(tab);
        inc = t;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const double o = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += o;
        }
        total = __shfl_sync(0xffffffffu, inc, 31);
        if (total > 0.0 || attempt) break;
        T = 0.0;  // nothing left: from the target's row itself
        ndead = 0;
    }
    if (rank == 0 && tid == 0) {
        accepted[b] = count;
        if (!(total > 0.0)) next[b] = -1;
    }
    if (!(total > 0.0)) return;
    const double goal = s.u[0] * total;
    // The lane, then its table entry, then the lane of a block and its entry: at each level the first
    // one with a positive weight whose running sum exceeds the goal, or, where the levels' sums differ in
    // their last bits so that none does, the last one with a positive weight.
    auto pick_lane = [&](double running, double own) -> int {
        const unsigned any = __ballot_sync(0xffffffffu, own > 0.0);
        const unsigned hit = __ballot_sync(0xffffffffu, own > 0.0 && running > goal);
        return hit ? __ffs(hit) - 1 : any ? 31 - __clz(any) : -1;
    };
    const int f = pick_lane(inc, t);
    double base = __shfl_up_sync(0xffffffffu, inc, 1);
    if (lane == 0) base = 0.0;
    int mine = -1;
    double mine_base = 0.0;
    for (int j = j0; j < j1; ++j) {
        if (tab[j] > 0.0) {
            mine = j;
            mine_base = base;
            if (base + tab[j] > goal) break;
        }
        base += tab[j];
    }
    const int chosen = __shfl_sync(0xffffffffu, mine, f);
    base = __shfl_sync(0xffffffffu, mine_base, f);
    if (chosen != k) return;
    int answer = -1;
    bool done = false;
    auto search = [&](int u, const double* w) {
        const double own = (w[0] + w[1]) + (w[2] + w[3]);
        double run = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const double o = __shfl_up_sync(0xffffffffu, run, d);
            if (lane >= d) run += o;
        }
        const double block = __shfl_sync(0xffffffffu, run, 31);
        double before = __shfl_up_sync(0xffffffffu, run, 1);
        const int l = pick_lane(base + run, own);
        if (done || l < 0) return;
        before = base + (lane == 0 ? 0.0 : before);
        int at = -1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool open = at < 0 || !(before > goal);  // not past the goal yet
            if (open && w[e] > 0.0) at = u * 128 + lane * 4 + e;
            if (open) before += w[e];
        }
        answer = __shfl_sync(0xffffffffu, at, l);
        done = base + block > goal;
        base += block;
    };
    for (int u = u0; u < uh && !done; ++u) {
        double w[4];
        weigh(u, held[(u - u0) * 64], held[(u - u0) * 64 + 32], w);
        search(u, w);
    }
    for (int u = uh; u < u1 && !done; ++u) {
        float4 p, q;
        double w[4];
        fetch(u, p, q);
        weigh(u, p, q, w);
        search(u, w);
    }
    if (lane == 0) next[b] = answer;
}

// ---------------------------------------------------------------- commit
// One CTA per (layer, sequence, K or V); a thread copies 16-byte pieces, several loads in flight (one load at a time,
// each behind its node's path entry, took 18.1 us for 32 x 24 caches; so 13.3, 4.8 TB/s of the 6.5 of a copy).
constexpr int kCommitThreads = 256;
constexpr int kCommitBatch = 5;

__global__ void __launch_bounds__(kCommitThreads, 5)
    tree_commit_k(const half* TK, const half* TV, size_t tree_layer_stride, half* K, half* V,
                  size_t layer_stride, int stride, int slot_rows, int num_slots, const int* slot,
                  const int* len, const int* path, const int* accepted, int N,
                  int cols, int* len_out) {
    __shared__ int node[kMaxNodes];  // the tree row of each committed row
    const int b = blockIdx.x, l = blockIdx.y, tid = threadIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    if (tid < N) node[tid] = tid ? path[(size_t)b * N + tid - 1] : 0;
    const int at = slot ? slot[b] : b, m = len[b], acc = accepted[b];
    const bool ok = at >= 0 && at < num_slots && m >= 0 && m <= slot_rows && acc >= 0;
    const int rows = ok ? min(1 + min(acc, N - 1), slot_rows - m) : 0;
    if (l == 0 && blockIdx.z == 0 && tid == 0 && len_out) len_out[b] = m + rows;
    __syncthreads();
    const half* src = (blockIdx.z ? TV : TK) + (size_t)l * tree_layer_stride + (size_t)b * N * cols;
    half* dst = (blockIdx.z ? V : K) + (size_t)l * layer_stride + ((size_t)(ok ? at : 0) * slot_rows + m) * stride;
    const int per = cols / 8, all = rows * per;  // 16-byte pieces
    for (int x0 = tid; x0 < all; x0 += kCommitBatch * kCommitThreads) {
        uint4 y[kCommitBatch];
        int row[kCommitBatch], e[kCommitBatch];
#pragma unroll
        for (int k = 0; k < kCommitBatch; ++k) {
            const int x = x0 + k * kCommitThreads;
            row[k] = x < all ? x / per : -1;
            e[k] = (x - row[k] * per) * 8;
            const int n = row[k] >= 0 ? node[row[k]] : -1;
            if (n < 0 || n >= N) row[k] = -1;  // past the end, or no node of this tree
            else y[k] = ld_once_u4(src + (size_t)n * cols + e[k]);
        }
#pragma unroll
        for (int k = 0; k < kCommitBatch; ++k)
            if (row[k] >= 0) *reinterpret_cast<uint4*>(dst + (size_t)row[k] * stride + e[k]) = y[k];
    }
}

int current_device() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 ? dev : -1;
}
int sm_count() {
    static std::atomic<int> known[64];
    const int dev = current_device();
    if (dev < 0) return 148;
    int n = known[dev];
    if (!n) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
        known[dev] = n;
    }
    return n;
}
// Clusters of more than 8 CTAs and more than 48 KB of shared memory have to be asked for, once per device.
cudaError_t ver_allow() {
    static std::atomic<bool> done[64];
    const int dev = current_device();
    if (dev >= 0 && done[dev]) return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(tree_verify_k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(tree_verify_k, cudaFuncAttributeMaxDynamicSharedMemorySize, kVerHeldBytes);
    if (e == cudaSuccess && dev >= 0) done[dev] = true;
    return e;
}

// Grid limits and products of sizes that index in 32 bits.
bool sizes_ok(int B, int N, int H, int KV) {
    return B > 0 && B <= 65535 && N > 0 && N <= kMaxNodes && KV > 0 && H >= KV && H % KV == 0 && H <= 1024;
}

}  // namespace

extern "C" {

int llmdiy_tree_layout(const int* parent, int n, int* depth, uint64_t* mask, int mask_words) {
    if (!parent || !depth || !mask || n < 1 || n > kMaxNodes || mask_words < (n + 63) / 64 || parent[0] != -1)
        return -1;
    for (int i = 1; i < n; ++i)
        if (parent[i] < 0 || parent[i] >= i) return -1;
    for (int i = 0; i < n; ++i) {
        const int p = parent[i];
        uint64_t* m = mask + (size_t)i * mask_words;
        for (int w = 0; w < mask_words; ++w) m[w] = p < 0 ? 0 : mask[(size_t)p * mask_words + w];
        m[i / 64] |= 1ull << (i % 64);
        depth[i] = p < 0 ? 0 : depth[p] + 1;
    }
    return 0;
}

int llmdiy_tree_rope(const uint16_t* qkv, const uint16_t* bias, const int* depth, const int* len,
                     const int* tree_len, int B, int N, int num_heads, int num_kv_heads, float rope_base,
                     uint16_t* Q, uint16_t* TK, uint16_t* TV, void* stream) {
    if (!sizes_ok(B, N, num_heads, num_kv_heads) || !qkv || !depth || !len || !Q || !TK || !TV || !aligned16(qkv) ||
        !aligned16(bias) || !aligned16(Q) || !aligned16(TK) || !aligned16(TV) || !words_aligned(depth, len, tree_len) ||
        !(rope_base > 0.f) || !(rope_base < INFINITY))
        return (int)cudaErrorInvalidValue;
    RopeFreqs freqs;
    const double step = -log2((double)rope_base) / (kDim / 2);
    double coarse[8], fine[8];  // base^(-t/64), t = 8 i + j, from 16 powers
    for (int i = 0; i < 8; ++i) {
        coarse[i] = exp2(step * 8 * i);
        fine[i] = exp2(step * i);
    }
    for (int t = 0; t < kDim / 2; ++t) freqs.f[t] = coarse[t >> 3] * fine[t & 7];
    return launch_pdl(tree_rope_k, dim3(N, B), kRopeThreads, S(stream), reinterpret_cast<const half*>(qkv),
                      reinterpret_cast<const half*>(bias), depth, len, tree_len, N, num_heads, num_kv_heads, freqs,
                      reinterpret_cast<half*>(Q), reinterpret_cast<half*>(TK), reinterpret_cast<half*>(TV));
}

int llmdiy_tree_verify(const float* target, int ldt, const float* draft, int ldd, const int* token,
                       const int* parent, const int* tree_len, const float* uniform, int B, int N, int V, int* path,
                       int* accepted, int* next, void* stream) {
    if (B <= 0 || B > 65535 || N <= 0 || N > kMaxNodes || V <= 0 || V > (1 << 30) || !target || ldt < V ||
        (draft && ldd < V) || !token || !parent || !uniform || !path || !accepted || !next ||
        !words_aligned(target, draft, token, parent, tree_len, uniform, path, accepted, next))
        return (int)cudaErrorInvalidValue;
    const int vec = aligned16(target) && ldt % 4 == 0 && (!draft || (aligned16(draft) && ldd % 4 == 0));
    // CTAs per sequence: as many as run at once (two per SM), 14 at most, and 10 rather than 11 to 13, of which 21 clusters fit
    // on 148 SMs.  Measured at V = 151936, trees of 16: 1 sequence 9.7 us with 14, 11.0 with 16, 13.1 with 8; 16 20.5, 24.5, 24.9;
    // 24 29.5 with 10, 33.5 with 12, 35.2 with 8; 32 36.4 with 9, 34.7 with 10; at V = 64000 48 sequences 24.8 with 6, 28.9 with 8.
    int C = kVerCtasPerSm * sm_count() / B;
    C = C >= kVerMaxCluster ? kVerMaxCluster : C > 10 ? 10 : std::max(C, 1);
    cudaError_t e = ver_allow();
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(B * C);
    lc.blockDim = dim3(kVerThreads);
    lc.dynamicSmemBytes = kVerHeldBytes;
    lc.stream = S(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = attr;
    lc.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&lc, tree_verify_k, target, ldt, draft, ldd, token, parent, tree_len, uniform, N, V,
                                   vec, path, accepted, next);
}

int llmdiy_tree_commit(const uint16_t* TK, const uint16_t* TV, size_t tree_layer_stride, uint16_t* K, uint16_t* V,
                       size_t layer_stride, int stride, int slot_rows, int num_slots, const int* slot,
                       const int* len, const int* path, const int* accepted, int B, int N, int num_kv_heads,
                       int layers, int* len_out, void* stream) {
    const int cols = num_kv_heads * kDim;
    if (!sizes_ok(B, N, num_kv_heads, num_kv_heads) || !TK || !TV || !K || !V || !len || !path || !accepted ||
        layers <= 0 || layers > 65535 || slot_rows <= 0 || num_slots <= 0 || stride < cols || (stride & 7) ||
        (layer_stride & 7) || (tree_layer_stride & 7) || len_out == len ||
        (layers > 1 && (layer_stride < ((size_t)num_slots * slot_rows - 1) * stride + cols ||
                        tree_layer_stride < (size_t)B * N * cols)) ||
        !aligned16(TK) || !aligned16(TV) || !aligned16(K) || !aligned16(V) ||
        !words_aligned(slot, len, path, accepted, len_out))
        return (int)cudaErrorInvalidValue;
    return launch_pdl(tree_commit_k, dim3(B, layers, 2), kCommitThreads, S(stream), reinterpret_cast<const half*>(TK),
                      reinterpret_cast<const half*>(TV), tree_layer_stride, reinterpret_cast<half*>(K),
                      reinterpret_cast<half*>(V), layer_stride, stride, slot_rows, num_slots, slot, len, path, accepted,
                      N, cols, len_out);
}

}  // extern "C"
