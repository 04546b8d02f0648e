/*
 * llmdiy_tree.h — C ABI of the speculative-decoding operators: one step that scores a tree of
 * drafted tokens per sequence in a single pass, verifies the drafts and commits what was accepted.
 *
 * No counterpart in the reference, which decodes one greedy token per step (QwenEngine::step,
 * framework_src/qwen_infer.cu:614-737); each operator stands beside the launcher of its kind in
 * llmdiy_kernels.h (RoPE + KV append, flash decoding, argmax).  The conventions are that header's:
 * device pointers owned by the caller on the current device, each aligned as its type, fp16 as uint16_t bit patterns, a trailing
 * stream (NULL = the legacy default stream), the cudaError_t of the launch as the return
 * value (cudaErrorInvalidValue for refused arguments, before anything is launched; B <= 65535, at most 1024 heads,
 * V <= 2^30), outputs that overlap no input and no other output, no allocation,
 * no synchronisation: every launcher can be captured into a CUDA graph, and the lengths, trees and slots are
 * read on the device when it runs.  Calls launch clusters of up to 16 CTAs; a part of a GPU that cannot place them
 * answers with the launch's error.
 *
 * The tree.  Sequence b (0 <= b < B) has nodes 0 .. tree_len[b]-1 (tree_len NULL: N each; values
 * are clamped to 0..N), N <= 256.  Node 0 is the root: the last token of the sequence, whose K/V
 * rows are not in the cache yet.  parent[b][i] < i is the node that node i continues (-1 for the root).
 * Arrays over nodes are [B][N]; what belongs to nodes at or past tree_len[b] has no
 * effect and, in the outputs of tree_rope and tree_attn, is left as it was.
 *
 * The cache.  The caller's, laid out as a batch's (llmdiy_batch.h), whose own is not handed out: row r of kv
 * head h of slot s is at (s * slot_rows + r) * stride + h * 128 elements, in K and in V; sequence b uses slot[b] (NULL: slot
 * b) and has len[b] committed rows (positions 0 .. len[b]-1).  The tree's own K/V rows live in buffers
 * [B][N][num_kv_heads*128] until llmdiy_tree_commit.  A slot outside 0..num_slots-1 has no rows.
 */
#ifndef LLMDIY_TREE_H
#define LLMDIY_TREE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Most nodes of a tree. */
#define LLMDIY_TREE_MAX_NODES 256

/* Host helper (no CUDA call): depth[n] and visibility mask of one tree from parent[n] (host arrays).
 * mask is [n][mask_words] 64-bit words, mask_words >= ceil(n/64): bit j % 64 of word j / 64 of node i is set
 * when node i sees node j (itself and its ancestors).  Returns 0, or -1 (nothing written) when n is out of
 * 1..256, mask_words is too small, parent[0] != -1 or some parent[i] is not in 0..i-1. */
int llmdiy_tree_layout(const int* parent, int n, int* depth, uint64_t* mask, int mask_words);

/* Bias and rotary position of the tree's rows (stands beside llmdiy_fused_qkv_rope_cache, whose pairing
 * (t, t + 64) it shares).  qkv is [B][N][(num_heads + 2 num_kv_heads) * 128] (queries, keys, values);
 * bias is one such row, or NULL.  Node i of sequence b turns by the angles (len[b] + depth[b][i]) *
 * rope_base^(-t/64), t < 64, formed and reduced to one turn in 64 bits; their cosines and sines are fp32, within 2^-21 for
 * angles up to 2^24.  The bias is added in fp32 and each output is rounded to fp16 once.  Writes Q [B][N][num_heads*128], TK and TV
 * [B][N][num_kv_heads*128], which may not overlap qkv.  All pointers to fp16 are 16-byte aligned. */
int llmdiy_tree_rope(const uint16_t* qkv, const uint16_t* bias, const int* depth, const int* len,
                     const int* tree_len, int B, int N, int num_heads, int num_kv_heads, float rope_base,
                     uint16_t* Q, uint16_t* TK, uint16_t* TV, void* stream);

/* Attention of the tree's nodes: O[b][i] = softmax(q k^T / sqrt(128)) v over the sequence's len[b]
 * committed rows, all of which every node sees, and the tree's rows that mask[b][i] names
 * ([B][N][ceil(N/64)] words as llmdiy_tree_layout writes them, any pattern).  N = 1 is plain decoding.
 * Head h uses kv head h / (num_heads / num_kv_heads).  Node rows of Q and O are ldq and ldo elements
 * apart (>= num_heads*128).  max_len bounds every len[b] (larger values are clamped); it sets the grid and the
 * workspace, so a captured graph serves every length up to it.  fp32 scores, statistics and
 * accumulation; probabilities as the sum of two fp16, which rounds each by 2^-22 of itself or 2^-32 of its row's largest,
 * whichever is more, whatever else is in the call.
 * A visible score of NaN or +inf makes its row NaN.  A row that sees nothing, or only scores of -inf, gives zeros; what
 * a node does not see (K and V rows at or past len[b], tree rows outside its mask) does not reach its
 * output even where it is Inf or NaN.
 * stride, ldq, ldo: multiples of 8 elements; fp16 pointers 16-byte aligned; num_slots * slot_rows < 2^31;
 * num_heads / num_kv_heads <= 128; max_len <= slot_rows.
 * work: llmdiy_tree_attn_work_bytes(...) bytes (16-byte aligned, zero-filled once before its first use),
 * which serves every smaller B, N and max_len with the same heads too; calls that may overlap on the GPU need
 * workspaces of their own. */
size_t llmdiy_tree_attn_work_bytes(int B, int N, int num_heads, int num_kv_heads, int max_len);
int llmdiy_tree_attn(const uint16_t* Q, int ldq, const uint16_t* K, const uint16_t* V, int stride, int slot_rows,
                     int num_slots, const int* slot, const int* len, int max_len, const uint16_t* TK,
                     const uint16_t* TV, const uint64_t* mask, const int* tree_len, int B, int N, int num_heads,
                     int num_kv_heads, uint16_t* O, int ldo, float* work, size_t work_bytes, void* stream);
/* Which way a call of these sizes runs on the current device: 0 all units' keys dealt in equal ranges over the SMs, cut
 * units joined by a second launch; 1 a cluster of CTAs per unit; 2 the same on the CUDA cores (one to four query rows per
 * kv head and sequence); -1 for sizes that are refused. */
int llmdiy_tree_attn_path(int B, int N, int num_heads, int num_kv_heads, int max_len);
/* After the stream is synchronised: 0, or -5 when a pipeline wait of a call with this workspace expired
 * since the last status query (that output is then not valid); the query clears the word. */
int llmdiy_tree_attn_status(const float* work);

/* Probabilities of R rows of V fp16 logits (row pitches ldl and ldp elements, >= V):
 * probs = exp((x - max) / temp[r]) / sum in fp32, temp NULL = 1.  temp <= 0 (or NaN) gives the limit: equal shares
 * of the row's largest entries (greedy; llmdiy_argmax picks one of them by a rule of its own).  Entries of -inf get 0; a
 * row with nothing above -inf gives zeros; one with a NaN or +inf is NaN throughout.  A bounded wait that expires (nothing
 * else reports it) makes NaN of its row, or of parts of it, and of those that were still to come.  Rows of up to 156600
 * entries are read once; of longer ones the rest is read three times and takes about twice as long an entry. */
int llmdiy_softmax_rows(const uint16_t* logits, int ldl, const float* temp, int R, int V, float* probs, int ldp,
                        void* stream);

/* Verification of the drafts against the target's probabilities (lossless: the tokens are distributed as
 * the target's).  Row b * N + i of `target` ([B*N] rows of V, pitch ldt) is the target's distribution
 * after node i; the same row of `draft` (pitch ldd) is the distribution that the children of node i were drawn from,
 * independently of each other.  token[b][i] is node i's drafted token (token[b][0] is not read),
 * uniform[b][i] a random number in [0, 1).
 * The walk starts at the root c = 0.  The children x_1, x_2, .. of c are tried in index order, with T_1 = 0, S_1 = 1:
 *   w_j(v) = max(0, p(v) - T_j q(v));  x_j is accepted when uniform * S_j * q(x_j) < w_j(x_j), and the walk
 *   goes on from it; otherwise T_{j+1} = T_j + S_j and S_{j+1} = sum_v w_{j+1}(v)
 * (the residual distributions norm(max(0, p - q)) applied j times).  draft NULL: deterministic
 * drafts, q(x_j) = 1; a refused token leaves the distribution: w_j is p without the tokens refused
 * so far and S_{j+1} = S_j - w_j(x_j).  When no child is accepted, next[b] is drawn from the last w: the first v whose running
 * sum exceeds uniform[b][0] * sum w (from p itself when w sums to 0).  Products and sums are in 64 bits.
 * Writes path[b][0..accepted-1] = the accepted nodes in order (then -1 up to N), accepted[b] and next[b].
 * A node whose token is outside 0..V-1 or whose parent is not in 0..i-1 is never tried; entries of the distributions that
 * are not > 0 count as 0; next is -1 when p has none above 0.  A sequence without nodes (tree_len 0)
 * gets accepted = -1, next = -1; one for which a bounded wait expired accepted = -2, next = -1 (its path is not valid, and
 * llmdiy_tree_commit moves nothing for it). */
int llmdiy_tree_verify(const float* target, int ldt, const float* draft, int ldd, const int* token,
                       const int* parent, const int* tree_len, const float* uniform, int B, int N, int V, int* path,
                       int* accepted, int* next, void* stream);

/* Moves the root's and the accepted nodes' K/V rows into the cache, for `layers` layers: rows 0, path[b][0], ..,
 * path[b][accepted[b]-1] of TK/TV become cache rows len[b], len[b]+1, .. of slot[b].  Layer l's tree buffers are
 * tree_layer_stride elements, its caches layer_stride elements after layer 0's.  len_out (may be NULL, may not be
 * len) gets len[b] + 1 + accepted[b] (of which N - 1 at most count).  Rows past slot_rows are dropped (len_out stops at slot_rows), a path entry
 * outside 0..N-1 leaves its cache row as it was, and accepted < 0 or a slot or len out of range moves
 * nothing (len_out = len).  No two sequences may share a slot; TK/TV may not overlap the caches. */
int llmdiy_tree_commit(const uint16_t* TK, const uint16_t* TV, size_t tree_layer_stride, uint16_t* K, uint16_t* V,
                       size_t layer_stride, int stride, int slot_rows, int num_slots, const int* slot,
                       const int* len, const int* path, const int* accepted, int B, int N, int num_kv_heads,
                       int layers, int* len_out, void* stream);

#ifdef __cplusplus
}
#endif
#endif
