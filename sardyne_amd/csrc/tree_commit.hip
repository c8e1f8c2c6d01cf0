// The end of a speculative step: the walk down the drafted tree along the sampled tokens, and the accepted nodes' K/V
// rows into the cache of every layer.
//
// From node 0, the step's own token, to the lowest child whose token is the one sampled at its parent, until there is
// none. A child has a higher index than its parent, so the walk ends after at most n_tok nodes.
#include "sdy_device.h"
#include "sdy_internal.h"
#include "sdy_ops.h"

namespace {

constexpr int MAX_NODES = 256, THREADS = 256;

// Bound by its launch: 8 nodes into 36 layers of 2 kv heads 2.9 us, 61 into 48 layers of 4 (f16 rows of 128) 3.0 us; what it
// moves is under 1 MB. One workgroup per layer, K or V, and kv head. Each walks the tree itself (a node's next one by an LDS minimum over its
// children, whose order does not matter), so one launch does it all. U: the unit that rows are copied in.
template <class U>
__global__ __launch_bounds__(THREADS) void k_tree_commit(sdy_tree_commit_args a, int row_units) {
    __shared__ int next[MAX_NODES], path[MAX_NODES], count;
    const int tid = threadIdx.x, n = a.n_tok;
    if (tid < n) next[tid] = n;
    __syncthreads();
    if (tid > 0 && tid < n) {
        const int p = a.parent[tid];
        if (p >= 0 && p < tid && a.token[tid] == a.sampled[p]) atomicMin(&next[p], tid);
    }
    __syncthreads();
    const int past = *a.n_past;
    if (tid == 0) {
        const int room = past < 0 || past >= a.max_seq || a.parent[0] < -1 ? 0 : a.max_seq - past;
        int c = 0;
        for (int t = 0; t < n && c < room; t = next[t]) path[c++] = t;
        count = c;
    }
    __syncthreads();
    const int acc = count;
    const int g = blockIdx.x, is_v = blockIdx.y, l = blockIdx.z;
    if (g == 0 && is_v == 0 && l == 0) {
        if (tid < n) a.path[tid] = tid < acc ? path[tid] : -1;
        if (tid == 0) *a.n_acc = acc;
        if (tid == 0 && acc > 0) {
            a.step[0] = a.sampled[path[acc - 1]];
            a.step[1] = past + acc;
        }
    }
    const U *src = (const U *)(is_v ? a.v_draft : a.k_draft);
    U *dst = (U *)(is_v ? a.v_cache : a.k_cache);
    const int per = a.hd / row_units;  // elements of a unit
    src += ((size_t)l * a.draft_layer_stride + (size_t)g * a.draft_stride) / per;
    dst += ((size_t)l * a.layer_stride + (size_t)g * a.head_stride) / per + (size_t)(acc ? past : 0) * row_units;
    for (int i = tid; i < acc * row_units; i += THREADS) {
        const int r = i / row_units, c = i - r * row_units;
        dst[i] = src[(size_t)path[r] * row_units + c];
    }
}

}  // namespace

extern "C" int sdy_tree_commit(const sdy_tree_commit_args *a, sdy_stream s) {
    if (!a) return sdy_fail(-1, "tree_commit: no arguments");
    if (a->n_tok < 1 || a->n_tok > MAX_NODES) return sdy_fail(-1, "tree_commit: n_tok %d (1..%d)", a->n_tok, MAX_NODES);
    const size_t elt = sdy_kv_elt_bytes(a->kv_type);
    if (!elt) return sdy_fail(-1, "tree_commit: KV type %d", a->kv_type);
    if (a->n_layer < 1 || a->n_layer > 65535 || a->n_kv_head < 1 || a->hd < 1 || a->hd > 512 || a->max_seq < 1)
        return sdy_fail(-1, "tree_commit: n_layer %d (1..65535), n_kv_head %d, head_dim %d (1..512), max_seq %d", a->n_layer,
                        a->n_kv_head, a->hd, a->max_seq);
    if (!a->token || !a->parent || !a->sampled || !a->n_past || !a->k_draft || !a->v_draft || !a->k_cache || !a->v_cache ||
        !a->path || !a->n_acc || !a->step)
        return sdy_fail(-1, "tree_commit: every array is needed");
    if ((a->n_kv_head > 1 && (a->draft_stride < (long)a->n_tok * a->hd || a->head_stride < (long)a->max_seq * a->hd)) ||
        (a->n_layer > 1 && (a->draft_layer_stride < (a->n_kv_head - 1) * a->draft_stride + (long)a->n_tok * a->hd ||
                            a->layer_stride < (a->n_kv_head - 1) * a->head_stride + (long)a->max_seq * a->hd)))
        return sdy_fail(-1, "tree_commit: a head's or layer's rows reach into the next one's (strides %ld, %ld, %ld, %ld)",
                        a->draft_stride, a->draft_layer_stride, a->head_stride, a->layer_stride);
    // every workgroup reads these while one writes those
    const int32_t *const in[4] = {a->token, a->parent, a->sampled, a->n_past};
    const int in_n[4] = {a->n_tok, a->n_tok, a->n_tok, 1};
    const int32_t *const out[3] = {a->path, a->n_acc, a->step};
    const int out_n[3] = {a->n_tok, 1, 2};
    for (int i = 0; i < 4; i++)
        for (int o = 0; o < 3; o++)
            if (in[i] < out[o] + out_n[o] && out[o] < in[i] + in_n[i])
                return sdy_fail(-1, "tree_commit: path, n_acc and step must not overlap token, parent, sampled or n_past");
    for (int o = 0; o < 3; o++)
        if (out[o] < out[(o + 1) % 3] + out_n[(o + 1) % 3] && out[(o + 1) % 3] < out[o] + out_n[o])
            return sdy_fail(-1, "tree_commit: path, n_acc and step must not overlap each other");
    // (the first head's: the others lie as these do)
    const void *const draft[2] = {a->k_draft, a->v_draft}, *const cache[2] = {a->k_cache, a->v_cache};
    for (int i = 0; i < 2; i++) {
        const char *const d = (const char *)draft[i], *const c = (const char *)cache[i];
        if (d < c + (size_t)a->max_seq * a->hd * elt && c < d + (size_t)a->n_tok * a->hd * elt)
            return sdy_fail(-1, "tree_commit: the drafted rows must not be the cache's own");
    }
    const uintptr_t all = (uintptr_t)a->k_draft | (uintptr_t)a->v_draft | (uintptr_t)a->k_cache | (uintptr_t)a->v_cache |
                          (uintptr_t)((a->draft_stride | a->draft_layer_stride | a->head_stride | a->layer_stride | a->hd) * (long)elt);
    const dim3 grid(a->n_kv_head, 2, a->n_layer);
    const int bytes = a->hd * (int)elt;
    if (all % 16 == 0)
        hipLaunchKernelGGL(k_tree_commit<uint4>, grid, dim3(THREADS), 0, (hipStream_t)s, *a, bytes / 16);
    else if (elt == 4)
        hipLaunchKernelGGL(k_tree_commit<uint32_t>, grid, dim3(THREADS), 0, (hipStream_t)s, *a, a->hd);
    else
        hipLaunchKernelGGL(k_tree_commit<uint16_t>, grid, dim3(THREADS), 0, (hipStream_t)s, *a, a->hd);
    return sdy_check_launch("tree_commit");
}
