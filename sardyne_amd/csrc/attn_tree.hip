// Attention of a tree of drafted tokens over the cache and over their own ancestors.
//
// Node t of a head takes the scores q_t.k_j / sqrt(head_dim) over every cached position j < n_past and over the drafted
// rows of t and the nodes above it (parent, its parent, ...), one softmax over them, and the weighted sum of the V rows.
// A parent outside [0, t) makes t a root; below -1 it marks a place without a node: its output row stays as it was and no
// node attends to it.
#include <type_traits>

#include "sdy_attn_dev.h"
#include "sdy_device.h"
#include "sdy_internal.h"
#include "sdy_ops.h"

namespace {

constexpr int MAX_NODES = 256, THREADS = 256;

SDY_DEV float block_reduce(float v, float *sh, bool max) {
    for (int off = 32; off >= 1; off >>= 1) {
        const float o = __shfl_xor(v, off);
        v = max ? fmaxf(v, o) : v + o;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    return max ? fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3])) : (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// One workgroup per node and head: 256 keys at a time, a key per thread, then a dim per thread.
template <class KT>
__global__ __launch_bounds__(THREADS) void k_attn_tree(sdy_attn_tree_args a, float scale) {
    __shared__ float q[256], p[THREADS], sh[4];
    __shared__ int key[THREADS], n_anc;
    const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
    const int past = *a.n_past;
    if (past < 0 || past > a.max_past || a.parent[t] < -1) return;
    const int g = h / (a.n_head / a.n_kv_head);
    if (tid < a.hd) q[tid] = a.q[(size_t)t * a.q_stride + (size_t)h * a.hd + tid];
    if (tid == 0) {
        int n = 0;
        for (int u = t;;) {
            key[n++] = u;
            const int up = a.parent[u];
            if (up < 0 || up >= u || a.parent[up] < -1) break;
            u = up;
        }
        n_anc = n;
    }
    __syncthreads();
    const KT *kc = (const KT *)a.k_cache + (size_t)g * a.head_stride, *vc = (const KT *)a.v_cache + (size_t)g * a.head_stride;
    const KT *kd = (const KT *)a.k_draft + (size_t)g * a.draft_stride, *vd = (const KT *)a.v_draft + (size_t)g * a.draft_stride;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (int j0 = 0; j0 < past + n_anc; j0 += THREADS) {
        const int left = past + n_anc - j0, j = j0 + tid;
        float s = -INFINITY;
        if (tid < left) {
            const KT *k = j < past ? kc + (size_t)j * a.hd : kd + (size_t)key[j - past] * a.hd;
            float d = 0.0f;
            for (int i = 0; i < a.hd; i += 4) {
                const sdy_f32x4 v = KvElt<KT>::ld4(k, i);
                for (int e = 0; e < 4; e++) d = __builtin_fmaf(q[i + e], v[e], d);
            }
            s = d * scale;
        }
        const float m_new = fmaxf(m, block_reduce(s, sh, true));
        const float mu = m_new == -INFINITY ? 0.0f : m_new;
        const float e = __expf(s - mu), corr = __expf(m - mu);
        p[tid] = e;
        l = l * corr + block_reduce(e, sh, false);
        m = m_new;
        __syncthreads();
        o *= corr;
        if (tid < a.hd)
            for (int i = 0; i < left && i < THREADS; i++) {
                const KT *v = j0 + i < past ? vc + (size_t)(j0 + i) * a.hd : vd + (size_t)key[j0 + i - past] * a.hd;
                o = __builtin_fmaf(p[i], KvElt<KT>::ld(v, tid), o);
            }
        __syncthreads();
    }
    if (tid < a.hd) a.out[(size_t)t * a.out_stride + (size_t)h * a.hd + tid] = o / l;
}

}  // namespace

extern "C" int sdy_attn_tree_ok(int n_tok, int n_head, int n_kv_head, int hd) {
    return n_tok >= 1 && n_tok <= MAX_NODES && n_head >= 1 && n_kv_head >= 1 && n_head % n_kv_head == 0 &&
           (hd == 64 || hd == 128 || hd == 256);
}

extern "C" size_t sdy_attn_tree_floats(int n_tok, int n_head, int n_kv_head, int hd, int max_past) {
    if (!sdy_attn_tree_ok(n_tok, n_head, n_kv_head, hd) || max_past < 0) return 0;
    return 64;
}

extern "C" int sdy_attn_tree(const sdy_attn_tree_args *a, sdy_stream s) {
    if (!a) return sdy_fail(-1, "attn_tree: no arguments");
    if (a->n_tok == 0) return 0;
    if (!sdy_attn_tree_ok(a->n_tok, a->n_head, a->n_kv_head, a->hd))
        return sdy_fail(-1, "attn_tree: n_tok 1..%d (%d), n_head a multiple of n_kv_head (%d, %d), head_dim 64, 128 or 256 (%d)",
                        MAX_NODES, a->n_tok, a->n_head, a->n_kv_head, a->hd);
    const size_t elt = sdy_kv_elt_bytes(a->kv_type);
    if (!elt) return sdy_fail(-1, "attn_tree: KV type %d", a->kv_type);
    if (!a->q || !a->k_draft || !a->v_draft || !a->parent || !a->n_past || !a->out || !a->part)
        return sdy_fail(-1, "attn_tree: q, the drafted rows, parent, n_past, out and part are needed");
    if (a->max_past < 0 || (a->max_past > 0 && (!a->k_cache || !a->v_cache)))
        return sdy_fail(-1, "attn_tree: max_past %d and the caches", a->max_past);
    if (a->n_kv_head > 1 && (a->head_stride < (long)a->max_past * a->hd || a->draft_stride < (long)a->n_tok * a->hd))
        return sdy_fail(-1, "attn_tree: a kv head's rows (%d cached, %d drafted) reach into the next one's (strides %ld, %ld)",
                        a->max_past, a->n_tok, a->head_stride, a->draft_stride);
    const uintptr_t rows = (uintptr_t)a->k_cache | (uintptr_t)a->v_cache | (uintptr_t)a->k_draft | (uintptr_t)a->v_draft |
                           (uintptr_t)((a->head_stride | a->draft_stride) * (long)elt);
    if (((uintptr_t)a->q | (uintptr_t)a->out | (uintptr_t)a->part | (uintptr_t)((a->q_stride | a->out_stride) * 4) | rows) & 15)
        return sdy_fail(-1, "attn_tree: q, out, part and K/V rows (and strides) aligned to 16 bytes");
    if (a->q_stride < (long)a->n_head * a->hd || a->out_stride < (long)a->n_head * a->hd)
        return sdy_fail(-1, "attn_tree: q and out rows of %d x %d floats (strides %ld, %ld)", a->n_head, a->hd, a->q_stride,
                        a->out_stride);
    const float scale = 1.0f / sqrtf((float)a->hd);
    if (a->kv_type == SDY_KV_F16)
        hipLaunchKernelGGL(k_attn_tree<uint16_t>, dim3(a->n_tok, a->n_head), dim3(THREADS), 0, (hipStream_t)s, *a, scale);
    else
        hipLaunchKernelGGL(k_attn_tree<float>, dim3(a->n_tok, a->n_head), dim3(THREADS), 0, (hipStream_t)s, *a, scale);
    return sdy_check_launch("attn_tree");
}
