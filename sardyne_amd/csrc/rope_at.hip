// Rotary positions of tokens that do not stand one after another: every token has its position and its cache slot.
//
// For pair i < n_rot / 2 of a head, (a, b) = dims (2i, 2i + 1) or (i, i + n_rot / 2):
//   angle = pos[t] freq[i] in 64 bits, c = f32(mscale cos angle), s = f32(mscale sin angle), (a, b) -> (a c - b s, a s + b c).
// Dims from n_rot on pass. q_norm / k_norm: the head's RMSNorm first. The rounding steps are those of the cached tables
// (sdy_rope_table_host and k_qk_rope_kv), so that a whole unscaled head at pos0 + t gives their values.
#include "sdy_attn_dev.h"
#include "sdy_device.h"
#include "sdy_internal.h"
#include "sdy_norm_dev.h"
#include "sdy_ops.h"

namespace {

// sin and cos of x in 64 bits, to about 1e-14: x = n pi/2 + r with pi/2 in two parts (the first step is exact for
// |n| < 2^31: the remainder is a multiple of 2^-52 below 1), then Taylor's series up to r^15 and r^16 for |r| <= pi/4.
SDY_DEV void sincos_f64(double x, double *sn, double *cs) {
    const double n = rint(x * 0.63661977236758134308);
    double r = fma(-n, 1.57079632679489655800, x);
    r = fma(-n, 6.12323399573676603587e-17, r);
    const double z = r * r;
    double s = -1.0 / 1307674368000.0;
    s = fma(s, z, 1.0 / 6227020800.0);
    s = fma(s, z, -1.0 / 39916800.0);
    s = fma(s, z, 1.0 / 362880.0);
    s = fma(s, z, -1.0 / 5040.0);
    s = fma(s, z, 1.0 / 120.0);
    s = fma(s, z, -1.0 / 6.0);
    s = fma(s * z, r, r);
    double c = 1.0 / 20922789888000.0;
    c = fma(c, z, -1.0 / 87178291200.0);
    c = fma(c, z, 1.0 / 479001600.0);
    c = fma(c, z, -1.0 / 3628800.0);
    c = fma(c, z, 1.0 / 40320.0);
    c = fma(c, z, -1.0 / 720.0);
    c = fma(c, z, 1.0 / 24.0);
    c = fma(c, z, -0.5);
    c = fma(c, z, 1.0);
    const int quad = (int)(n - 4.0 * floor(n * 0.25));
    const double a = quad & 1 ? c : s, b = quad & 1 ? s : c;
    *sn = quad & 2 ? -a : a;
    *cs = (quad + 1) & 2 ? -b : b;
}

// One workgroup per token and head-group: one wave per head of q, k or v, the head in LDS.
template <class KT>
__global__ __launch_bounds__(256) void k_qk_rope_at(sdy_rope_at_args a) {
    __shared__ float cs[256], sn[256], heads[4][512];
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int half = a.n_rot / 2;
    const int pos = a.pos[t];
    const long slot = a.slot ? a.slot[t] : pos;
    if (tid < half) {
        double s, c;
        sincos_f64((double)pos * a.freq[tid], &s, &c);
        cs[tid] = (float)((double)a.mscale * c);
        sn[tid] = (float)((double)a.mscale * s);
    }
    // of two tokens with one slot the later one's row stays
    int keep = a.k && slot >= 0 && slot < a.n_slot;
    if (keep)
        for (int u = t + 1 + tid; u < a.n_tok; u += 256) keep &= (a.slot ? a.slot[u] : a.pos[u]) != slot;
    keep = __syncthreads_and(keep);
    const int n_q = a.q ? a.n_head : 0, n_k = keep ? a.n_kv_head : 0;
    float *buf = heads[wave];
    for (int h = wave; h < n_q + n_k; h += 4) {
        const bool is_q = h < n_q;
        const int g = h - n_q;
        const float *src = is_q ? a.q + (size_t)t * a.q_stride + (size_t)h * a.hd
                                : a.k + (size_t)t * a.k_stride + (size_t)g * a.hd;
        const float *nw = is_q ? a.q_norm : a.k_norm;
        double ss = 0.0;
        for (int i = lane; i < a.hd; i += 64) {
            buf[i] = src[i];
            ss += (double)buf[i] * (double)buf[i];
        }
        if (nw) {
            ss = sdy_wave_sum_f64(ss);
            const float sc = (float)(1.0 / sqrt(ss / (double)a.hd + (double)a.eps));
            for (int i = lane; i < a.hd; i += 64) buf[i] = buf[i] * sc * nw[i];
        }
        sdy_wave_sync();
        for (int i = lane; i < half; i += 64) {
            const int ia = a.interleaved ? 2 * i : i, ib = a.interleaved ? 2 * i + 1 : i + half;
            const float x = buf[ia], y = buf[ib];
            const float xc = x * cs[i], ys = y * sn[i], xs = x * sn[i], yc = y * cs[i];
            buf[ia] = xc - ys;
            buf[ib] = xs + yc;
        }
        sdy_wave_sync();
        if (is_q) {
            float *dst = a.q_out + (size_t)t * a.q_out_stride + (size_t)h * a.hd;
            for (int i = lane; i < a.hd; i += 64) dst[i] = buf[i];
        } else {
            KT *kr = (KT *)a.k_rows + (size_t)g * a.head_stride + (size_t)slot * a.hd;
            KT *vr = (KT *)a.v_rows + (size_t)g * a.head_stride + (size_t)slot * a.hd;
            const float *v = a.v + (size_t)t * a.v_stride + (size_t)g * a.hd;
            for (int i = lane; i < a.hd; i += 64) {
                KvElt<KT>::st(kr, i, buf[i]);
                KvElt<KT>::st(vr, i, v[i]);
            }
        }
        sdy_wave_sync();
    }
}

}  // namespace

extern "C" int sdy_qk_rope_at(const sdy_rope_at_args *a, sdy_stream s) {
    if (!a) return sdy_fail(-1, "qk_rope_at: no arguments");
    if (a->n_tok < 0) return sdy_fail(-1, "qk_rope_at: n_tok %d", a->n_tok);
    if (a->n_tok == 0) return 0;
    if (a->hd < 2 || a->hd > 512 || a->hd % 2) return sdy_fail(-1, "qk_rope_at: head_dim %d (even, 2..512)", a->hd);
    if (a->n_rot < 0 || a->n_rot > a->hd || a->n_rot % 2)
        return sdy_fail(-1, "qk_rope_at: n_rot %d (even, 0..head_dim %d)", a->n_rot, a->hd);
    if (!sdy_kv_elt_bytes(a->kv_type)) return sdy_fail(-1, "qk_rope_at: KV type %d", a->kv_type);
    if (!a->q && !a->k) return sdy_fail(-1, "qk_rope_at: neither q nor k");
    if (!a->pos || (a->n_rot && !a->freq)) return sdy_fail(-1, "qk_rope_at: pos and freq are needed");
    if (a->q && (a->n_head < 1 || !a->q_out)) return sdy_fail(-1, "qk_rope_at: q needs n_head (%d) and q_out", a->n_head);
    if (a->k && (a->n_kv_head < 1 || !a->v || !a->k_rows || !a->v_rows))
        return sdy_fail(-1, "qk_rope_at: k needs n_kv_head (%d), v, k_rows and v_rows", a->n_kv_head);
    if (a->k && (a->n_slot < 0 || (a->n_kv_head > 1 && a->head_stride < (long)a->n_slot * a->hd)))
        return sdy_fail(-1, "qk_rope_at: %d slots of %d need a head stride of as many elements (%ld)", a->n_slot, a->hd,
                        a->head_stride);
    // rows may share memory only where they are the same rows: a token's heads are written while others are read
    if (a->q && a->q_out == a->q && a->q_out_stride != a->q_stride)
        return sdy_fail(-1, "qk_rope_at: q in place needs q_out_stride %ld to be q_stride %ld", a->q_out_stride, a->q_stride);
    if (a->kv_type == SDY_KV_F16)
        hipLaunchKernelGGL(k_qk_rope_at<uint16_t>, dim3(a->n_tok), dim3(256), 0, (hipStream_t)s, *a);
    else
        hipLaunchKernelGGL(k_qk_rope_at<float>, dim3(a->n_tok), dim3(256), 0, (hipStream_t)s, *a);
    return sdy_check_launch("qk_rope_at");
}
