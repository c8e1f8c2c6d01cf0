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

// The token's slot, or -1 where this workgroup is to write no rows: of two tokens with one slot the later one's row stays.
// All 256 threads compare the slots behind it, n_tok^2 / 2 in all: not seen beside the rows up to some 16384 tokens (3 heads of 64
// 60 us, 48 of 128 199 with 144 for the bytes alone), 0.6 of 1.4 ms at 65536. Four slots to a load took twice as long.
SDY_DEV long slot_of(const sdy_rope_at_args &a, int t) {
    const long slot = a.slot ? a.slot[t] : a.pos[t];
    int keep = a.k && slot >= 0 && slot < a.n_slot;
    if (keep)
        for (int u = t + 1 + (int)threadIdx.x; u < a.n_tok; u += 256) keep &= (a.slot ? a.slot[u] : a.pos[u]) != slot;
    return __syncthreads_and(keep) ? slot : -1;
}

// Heads of 32, 64, 128 or 256 dims in aligned rows: HD / 4 lanes to a row of q, k or v, four dims each. A workgroup takes
// `rows` rows of one token, 256 / (HD / 4) at a time, the next ones' loads in flight. Bound by memory: 2048 tokens of 32 + 8
// heads of 128 dims with f16 rows, 92 MB, 17.9 us, 5.2 TB/s (k_rope_any: 20.7; heads of 32 dims 17.8 against 42.9, of 64 18.0
// against 25.7, of 256 18.1 against 20.1). One token takes 3.6 us (9.1), of which a launch is 1.5 and two dependent loads and
// the sine most of the rest.
template <int HD, class KT>
__global__ __launch_bounds__(256) void k_rope_rows(sdy_rope_at_args a, int rows) {
    constexpr int L = HD / 4, RPP = 256 / L;
    __shared__ __align__(16) float cs[HD / 2], sn[HD / 2];
    const int t = blockIdx.x, tid = threadIdx.x, c = tid % L, d = 4 * c;
    const int half = a.n_rot / 2;
    const int n_q = a.q ? a.n_head : 0, n_k = a.k ? a.n_kv_head : 0, all = n_q + 2 * n_k;
    const int r0 = blockIdx.y * rows + tid / L, end = (int)(blockIdx.y + 1) * rows < all ? (int)(blockIdx.y + 1) * rows : all;
    auto load = [&](int r) {
        if (r >= end) return make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const float *src = r < n_q         ? a.q + (size_t)t * a.q_stride + (size_t)r * HD
                           : r < n_q + n_k ? a.k + (size_t)t * a.k_stride + (size_t)(r - n_q) * HD
                                           : a.v + (size_t)t * a.v_stride + (size_t)(r - n_q - n_k) * HD;
        return *reinterpret_cast<const float4 *>(src + d);
    };
    float4 x = load(r0);
    const int pos = a.pos[t];
    if (tid < half) {
        double s, c2;
        sincos_f64((double)pos * a.freq[tid], &s, &c2);
        cs[tid] = (float)((double)a.mscale * c2);
        sn[tid] = (float)((double)a.mscale * s);
    }
    long slot = -1;
    if (end > n_q) slot = slot_of(a, t);
    else __syncthreads();
    for (int r = r0; r - tid / L < end; r += RPP) {
        const float4 next = load(r + RPP);
        const bool is_q = r < n_q, is_v = r >= n_q + n_k;
        const float *nw = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
        if (a.q_norm || a.k_norm) {
            double ss = ((double)x.x * (double)x.x + (double)x.y * (double)x.y) + ((double)x.z * (double)x.z + (double)x.w * (double)x.w);
#pragma unroll
            for (int off = L / 2; off >= 1; off /= 2) ss += __shfl_xor(ss, off);
            if (nw) {
                const float sc = (float)(1.0 / sqrt(ss / (double)HD + (double)a.eps));
                const float4 w = *reinterpret_cast<const float4 *>(nw + d);
                x = make_float4(x.x * sc * w.x, x.y * sc * w.y, x.z * sc * w.z, x.w * sc * w.w);
            }
        }
        float4 y = x;
        if (a.interleaved) {
            if (d < a.n_rot && !is_v) {
                const float2 co = *reinterpret_cast<const float2 *>(cs + d / 2), si = *reinterpret_cast<const float2 *>(sn + d / 2);
                const float ac = x.x * co.x, bs = x.y * si.x, as = x.x * si.x, bc = x.y * co.x;
                const float ec = x.z * co.y, fs = x.w * si.y, es = x.z * si.y, fc = x.w * co.y;
                y = make_float4(ac - bs, as + bc, ec - fs, es + fc);
            }
        } else {
            const bool low = d < half;
            const int from = (tid & 63 & ~(L - 1)) + (low ? c + half / 4 : d < a.n_rot ? c - half / 4 : c);
            const float4 o = make_float4(__shfl(x.x, from), __shfl(x.y, from), __shfl(x.z, from), __shfl(x.w, from));
            if (d < a.n_rot && !is_v) {
                const int i = low ? d : d - half;
                const float4 co = *reinterpret_cast<const float4 *>(cs + i), si = *reinterpret_cast<const float4 *>(sn + i);
                const float4 xc = make_float4(x.x * co.x, x.y * co.y, x.z * co.z, x.w * co.w);
                const float4 os = make_float4(o.x * si.x, o.y * si.y, o.z * si.z, o.w * si.w);
                // a c - b s for the first of a pair, a s + b c for the second
                y = low ? make_float4(xc.x - os.x, xc.y - os.y, xc.z - os.z, xc.w - os.w)
                        : make_float4(os.x + xc.x, os.y + xc.y, os.z + xc.z, os.w + xc.w);
            }
        }
        if (r < end) {
            if (is_q) {
                *reinterpret_cast<float4 *>(a.q_out + (size_t)t * a.q_out_stride + (size_t)r * HD + d) = y;
            } else if (slot >= 0) {
                KT *dst = (KT *)(is_v ? a.v_rows : a.k_rows) + (size_t)(r - n_q - (is_v ? n_k : 0)) * a.head_stride + (size_t)slot * HD + d;
                if constexpr (KvElt<KT>::BYTES == 4)
                    *reinterpret_cast<float4 *>(dst) = y;
                else
                    *reinterpret_cast<uint2 *>(dst) = make_uint2(sdy_f2h(y.x) | (uint32_t)sdy_f2h(y.y) << 16, sdy_f2h(y.z) | (uint32_t)sdy_f2h(y.w) << 16);
            }
        }
        x = next;
    }
}

// Any even head: one workgroup per token, one wave per head of q or k (with its v), the head in LDS.
template <class KT>
__global__ __launch_bounds__(256) void k_rope_any(sdy_rope_at_args a) {
    __shared__ float cs[256], sn[256], heads[4][512];
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int half = a.n_rot / 2;
    const int pos = a.pos[t];
    if (tid < half) {
        double s, c;
        sincos_f64((double)pos * a.freq[tid], &s, &c);
        cs[tid] = (float)((double)a.mscale * c);
        sn[tid] = (float)((double)a.mscale * s);
    }
    const long slot = slot_of(a, t);
    const int n_q = a.q ? a.n_head : 0, n_k = slot >= 0 ? a.n_kv_head : 0;
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

// Few tokens: a workgroup for every 256 lanes' rows; where that would be more than 2048 of them, one per token, which makes
// a token's sines once (against split, 32 + 8 heads of 128 dims: 1 token 6.0 against 3.6 us, 61 6.6 against 4.2, 200 7.0
// against 5.3, 400 7.8 against 7.2, 2048 17.8 against 20.7).
template <int HD, class KT>
int launch_rows(const sdy_rope_at_args &a, hipStream_t st) {
    constexpr int RPP = 256 / (HD / 4);
    const int all = (a.q ? a.n_head : 0) + (a.k ? 2 * a.n_kv_head : 0), parts = (all + RPP - 1) / RPP;
    const bool few = (long)a.n_tok * parts <= 2048 && parts <= 65535;
    hipLaunchKernelGGL((k_rope_rows<HD, KT>), dim3(a.n_tok, few ? parts : 1), dim3(256), 0, st, a, few ? RPP : all);
    return sdy_check_launch("qk_rope_at");
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
    if (a->q && a->n_tok > 1 && a->q_out_stride < (long)a->n_head * a->hd)
        return sdy_fail(-1, "qk_rope_at: rows of %d heads %ld apart in q_out", a->n_head, a->q_out_stride);
    hipStream_t st = (hipStream_t)s;
    const bool f16 = a->kv_type == SDY_KV_F16;
    // rows of float4 (and of 4 stored values), no four dims half turned
    const bool wide = (a->hd == 32 || a->hd == 64 || a->hd == 128 || a->hd == 256) && a->n_rot % (a->interleaved ? 4 : 8) == 0 &&
                      (!a->q || !(((uintptr_t)a->q | (uintptr_t)a->q_out) & 15 || (a->q_stride | a->q_out_stride) & 3)) &&
                      (!a->k || !(((uintptr_t)a->k | (uintptr_t)a->v) & 15 || (a->k_stride | a->v_stride | a->head_stride) & 3 ||
                                  ((uintptr_t)a->k_rows | (uintptr_t)a->v_rows) & (f16 ? 7 : 15))) &&
                      !(((uintptr_t)a->q_norm | (uintptr_t)a->k_norm) & 15);
    if (wide) {
        switch (a->hd) {
            case 32: return f16 ? launch_rows<32, uint16_t>(*a, st) : launch_rows<32, float>(*a, st);
            case 64: return f16 ? launch_rows<64, uint16_t>(*a, st) : launch_rows<64, float>(*a, st);
            case 128: return f16 ? launch_rows<128, uint16_t>(*a, st) : launch_rows<128, float>(*a, st);
            default: return f16 ? launch_rows<256, uint16_t>(*a, st) : launch_rows<256, float>(*a, st);
        }
    }
    if (f16) hipLaunchKernelGGL(k_rope_any<uint16_t>, dim3(a->n_tok), dim3(256), 0, st, *a);
    else hipLaunchKernelGGL(k_rope_any<float>, dim3(a->n_tok), dim3(256), 0, st, *a);
    return sdy_check_launch("qk_rope_at");
}
