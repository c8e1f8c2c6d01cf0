// A token per row of logits: temperature, top-k, top-p and min-p, from a given uniform number.
//
// A row's tokens stand in the order of their logits, the greatest first and of equal ones the lowest index (NaN counts as
// -inf). w_i = exp((x_i - max x) / T). Kept are the first top_k; of these the shortest prefix whose sum reaches top_p of
// theirs; of these the ones with w_i >= min_p; the first always. The token is the first one, by index, at which the running
// sum of the kept w exceeds u times their whole. T <= 0 keeps the first alone.
//
// The w are made in 64 bits and summed as whole multiples of 2^-S (S = 62 - ceil log2 n_vocab: 2^-44 for 151936 tokens): sums
// of integers, so no order of adding, split or atomic changes a token. A w below 2^-S, 30 T under the greatest logit for that
// vocabulary, is never chosen.
#include "sdy_device.h"
#include "sdy_internal.h"
#include "sdy_ops.h"

namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int MAX_VOCAB = 1 << 22;  // a token's place in the order fits 32 + 22 bits

// A logit's place in the order: 32 bits that grow with x (-0 as 0, NaN as -inf), then 22 that fall with the index.
SDY_DEV uint64_t place_of(float x, int i) {
    x = x == x ? x + 0.0f : -INFINITY;
    const uint32_t b = __float_as_uint(x);
    const uint32_t k = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (uint64_t)k << 22 | (uint64_t)(MAX_VOCAB - 1 - i);
}

struct Row {
    const float *x;
    int n;
    float best;       // the greatest logit
    double inv_t;
    double one;       // 2^S
    // w as a whole number of 2^-S
    SDY_DEV double weight(float v) const {
        if (v == best) return 1.0;
        if (!(v > -INFINITY) || best == INFINITY) return 0.0;
        return exp(((double)v - (double)best) * inv_t);
    }
    SDY_DEV uint64_t fixed(float v) const { return (uint64_t)(weight(v) * one); }
};

struct Shared {
    unsigned count[2048];
    unsigned long long sum[2048];
    unsigned long long part[WAVES];
    unsigned long long found, before;
};

SDY_DEV uint64_t wave_sum(uint64_t v) {
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor((unsigned long long)v, off);
    return v;
}

SDY_DEV uint64_t block_sum(uint64_t v, Shared &sh) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.part[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t r = 0;
    for (int w = 0; w < WAVES; w++) r += sh.part[w];
    return r;
}

SDY_DEV uint64_t block_max(uint64_t v, Shared &sh) {
    for (int off = 32; off >= 1; off >>= 1) {
        const uint64_t o = __shfl_xor((unsigned long long)v, off);
        v = o > v ? o : v;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.part[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t r = 0;
    for (int w = 0; w < WAVES; w++) r = sh.part[w] > r ? sh.part[w] : r;
    return r;
}

// The place of the last token of the shortest prefix, among tokens from place `least` on, that has `want` tokens
// (by_sum false) or a sum of `want` (true): 54 bits, 11 at a time from the top.
SDY_DEV uint64_t prefix_end(const Row &r, uint64_t least, bool by_sum, uint64_t want, Shared &sh) {
    uint64_t head = 0, before = 0;
    for (int shift = 44; shift > -11; shift -= 11) {
        const int s = shift < 0 ? 0 : shift, bits = shift < 0 ? 11 + shift : 11;
        __syncthreads();
        for (int i = threadIdx.x; i < 2048; i += THREADS) sh.count[i] = 0, sh.sum[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < r.n; i += THREADS) {
            const float v = r.x[i];
            const uint64_t at = place_of(v, i);
            if (at < least || at >> (s + bits) != head) continue;
            const int d = (int)(at >> s) & ((1 << bits) - 1);
            if (by_sum) atomicAdd(&sh.sum[d], (unsigned long long)r.fixed(v));
            else atomicAdd(&sh.count[d], 1u);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint64_t sum = before;
            int d = (1 << bits) - 1;
            for (; d > 0; d--) {
                const uint64_t more = by_sum ? sh.sum[d] : sh.count[d];
                if (sum + more >= want) break;
                sum += more;
            }
            sh.found = d;
            sh.before = sum;
        }
        __syncthreads();
        head = head << bits | sh.found;
        before = sh.before;
    }
    return head;
}

__global__ __launch_bounds__(THREADS) void k_sample_row(sdy_sample_args a, int shift) {
    __shared__ Shared sh;
    const int row = blockIdx.x, tid = threadIdx.x;
    Row r;
    r.x = a.logits + (size_t)row * a.stride;
    r.n = a.n_vocab;
    r.one = __longlong_as_double((1023ll + shift) << 52);
    uint64_t first = 0;
    for (int i = tid; i < r.n; i += THREADS) {
        const uint64_t at = place_of(r.x[i], i);
        first = at > first ? at : first;
    }
    first = block_max(first, sh);
    const int i_first = MAX_VOCAB - 1 - (int)(first & (MAX_VOCAB - 1));
    r.best = r.x[i_first];
    const bool none = !(r.best > -INFINITY);
    const float temp = a.temp ? a.temp[row] : 1.0f;
    if (none || !(temp > 0.0f)) {
        if (tid == 0) {
            a.token[row] = none ? -1 : i_first;
            if (a.prob) a.prob[row] = none ? 0.0f : 1.0f;
        }
        return;
    }
    r.inv_t = 1.0 / (double)temp;
    const int top_k = a.top_k ? a.top_k[row] : 0;
    const float top_p = a.top_p ? a.top_p[row] : 1.0f, min_p = a.min_p ? a.min_p[row] : 0.0f;
    uint64_t least = 0;
    if (top_k > 0 && top_k < r.n) least = prefix_end(r, 0, false, (uint64_t)top_k, sh);
    if (top_p < 1.0f) {
        uint64_t sum = 0;
        for (int i = tid; i < r.n; i += THREADS)
            if (place_of(r.x[i], i) >= least) sum += r.fixed(r.x[i]);
        sum = block_sum(sum, sh);
        const double want = ceil((double)top_p * (double)sum);
        least = prefix_end(r, least, true, want > 1.0 ? (uint64_t)want : 1, sh);
    }
    // the kept ones' sums: of the row, then of ever smaller pieces of it
    auto kept = [&](int i) -> uint64_t {
        const float v = r.x[i];
        const uint64_t at = place_of(v, i);
        if (at < least) return 0;
        const double w = r.weight(v);
        return at == first || !(w < (double)min_p) ? (uint64_t)(w * r.one) : 0;
    };
    uint64_t whole = 0;
    for (int i = tid; i < r.n; i += THREADS) whole += kept(i);
    whole = block_sum(whole, sh);
    const float u = a.u[row];
    uint64_t left = u > 0.0f ? (uint64_t)((double)u * (double)whole) : 0;  // (a u beyond 2^62 / whole: clamped below)
    if (!(u < 1.0f) || left >= whole) left = u > 0.0f ? whole - 1 : 0;
    int lo = 0, hi = r.n;
    while (hi - lo > 1) {  // the piece in which the running sum passes `left`
        const int wave = tid >> 6, len = (hi - lo + WAVES - 1) / WAVES;
        const int b = lo + wave * len < hi ? lo + wave * len : hi, e = b + len < hi ? b + len : hi;
        uint64_t sum = 0;
        for (int i = b + (tid & 63); i < e; i += 64) sum += kept(i);
        sum = wave_sum(sum);
        __syncthreads();
        if ((tid & 63) == 0) sh.part[wave] = sum;
        __syncthreads();
        int w = 0;
        while (w < WAVES - 1 && sh.part[w] <= left) left -= sh.part[w++];
        lo = lo + w * len;
        hi = lo + len < hi ? lo + len : hi;
    }
    if (tid == 0) {
        a.token[row] = lo;
        if (a.prob) a.prob[row] = (float)((double)kept(lo) / (double)whole);
    }
}

}  // namespace

extern "C" size_t sdy_sample_ws_bytes(int n_rows, int n_vocab) {
    if (n_rows < 1 || n_vocab < 1 || n_vocab > MAX_VOCAB) return 0;
    return 256;
}

extern "C" int sdy_sample(const sdy_sample_args *a, sdy_stream s) {
    if (!a) return sdy_fail(-1, "sample: no arguments");
    if (a->n_rows < 0) return sdy_fail(-1, "sample: n_rows %d", a->n_rows);
    if (a->n_rows == 0) return 0;
    if (a->n_vocab < 1 || a->n_vocab > MAX_VOCAB) return sdy_fail(-1, "sample: n_vocab %d (1..%d)", a->n_vocab, MAX_VOCAB);
    if (a->n_rows > 1 && a->stride < a->n_vocab)
        return sdy_fail(-1, "sample: rows of %d logits %ld apart", a->n_vocab, a->stride);
    if (!a->logits || !a->u || !a->token || !a->ws) return sdy_fail(-1, "sample: logits, u, token and ws are needed");
    if ((uintptr_t)a->ws & 15) return sdy_fail(-1, "sample: ws aligned to 16 bytes");
    int log2 = 0;
    while ((1 << log2) < a->n_vocab) log2++;
    hipLaunchKernelGGL(k_sample_row, dim3(a->n_rows), dim3(THREADS), 0, (hipStream_t)s, *a, 62 - log2);
    return sdy_check_launch("sample");
}
