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
//
// Every kept set is a prefix of the order, so what is looked for is where it ends, without sorting the row. The row is cut
// into pieces, a workgroup each (as many as fill the GPU), and read three times, the second and third from the caches:
//   k_sample_max   each piece's greatest and lowest logit;
//   k_sample_bins  each piece's tokens counted, and their w added, by distance from the greatest logit in 1024 bins;
//   k_sample_list  from the bins, the one in which the prefix ends (with a small top_k all up to there): its tokens;
//   k_sample_pick  one workgroup per row: these tokens sorted, the prefix's end among them, the pieces' sums, and the token
//                  in its piece. A row whose end lies among more than 4096 tokens (nearly equal logits) is searched digit by
//                  digit instead.
#include "sdy_device.h"
#include "sdy_internal.h"
#include "sdy_ops.h"

namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int MAX_VOCAB = 1 << 22;  // a token's place in the order fits 32 + 22 bits
constexpr int BINS = THREADS;       // a thread each
constexpr int LIST = 4096;          // tokens that are sorted
constexpr int SMALL_K = 1024;       // up to here the bins' sums are not made: the first top_k tokens are listed themselves
constexpr int MAX_PIECES = 16;

// A logit's place in the order: 32 bits that grow with x (-0 as 0, NaN as -inf), then 22 that fall with the index.
SDY_DEV float value_at(uint64_t place) {
    const uint32_t k = (uint32_t)(place >> 22);
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
SDY_DEV int index_at(uint64_t place) { return MAX_VOCAB - 1 - (int)(place & (MAX_VOCAB - 1)); }
SDY_DEV uint64_t place_of(float x, int i) {
    x = x == x ? x + 0.0f : -INFINITY;
    const uint32_t b = __float_as_uint(x);
    const uint32_t k = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (uint64_t)k << 22 | (uint64_t)(MAX_VOCAB - 1 - i);
}

// What the kernels leave for each other, per row.
struct Work {
    unsigned long long first[MAX_PIECES];  // the greatest place
    unsigned long long sums[MAX_PIECES];   // kept w before the listed bins
    float low[MAX_PIECES];                 // the lowest finite logit
    int mode, n_list, bin_k, pad;
    unsigned long long before;             // count or sum before the listed bins
    unsigned long long want;               // the sum that the prefix has to reach
    unsigned long long list[LIST];
};
// after them: per row and piece, BINS counts; then BINS sums

enum { ROW_ALONE = 0,  // the first token, or none
       ROW_ALL,        // nothing is left out
       ROW_TOP,        // the listed tokens hold the whole prefix
       ROW_SUM,        // the prefix ends by its sum (or min-p) in the listed bins
       ROW_COUNT,      // the first top_k tokens end in the listed bin
       ROW_SLOW,       // it ends among too many tokens to list
       ROW_KNOWN };    // where it ends has been found

struct Args {
    sdy_sample_args a;
    int shift;    // S
    int pieces, len;
    Work *work;
    unsigned *count;           // [n_rows][pieces][BINS]
    unsigned long long *sum;   // [n_rows][pieces][BINS]
};

struct Row {
    const float *x;
    int n;
    uint64_t first;   // the greatest place
    float best;       // its logit
    float temp, top_p, min_p;
    int top_k;
    double inv_t;
    double one;       // 2^S
    float per_bin;    // bins per unit of logit
    bool alone, none;
    SDY_DEV void params(const Args &A, int row) {
        const sdy_sample_args &a = A.a;
        x = a.logits + (size_t)row * a.stride;
        n = a.n_vocab;
        temp = a.temp ? a.temp[row] : 1.0f;
        top_k = a.top_k ? a.top_k[row] : 0;
        if (top_k <= 0 || top_k >= n) top_k = 0;
        top_p = a.top_p ? a.top_p[row] : 1.0f;
        if (!(top_p < 1.0f)) top_p = 1.0f;
        min_p = a.min_p ? a.min_p[row] : 0.0f;
        if (!(min_p > 0.0f)) min_p = 0.0f;
        one = __longlong_as_double((1023ll + A.shift) << 52);
    }
    SDY_DEV void maxima(const Args &A, int row) {
        const Work &w = A.work[row];
        first = 0;
        float low = INFINITY;
        for (int c = 0; c < A.pieces; c++) {
            first = w.first[c] > first ? w.first[c] : first;
            low = fminf(low, w.low[c]);
        }
        best = value_at(first);
        none = !(best > -INFINITY);
        alone = none || !(temp > 0.0f);
        inv_t = 1.0 / (double)temp;
        // over the whole of the finite logits, or as far down as a w counts (2^-62 is exp(-43))
        const float range = fminf(best - low, 43.0f * temp);
        per_bin = range > 0.0f ? (float)BINS / range : 0.0f;
    }
    SDY_DEV bool cut() const { return top_k || top_p < 1.0f || min_p > 0.0f; }
    SDY_DEV double weight(float v) const {
        if (v == best) return 1.0;
        if (!(v > -INFINITY) || best == INFINITY) return 0.0;
        return exp(((double)v - (double)best) * inv_t);
    }
    SDY_DEV uint64_t fixed(float v) const { return (uint64_t)(weight(v) * one); }  // w as a whole number of 2^-S
    // never less for a lower logit
    SDY_DEV int bin(float v) const { return v == best ? 0 : (int)fminf((best - v) * per_bin, (float)(BINS - 1)); }
};

// f(logit, index) of the tokens [lo, hi), eight loads in flight
template <class F>
SDY_DEV void each(const float *x, int lo, int hi, const F &f) {
    for (int i0 = lo + (int)threadIdx.x; i0 < hi; i0 += 8 * THREADS) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; u++) v[u] = x[i0 + u * THREADS < hi ? i0 + u * THREADS : hi - 1];
#pragma unroll
        for (int u = 0; u < 8; u++)
            if (i0 + u * THREADS < hi) f(v[u], i0 + u * THREADS);
    }
}

struct Shared {
    float low[WAVES];
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

// The sum over the threads before this one; *whole the sum over all.
SDY_DEV uint64_t block_scan(uint64_t v, uint64_t *whole, Shared &sh) {
    uint64_t run = v;
    for (int off = 1; off < 64; off *= 2) {
        const uint64_t o = __shfl_up((unsigned long long)run, off);
        if ((int)(threadIdx.x & 63) >= off) run += o;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.part[threadIdx.x >> 6] = run;
    __syncthreads();
    uint64_t before = 0, all = 0;
    for (int w = 0; w < WAVES; w++) {
        if (w < (int)(threadIdx.x >> 6)) before += sh.part[w];
        all += sh.part[w];
    }
    *whole = all;
    return before + run - v;
}

__global__ __launch_bounds__(THREADS) void k_sample_max(Args A) {
    __shared__ Shared sh;
    const int c = blockIdx.x, row = blockIdx.y;
    const float *x = A.a.logits + (size_t)row * A.a.stride;
    const int lo = c * A.len, hi = lo + A.len < A.a.n_vocab ? lo + A.len : A.a.n_vocab;
    uint64_t first = 0;
    float low = INFINITY;
    each(x, lo, hi, [&](float v, int i) {
        const uint64_t at = place_of(v, i);
        first = at > first ? at : first;
        if (v > -INFINITY) low = fminf(low, v);
    });
    for (int off = 32; off >= 1; off >>= 1) low = fminf(low, __shfl_xor(low, off));
    if ((threadIdx.x & 63) == 0) sh.low[threadIdx.x >> 6] = low;
    first = block_max(first, sh);
    if (threadIdx.x == 0) {
        for (int w = 0; w < WAVES; w++) low = fminf(low, sh.low[w]);
        A.work[row].first[c] = first;
        A.work[row].low[c] = low;
    }
}

__global__ __launch_bounds__(THREADS) void k_sample_bins(Args A) {
    __shared__ Shared sh;
    const int c = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
    Row r;
    r.params(A, row);
    r.maxima(A, row);
    if (r.alone) return;
    const int lo = c * A.len, hi = lo + A.len < r.n ? lo + A.len : r.n;
    if (!r.cut()) {
        uint64_t sum = 0;
        each(r.x, lo, hi, [&](float v, int) { sum += r.fixed(v); });
        sum = block_sum(sum, sh);
        if (tid == 0) A.work[row].sums[c] = sum;
        return;
    }
    const bool sums = !r.top_k || r.top_k > SMALL_K;
    sh.count[tid] = 0;
    sh.sum[tid] = 0;
    __syncthreads();
    each(r.x, lo, hi, [&](float v, int) {
        if (!(v > -INFINITY)) return;
        const int b = r.bin(v);
        atomicAdd(&sh.count[b], 1u);
        if (sums) atomicAdd(&sh.sum[b], (unsigned long long)r.fixed(v));
    });
    __syncthreads();
    const size_t at = ((size_t)row * A.pieces + c) * BINS + tid;
    A.count[at] = sh.count[tid];
    if (sums) A.sum[at] = sh.sum[tid];
}

// The row's bins: this thread's count, sum, and the count in the pieces before c.
SDY_DEV void bins_of(const Args &A, int row, int c, bool sums, unsigned *count, unsigned *before, uint64_t *sum) {
    unsigned n = 0, nb = 0;
    uint64_t w = 0;
    const size_t at = (size_t)row * A.pieces * BINS + threadIdx.x;
    for (int p = 0; p < A.pieces; p++) {
        const unsigned x = A.count[at + (size_t)p * BINS];
        n += x;
        if (p < c) nb += x;
        if (sums) w += A.sum[at + (size_t)p * BINS];
    }
    *count = n;
    *before = nb;
    *sum = w;
}

// The least sum that reaches top_p of the whole
SDY_DEV uint64_t wanted(float top_p, uint64_t whole) {
    const double want = ceil((double)top_p * (double)whole);
    return want > 1.0 ? (uint64_t)want : 1;
}

// The first bin up to which there are `want` of v (the last one with any if there are fewer), and what is before it.
SDY_DEV int bin_that_reaches(uint64_t v, uint64_t want, uint64_t *before, Shared &sh) {
    uint64_t whole;
    const uint64_t b = block_scan(v, &whole, sh);
    if (want > whole) want = whole;
    if (threadIdx.x == 0) sh.found = 0, sh.before = 0;
    __syncthreads();
    if (v && b < want && b + v >= want) sh.found = threadIdx.x, sh.before = b;
    __syncthreads();
    *before = sh.before;
    const int f = (int)sh.found;
    __syncthreads();
    return f;
}

__global__ __launch_bounds__(THREADS) void k_sample_list(Args A) {
    __shared__ Shared sh;
    __shared__ unsigned n_mine;
    const int c = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
    Work &w = A.work[row];
    Row r;
    r.params(A, row);
    r.maxima(A, row);
    if (r.alone || !r.cut()) {
        if (c == 0 && tid == 0) w.mode = r.alone ? ROW_ALONE : ROW_ALL;
        return;
    }
    const bool sums = !r.top_k || r.top_k > SMALL_K;
    unsigned count, mine_before;
    uint64_t sum;
    bins_of(A, row, c, sums, &count, &mine_before, &sum);
    int b0 = 0, b1 = BINS - 1, mode = ROW_SUM, bk = 0;
    uint64_t before = 0, want = ~0ull;
    if (r.top_k) {
        bk = bin_that_reaches(count, (uint64_t)r.top_k, &before, sh);
        uint64_t all;
        block_scan(tid <= bk ? count : 0, &all, sh);
        b1 = bk;
        mode = ROW_TOP;
        if (all > LIST) {
            b0 = bk;
            mode = sums ? ROW_COUNT : ROW_SLOW;
        } else {
            before = 0;
        }
    } else {
        if (r.top_p < 1.0f) {
            uint64_t whole;
            block_scan(sum, &whole, sh);
            want = wanted(r.top_p, whole);
            b0 = b1 = bin_that_reaches(sum, want, &before, sh);
        }
        if (r.min_p > 0.0f) {
            // the bins that the border can be in: their arithmetic is in 32 bits
            const float far = r.min_p < 1.0f ? -logf(r.min_p) * r.temp * r.per_bin : 0.0f;
            const int lo = (int)fminf(far * (1.0f - 1e-5f), (float)(BINS - 1));
            const int hi = (int)fminf(far * (1.0f + 1e-5f) + 1e-5f, (float)(BINS - 1));
            b0 = r.top_p < 1.0f && b0 < lo ? b0 : lo;
            b1 = hi < b1 ? hi : b1;
        }
        uint64_t b = block_sum(tid < b0 ? sum : 0, sh);
        before = b;
    }
    uint64_t listed;
    const bool in = tid >= b0 && tid <= b1;
    listed = block_sum(in ? count : 0, sh);
    const uint64_t offset = block_sum(in ? mine_before : 0, sh);
    const uint64_t above = block_sum(sums && tid < b0 ? A.sum[((size_t)row * A.pieces + c) * BINS + tid] : 0, sh);
    if (listed > LIST) mode = ROW_SLOW;
    if (tid == 0) {
        w.sums[c] = above;
        n_mine = (unsigned)offset;
        if (c == 0) {
            w.mode = mode;
            w.n_list = (int)listed;
            w.bin_k = bk;
            w.before = before;
            w.want = want;
        }
    }
    if (mode == ROW_SLOW) return;
    __syncthreads();
    const int lo = c * A.len, hi = lo + A.len < r.n ? lo + A.len : r.n;
    each(r.x, lo, hi, [&](float v, int i) {
        if (!(v > -INFINITY)) return;
        const int b = r.bin(v);
        if (b >= b0 && b <= b1) w.list[atomicAdd(&n_mine, 1u)] = place_of(v, i);
    });
}

// list[0 .. n) in falling order (a power of two from n on is sorted, padded with zeros)
SDY_DEV void sort_falling(unsigned long long *list, int n) {
    int n2 = 1;
    while (n2 < n) n2 *= 2;
    for (int i = n + threadIdx.x; i < n2; i += THREADS) list[i] = 0;
    __syncthreads();
    for (int k = 2; k <= n2; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            for (int t = threadIdx.x; t < n2 / 2; t += THREADS) {
                const int i = (t / j) * 2 * j + t % j;
                const unsigned long long x = list[i], y = list[i + j];
                if ((x < y) == ((i & k) == 0)) list[i] = y, list[i + j] = x;
            }
            __syncthreads();
        }
}

// The piece [lo, hi) narrowed to the token at which the running sum of kept(i) passes `left`
template <class F>
SDY_DEV int narrow(int lo, int hi, uint64_t left, const F &kept, Shared &sh) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    while (hi - lo > 1) {
        const int len = (hi - lo + WAVES - 1) / WAVES;
        const int b = lo + wave * len < hi ? lo + wave * len : hi, e = b + len < hi ? b + len : hi;
        uint64_t sum = 0;
        for (int i = b + lane; i < e; i += 64) sum += kept(i);
        sum = wave_sum(sum);
        __syncthreads();
        if (lane == 0) sh.part[wave] = sum;
        __syncthreads();
        int w = 0;
        while (w < WAVES - 1 && sh.part[w] <= left) left -= sh.part[w++];
        lo = lo + w * len;
        hi = lo + len < hi ? lo + len : hi;
    }
    return lo;
}

// u of the whole, in 0 .. whole - 1
SDY_DEV uint64_t share(float u, uint64_t whole) {
    if (!(u > 0.0f)) return 0;
    if (u >= 1.0f) return whole - 1;
    const uint64_t t = (uint64_t)((double)u * (double)whole);
    return t < whole ? t : whole - 1;
}

__global__ __launch_bounds__(THREADS) void k_sample_pick(Args A) {
    __shared__ Shared sh;
    __shared__ unsigned long long list[LIST];
    __shared__ unsigned long long sums[MAX_PIECES];
    __shared__ int n_list;
    const sdy_sample_args &a = A.a;
    const int row = blockIdx.x, tid = threadIdx.x;
    Work &w = A.work[row];
    Row r;
    r.params(A, row);
    r.maxima(A, row);
    if (r.alone) {
        if (tid == 0) {
            a.token[row] = r.none ? -1 : index_at(r.first);
            if (a.prob) a.prob[row] = r.none ? 0.0f : 1.0f;
        }
        return;
    }
    const float u = a.u[row];
    int mode = w.mode, n = w.n_list;
    uint64_t least = 0;  // the place that the prefix ends at
    auto kept_place = [&](uint64_t at) -> uint64_t {
        if (at < least) return 0;
        const double x = r.weight(value_at(at));
        return at == r.first || !(x < (double)r.min_p) ? (uint64_t)(x * r.one) : 0;
    };
    auto kept = [&](int i) { return kept_place(place_of(r.x[i], i)); };
    auto take = [&](int i, uint64_t v, uint64_t whole) {
        if (tid == 0) {
            a.token[row] = i;
            if (a.prob) a.prob[row] = (float)((double)v / (double)whole);
        }
    };
    if (mode == ROW_TOP || mode == ROW_SUM || mode == ROW_COUNT) {
        for (int i = tid; i < n; i += THREADS) list[i] = w.list[i];
        __syncthreads();
        sort_falling(list, n);
    }
    // thread t holds the sorted tokens t * LIST / THREADS ..
    constexpr int PER = LIST / THREADS;
    auto weights = [&](uint64_t v[PER], int limit) {
        uint64_t s = 0;
#pragma unroll
        for (int e = 0; e < PER; e++) {
            const int i = tid * PER + e;
            v[e] = i < limit ? r.fixed(value_at(list[i])) : 0;
            s += v[e];
        }
        return s;
    };
    // the place that a prefix by sum ends at, `before` of it standing ahead of the list
    auto end_by_sum = [&](int limit, uint64_t before, uint64_t want) {
        uint64_t v[PER], whole;
        uint64_t run = before + block_scan(weights(v, limit), &whole, sh);
        uint64_t last = ~0ull;
#pragma unroll
        for (int e = 0; e < PER; e++) {
            const int i = tid * PER + e;
            if (i < limit && run < want) last = list[i];
            run += v[e];
        }
        const uint64_t m = block_max(last == ~0ull ? 0 : ~last, sh);  // the least of them
        return m ? ~m : 0ull;
    };
    if (mode == ROW_COUNT) {  // many tokens by count: the end of the first top_k is known now, and with it their sum
        const int rest = r.top_k - (int)w.before, end = rest < n ? rest : n;  // of the list
        least = list[end - 1];
        if (r.top_p < 1.0f) {
            unsigned count, none;
            uint64_t sum, whole, before;
            bins_of(A, row, 0, true, &count, &none, &sum);
            const uint64_t above = block_sum(tid < w.bin_k ? sum : 0, sh);
            uint64_t v[PER];
            whole = above + block_sum(weights(v, end), sh);
            const uint64_t want = wanted(r.top_p, whole);
            if (above < want) {
                least = end_by_sum(end, above, want);
            } else {  // the sum ends in an earlier bin, whose tokens nobody has listed
                const int b = bin_that_reaches(tid < w.bin_k ? sum : 0, want, &before, sh);
                const uint64_t c = block_sum(tid == b ? count : 0, sh);
                if (c > LIST) {
                    mode = ROW_SLOW;
                } else {
                    if (tid == 0) n_list = 0;
                    __syncthreads();
                    each(r.x, 0, r.n, [&](float x, int i) {
                        if (x > -INFINITY && r.bin(x) == b) list[atomicAdd(&n_list, 1)] = place_of(x, i);
                    });
                    __syncthreads();
                    sort_falling(list, (int)c);
                    least = end_by_sum((int)c, before, want);
                }
            }
        }
        if (mode == ROW_COUNT) mode = ROW_KNOWN;
    } else if (mode == ROW_TOP) {
        if (n > r.top_k) n = r.top_k;
        if (r.top_p < 1.0f) {
            uint64_t v[PER];
            const uint64_t whole = block_sum(weights(v, n), sh);
            least = end_by_sum(n, 0, wanted(r.top_p, whole));
        }
        // the kept ones, a prefix of the list, by index: the place's halves change sides
        int end = 0;
        for (int i = tid; i < n; i += THREADS) {
            const uint64_t at = list[i];
            const bool in = at >= least && (at == r.first || !(r.weight(value_at(at)) < (double)r.min_p));
            end += in;
            list[i] = in ? (at & (MAX_VOCAB - 1)) << 32 | at >> 22 : 0;
        }
        n = (int)block_sum((uint64_t)end, sh);
        sort_falling(list, n);
        uint64_t v[PER], sum = 0, whole;
#pragma unroll
        for (int e = 0; e < PER; e++) {
            const int i = tid * PER + e;
            v[e] = i < n ? r.fixed(value_at((list[i] & 0xFFFFFFFFu) << 22)) : 0;
            sum += v[e];
        }
        uint64_t run = block_scan(sum, &whole, sh);
        const uint64_t left = share(u, whole);
        if (run <= left && left < run + sum) {
#pragma unroll
            for (int e = 0; e < PER; e++) {
                if (run <= left && left < run + v[e]) {
                    const int i = tid * PER + e;
                    a.token[row] = MAX_VOCAB - 1 - (int)(list[i] >> 32);
                    if (a.prob) a.prob[row] = (float)((double)v[e] / (double)whole);
                }
                run += v[e];
            }
        }
        return;
    } else if (mode == ROW_SUM || mode == ROW_ALL) {
        if (tid < A.pieces) sums[tid] = w.sums[tid];
        __syncthreads();
        if (mode == ROW_SUM) {
            if (r.top_p < 1.0f) least = end_by_sum(n, w.before, w.want);
            if (least == 0 && n) least = list[n - 1];
            for (int i = tid; i < n; i += THREADS) {
                const uint64_t v = kept_place(list[i]);
                if (v) atomicAdd(&sums[index_at(list[i]) / A.len], (unsigned long long)v);
            }
            __syncthreads();
        }
        uint64_t whole = 0;
        for (int p = 0; p < A.pieces; p++) whole += sums[p];
        uint64_t left = share(u, whole);
        int p = 0;
        while (p < A.pieces - 1 && sums[p] <= left) left -= sums[p++];
        const int lo = p * A.len, i = narrow(lo, lo + A.len < r.n ? lo + A.len : r.n, left, kept, sh);
        take(i, kept(i), whole);
        return;
    }
    if (mode == ROW_SLOW) {
        least = 0;
        if (r.top_k) least = prefix_end(r, 0, false, (uint64_t)r.top_k, sh);
        if (r.top_p < 1.0f) {
            uint64_t sum = 0;
            for (int i = tid; i < r.n; i += THREADS)
                if (place_of(r.x[i], i) >= least) sum += r.fixed(r.x[i]);
            sum = block_sum(sum, sh);
            least = prefix_end(r, least, true, wanted(r.top_p, sum), sh);
        }
    }
    uint64_t whole = 0;
    for (int i = tid; i < r.n; i += THREADS) whole += kept(i);
    whole = block_sum(whole, sh);
    const int i = narrow(0, r.n, share(u, whole), kept, sh);
    take(i, kept(i), whole);
}

// Pieces per row: enough workgroups for the GPU where there are few rows, none shorter than 4096 tokens.
int pieces_of(int n_rows, int n_vocab) {
    int p = 256 / n_rows;
    if (p > MAX_PIECES) p = MAX_PIECES;
    if (p > (n_vocab + 4095) / 4096) p = (n_vocab + 4095) / 4096;
    return p < 1 ? 1 : p;
}

}  // namespace

extern "C" size_t sdy_sample_ws_bytes(int n_rows, int n_vocab) {
    if (n_rows < 1 || n_vocab < 1 || n_vocab > MAX_VOCAB) return 0;
    return (size_t)n_rows * (sizeof(Work) + (size_t)pieces_of(n_rows, n_vocab) * BINS * 12);
}

extern "C" int sdy_sample(const sdy_sample_args *a, sdy_stream s) {
    if (!a) return sdy_fail(-1, "sample: no arguments");
    if (a->n_rows < 0 || a->n_rows > 65535) return sdy_fail(-1, "sample: n_rows %d (0..65535)", a->n_rows);
    if (a->n_rows == 0) return 0;
    if (a->n_vocab < 1 || a->n_vocab > MAX_VOCAB) return sdy_fail(-1, "sample: n_vocab %d (1..%d)", a->n_vocab, MAX_VOCAB);
    if (a->n_rows > 1 && a->stride < a->n_vocab)
        return sdy_fail(-1, "sample: rows of %d logits %ld apart", a->n_vocab, a->stride);
    if (!a->logits || !a->u || !a->token || !a->ws) return sdy_fail(-1, "sample: logits, u, token and ws are needed");
    if ((uintptr_t)a->ws & 15) return sdy_fail(-1, "sample: ws aligned to 16 bytes");
    Args A;
    A.a = *a;
    int log2 = 0;
    while ((1 << log2) < a->n_vocab) log2++;
    A.shift = 62 - log2;
    A.pieces = pieces_of(a->n_rows, a->n_vocab);
    A.len = (a->n_vocab + A.pieces - 1) / A.pieces;
    A.work = (Work *)a->ws;
    A.sum = (unsigned long long *)(A.work + a->n_rows);
    A.count = (unsigned *)(A.sum + (size_t)a->n_rows * A.pieces * BINS);
    const dim3 grid(A.pieces, a->n_rows), block(THREADS);
    hipStream_t st = (hipStream_t)s;
    hipLaunchKernelGGL(k_sample_max, grid, block, 0, st, A);
    hipLaunchKernelGGL(k_sample_bins, grid, block, 0, st, A);
    hipLaunchKernelGGL(k_sample_list, grid, block, 0, st, A);
    hipLaunchKernelGGL(k_sample_pick, dim3(a->n_rows), block, 0, st, A);
    return sdy_check_launch("sample");
}
