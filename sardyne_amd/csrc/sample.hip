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
//   k_sample_cut   one workgroup per row: the bin in which the prefix ends, and what is before it;
//   k_sample_list  that bin's tokens (with a small top_k all up to there);
//   k_sample_pick  one workgroup per row: these tokens sorted, the prefix's end among them, the pieces' sums, and the token
//                  in its piece. A row whose end lies among more than 4096 tokens (nearly equal logits) is searched digit by
//                  digit instead.
#include "sdy_device.h"
#include "sdy_internal.h"
#include "sdy_ops.h"

namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int MAX_VOCAB = 1 << 22;  // a token's place in the order fits 32 + 22 bits
constexpr int BINS = 1024, PER = BINS / THREADS;  // a thread's bins
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
    unsigned offset[MAX_PIECES];           // where a piece's listed tokens start
    int mode, n_list, b0, b1;              // the listed bins b0 .. b1
    unsigned long long before;             // count or sum before them
    unsigned long long want;               // the sum that the prefix has to reach
    unsigned long long list[LIST];
};
// after them: per row and piece, BINS sums; then BINS counts

enum { ROW_ALONE = 0,  // the first token, or none
       ROW_ALL,        // nothing is left out
       ROW_TOP,        // the listed tokens hold the whole prefix
       ROW_SUM,        // the prefix ends by its sum (or min-p) in the listed bins
       ROW_COUNT,      // the first top_k tokens end in the listed bin
       ROW_SLOW };     // it ends among too many tokens to list

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
    // from the pieces' maxima, by each wave for itself
    SDY_DEV void maxima(const Args &A, int row) {
        const Work &w = A.work[row];
        const int c = (int)(threadIdx.x & 63) < A.pieces ? threadIdx.x & 63 : 0;
        uint64_t m = w.first[c];
        float low = w.low[c];
#pragma unroll
        for (int off = MAX_PIECES / 2; off >= 1; off /= 2) {
            const uint64_t o = __shfl_xor((unsigned long long)m, off);
            m = o > m ? o : m;
            low = fminf(low, __shfl_xor(low, off));
        }
        first = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(m >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)m);
        low = __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(low)));
        best = value_at(first);
        none = !(best > -INFINITY);
        alone = none || !(temp > 0.0f);
        inv_t = 1.0 / (double)temp;
        // over the whole of the finite logits, or as far down as a w counts (2^-62 is exp(-43))
        const float range = fminf(best - low, 43.0f * temp);
        per_bin = range > 0.0f ? (float)BINS / range : 0.0f;
    }
    SDY_DEV bool sums() const { return !top_k || top_k > SMALL_K; }  // whether the bins' sums are made
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

// f(logit, index) of the tokens [lo, hi) (lo a multiple of 4), four 16-byte loads in flight where the row allows them
template <class F>
SDY_DEV void each(const float *x, int lo, int hi, const F &f) {
    int i = lo;
    if (((uintptr_t)x & 15) == 0) {
        const int end = lo + (hi - lo) / 4 * 4;
        for (int i0 = lo + 4 * (int)threadIdx.x; i0 < end; i0 += 16 * THREADS) {
            float4 v[4];
#pragma unroll
            for (int u = 0; u < 4; u++) v[u] = *reinterpret_cast<const float4 *>(x + (i0 + 4 * u * THREADS < end ? i0 + 4 * u * THREADS : lo));
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int j = i0 + 4 * u * THREADS;
                if (j >= end) continue;
                f(v[u].x, j);
                f(v[u].y, j + 1);
                f(v[u].z, j + 2);
                f(v[u].w, j + 3);
            }
        }
        i = end;
    }
    for (int i0 = i + (int)threadIdx.x; i0 < hi; i0 += 8 * THREADS) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; u++) v[u] = x[i0 + u * THREADS < hi ? i0 + u * THREADS : hi - 1];
#pragma unroll
        for (int u = 0; u < 8; u++)
            if (i0 + u * THREADS < hi) f(v[u], i0 + u * THREADS);
    }
}

struct Parts {
    float low[WAVES];
    unsigned long long part[WAVES];
    unsigned long long found, before;
};
struct Shared : Parts {
    union {
        struct {
            unsigned long long sum[2048];
            unsigned count[2048];
        };
        unsigned long long w[LIST];  // the sorted tokens' w
    };
};

SDY_DEV uint64_t wave_sum(uint64_t v) {
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor((unsigned long long)v, off);
    return v;
}

SDY_DEV uint64_t block_sum(uint64_t v, Parts &sh) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.part[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t r = 0;
    for (int w = 0; w < WAVES; w++) r += sh.part[w];
    return r;
}

SDY_DEV uint64_t block_max(uint64_t v, Parts &sh) {
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
SDY_DEV uint64_t block_scan(uint64_t v, uint64_t *whole, Parts &sh) {
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
    __shared__ Parts sh;
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
    __shared__ Parts sh;
    __shared__ unsigned count[BINS];
    __shared__ unsigned long long sums_of[BINS];
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
    const bool sums = r.sums();
    for (int b = tid; b < BINS; b += THREADS) count[b] = 0, sums_of[b] = 0;
    __syncthreads();
    each(r.x, lo, hi, [&](float v, int) {
        if (!(v > -INFINITY)) return;
        const int b = r.bin(v);
        atomicAdd(&count[b], 1u);
        if (sums) atomicAdd(&sums_of[b], (unsigned long long)r.fixed(v));
    });
    __syncthreads();
    const size_t at = ((size_t)row * A.pieces + c) * BINS;
    for (int b = tid; b < BINS; b += THREADS) {
        A.count[at + b] = count[b];
        if (sums) A.sum[at + b] = sums_of[b];
    }
}

// The least sum that reaches top_p of the whole
SDY_DEV uint64_t wanted(float top_p, uint64_t whole) {
    const double want = ceil((double)top_p * (double)whole);
    return want > 1.0 ? (uint64_t)want : 1;
}

// The row's bins PER * tid .. of this thread: counts and sums over the pieces.
SDY_DEV void bins_of(const Args &A, int row, bool sums, uint64_t count[PER], uint64_t sum[PER]) {
    static_assert(PER == 4, "a thread's bins are one 16-byte load of counts");
    const size_t at = (size_t)row * A.pieces * BINS + PER * threadIdx.x;
    for (int e = 0; e < PER; e++) count[e] = sum[e] = 0;
#pragma unroll 4
    for (int p = 0; p < A.pieces; p++) {
        const uint4 n = *reinterpret_cast<const uint4 *>(A.count + at + (size_t)p * BINS);
        count[0] += n.x, count[1] += n.y, count[2] += n.z, count[3] += n.w;
        if (sums) {
            const ulonglong2 a = *reinterpret_cast<const ulonglong2 *>(A.sum + at + (size_t)p * BINS);
            const ulonglong2 b = *reinterpret_cast<const ulonglong2 *>(A.sum + at + (size_t)p * BINS + 2);
            sum[0] += a.x, sum[1] += a.y, sum[2] += b.x, sum[3] += b.y;
        }
    }
}

// The threads' bins: v's running sums, the whole, the bin at which `want` is reached (the last one with any if it never is)
// and what is before it.
struct Reach {
    uint64_t whole, before;
    int bin;
};
SDY_DEV Reach bin_that_reaches(const uint64_t v[PER], uint64_t want, float top_p, Parts &sh) {
    Reach r;
    const uint64_t mine = v[0] + v[1] + v[2] + v[3];
    uint64_t run = block_scan(mine, &r.whole, sh);
    if (top_p < 1.0f) want = wanted(top_p, r.whole);
    if (want > r.whole) want = r.whole;
    if (threadIdx.x == 0 && r.whole == 0) sh.found = 0, sh.before = 0;
    if (run < want && run + mine >= want) {
        int e = 0;
        while (e < PER - 1 && run + v[e] < want) run += v[e++];
        sh.found = PER * threadIdx.x + e;
        sh.before = run;
    }
    __syncthreads();
    r.bin = (int)sh.found;
    r.before = sh.before;
    return r;
}

__global__ __launch_bounds__(THREADS) void k_sample_cut(Args A) {
    __shared__ Parts sh;
    __shared__ unsigned listed_of[MAX_PIECES];
    const int row = blockIdx.x, tid = threadIdx.x;
    Work &w = A.work[row];
    Row r;
    r.params(A, row);
    r.maxima(A, row);
    if (r.alone || !r.cut()) {
        if (tid == 0) w.mode = r.alone ? ROW_ALONE : ROW_ALL;
        return;
    }
    const bool sums = r.sums();
    uint64_t count[PER], sum[PER];
    bins_of(A, row, sums, count, sum);
    int b0 = 0, b1 = BINS - 1, mode = ROW_SUM;
    uint64_t want = ~0ull;
    if (r.top_k) {
        const Reach k = bin_that_reaches(count, (uint64_t)r.top_k, 1.0f, sh);
        b1 = k.bin;
        mode = ROW_TOP;
        uint64_t all = 0;
        for (int e = 0; e < PER; e++) all += PER * tid + e <= b1 ? count[e] : 0;
        if (block_sum(all, sh) > LIST) {
            b0 = b1;
            mode = sums ? ROW_COUNT : ROW_SLOW;
        }
    } else {
        if (r.top_p < 1.0f) {
            const Reach p = bin_that_reaches(sum, 0, r.top_p, sh);
            want = wanted(r.top_p, p.whole);
            b0 = b1 = p.bin;
        }
        if (r.min_p > 0.0f) {
            // the bins that the border can be in: their arithmetic is in 32 bits
            const float far = r.min_p < 1.0f ? -logf(r.min_p) * r.temp * r.per_bin : 0.0f;
            const int lo = (int)fminf(far * (1.0f - 1e-5f), (float)(BINS - 1));
            const int hi = (int)fminf(far * (1.0f + 1e-5f) + 1e-5f, (float)(BINS - 1));
            b0 = r.top_p < 1.0f && b0 < lo ? b0 : lo;
            b1 = hi < b1 ? hi : b1;
        }
    }
    uint64_t listed = 0, before = 0;
    for (int e = 0; e < PER; e++) {
        const int b = PER * tid + e;
        listed += b >= b0 && b <= b1 ? count[e] : 0;
        before += b < b0 ? (mode == ROW_COUNT ? count[e] : sum[e]) : 0;
    }
    listed = block_sum(listed, sh);
    before = block_sum(before, sh);
    if (listed > LIST) mode = ROW_SLOW;
    if (tid == 0) {
        w.mode = mode;
        w.n_list = (int)listed;
        w.b0 = b0;
        w.b1 = b1;
        w.before = before;
        w.want = want;
    }
    // per piece, a wave each in turn: its listed tokens, then their offsets, and its sum before the listed bins
    const int lane = tid & 63;
    for (int p = tid >> 6; p < A.pieces; p += WAVES) {
        const size_t at = ((size_t)row * A.pieces + p) * BINS;
        uint64_t n = 0, s = 0;
        for (int b = b0 + lane; b <= b1; b += 64) n += A.count[at + b];
        if (sums)
            for (int b = lane; b < b0; b += 64) s += A.sum[at + b];
        n = wave_sum(n);
        s = wave_sum(s);
        if (lane == 0) {
            listed_of[p] = (unsigned)n;
            w.sums[p] = s;
        }
    }
    __syncthreads();
    if (tid < A.pieces) {
        unsigned n = 0;
        for (int p = 0; p < tid; p++) n += listed_of[p];
        w.offset[tid] = n;
    }
}

__global__ __launch_bounds__(THREADS) void k_sample_list(Args A) {
    __shared__ unsigned next;
    const int c = blockIdx.x, row = blockIdx.y;
    Work &w = A.work[row];
    const int mode = w.mode;
    if (mode != ROW_TOP && mode != ROW_SUM && mode != ROW_COUNT) return;
    Row r;
    r.params(A, row);
    r.maxima(A, row);
    const int b0 = w.b0, b1 = w.b1;
    if (threadIdx.x == 0) next = w.offset[c];
    __syncthreads();
    const int lo = c * A.len, hi = lo + A.len < r.n ? lo + A.len : r.n;
    each(r.x, lo, hi, [&](float v, int i) {
        if (!(v > -INFINITY)) return;
        const int b = r.bin(v);
        if (b >= b0 && b <= b1) w.list[atomicAdd(&next, 1u)] = place_of(v, i);
    });
}

// list[0 .. n) in falling order, all different. Up to 256: each one's rank counted, one round. Above: a bitonic sort of the
// next power of two, padded with zeros.
SDY_DEV void sort_falling(unsigned long long *list, int n) {
    __syncthreads();
    if (n <= THREADS) {
        const unsigned long long mine = (int)threadIdx.x < n ? list[threadIdx.x] : 0;
        int rank = 0;
#pragma unroll 8
        for (int i = 0; i < n; i++) rank += list[i] > mine;
        __syncthreads();
        if ((int)threadIdx.x < n) list[rank] = mine;
        __syncthreads();
        return;
    }
    int n2 = 2 * THREADS;
    while (n2 < n) n2 *= 2;
    for (int i = n + threadIdx.x; i < n2; i += THREADS) list[i] = 0;
    __syncthreads();
    for (int k = 2; k <= n2; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            for (int t = threadIdx.x; t < n2 / 2; t += THREADS) {
                const int i = ((t & ~(j - 1)) << 1) | (t & (j - 1));
                const unsigned long long x = list[i], y = list[i + j];
                if ((x < y) == ((i & k) == 0)) list[i] = y, list[i + j] = x;
            }
            __syncthreads();
        }
}

// The piece [lo, hi) narrowed to the token at which the running sum of kept(i) passes `left`
template <class F>
SDY_DEV int narrow(int lo, int hi, uint64_t left, const F &kept, Parts &sh) {
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

struct Pick {
    Shared sh;
    unsigned long long list[LIST];
    unsigned long long sums[MAX_PIECES];
    int n_list;
};

__global__ __launch_bounds__(THREADS) void k_sample_pick(Args A) {
    extern __shared__ __align__(16) unsigned char lds_bytes[];
    Pick &k = *reinterpret_cast<Pick *>(lds_bytes);
    Shared &sh = k.sh;
    unsigned long long *const list = k.list;
    const sdy_sample_args &a = A.a;
    const int row = blockIdx.x, tid = threadIdx.x;
    const Work &w = A.work[row];
    int mode = w.mode, n = w.n_list;
    if (mode == ROW_TOP || mode == ROW_SUM || mode == ROW_COUNT)
        for (int i = tid; i < n; i += THREADS) list[i] = w.list[i];
    Row r;
    r.params(A, row);
    r.maxima(A, row);
    if (mode == ROW_ALONE) {
        if (tid == 0) {
            a.token[row] = r.none ? -1 : index_at(r.first);
            if (a.prob) a.prob[row] = r.none ? 0.0f : 1.0f;
        }
        return;
    }
    const float u = a.u[row];
    uint64_t least = 0;  // the place that the prefix ends at
    auto kept_place = [&](uint64_t at) -> uint64_t {
        if (at < least) return 0;
        const double x = r.weight(value_at(at));
        return at == r.first || !(x < (double)r.min_p) ? (uint64_t)(x * r.one) : 0;
    };
    auto kept = [&](int i) { return kept_place(place_of(r.x[i], i)); };
    auto take = [&](int i, uint64_t v, uint64_t whole) {
        a.token[row] = i;
        if (a.prob) a.prob[row] = (float)((double)v / (double)whole);
    };
    if (mode == ROW_TOP || mode == ROW_SUM || mode == ROW_COUNT) sort_falling(list, n);
    // thread t holds the sorted tokens t * per .. t * per + per - 1 of the first `limit`; sh.w[i] is the i-th one's w
    auto weights = [&](int limit, int per) {
        uint64_t s = 0;
        for (int i = tid * per; i < limit && i < tid * per + per; i++) s += sh.w[i] = r.fixed(value_at(list[i]));
        return s;
    };
    // the place that a prefix by sum ends at, `before` of it standing ahead of the list. want 0: top_p of the list
    auto end_by_sum = [&](int limit, uint64_t before, uint64_t want) {
        const int per = (limit + THREADS - 1) / THREADS;
        __syncthreads();  // (sh.w shares its memory)
        uint64_t whole;
        uint64_t run = before + block_scan(weights(limit, per), &whole, sh);
        if (want == 0) want = wanted(r.top_p, whole);
        uint64_t last = ~0ull;
        for (int i = tid * per; i < limit && i < tid * per + per && run < want; i++) {
            last = list[i];
            run += sh.w[i];
        }
        const uint64_t m = block_max(~last, sh);  // the least of them
        return m ? ~m : 0ull;
    };
    if (mode == ROW_TOP) {
        if (n > r.top_k) n = r.top_k;
        if (r.top_p < 1.0f) least = end_by_sum(n, 0, 0);
        // the kept ones, a prefix of the list, by index: the place's halves change sides
        uint64_t end = 0;
        for (int i = tid; i < n; i += THREADS) {
            const uint64_t at = list[i];
            const bool in = at >= least && (at == r.first || !(r.weight(value_at(at)) < (double)r.min_p));
            end += in;
            list[i] = in ? (at & (MAX_VOCAB - 1)) << 32 | at >> 22 : 0;
        }
        n = (int)block_sum(end, sh);
        sort_falling(list, n);
        const int per = (n + THREADS - 1) / THREADS;
        uint64_t sum = 0, whole;
        for (int i = tid * per; i < n && i < tid * per + per; i++) sum += sh.w[i] = r.fixed(value_at((list[i] & 0xFFFFFFFFu) << 22));
        uint64_t run = block_scan(sum, &whole, sh);
        const uint64_t left = share(u, whole);
        if (run <= left && left < run + sum) {
            int i = tid * per;
            while (run + sh.w[i] <= left) run += sh.w[i++];
            take(MAX_VOCAB - 1 - (int)(list[i] >> 32), sh.w[i], whole);
        }
        return;
    }
    if (mode == ROW_SUM || mode == ROW_ALL) {
        if (tid < A.pieces) k.sums[tid] = w.sums[tid];
        __syncthreads();
        if (mode == ROW_SUM) {
            if (r.top_p < 1.0f) least = end_by_sum(n, w.before, w.want);
            if (least == 0 && n) least = list[n - 1];
            for (int i = tid; i < n; i += THREADS) {
                const uint64_t v = kept_place(list[i]);
                if (v) atomicAdd(&k.sums[index_at(list[i]) / A.len], (unsigned long long)v);
            }
            __syncthreads();
        }
        uint64_t whole = 0;
        for (int p = 0; p < A.pieces; p++) whole += k.sums[p];
        uint64_t left = share(u, whole);
        int p = 0;
        while (p < A.pieces - 1 && k.sums[p] <= left) left -= k.sums[p++];
        const int lo = p * A.len, i = narrow(lo, lo + A.len < r.n ? lo + A.len : r.n, left, kept, sh);
        if (tid == 0) take(i, kept(i), whole);
        return;
    }
    if (mode == ROW_COUNT) {  // many tokens by count: the end of the first top_k is known now, and with it their sum
        const int rest = r.top_k - (int)w.before, end = rest < n ? rest : n;  // of the list
        least = list[end - 1];
        if (r.top_p < 1.0f) {
            uint64_t count[PER], sum[PER], ahead = 0, in_list = 0;
            bins_of(A, row, true, count, sum);
            for (int e = 0; e < PER; e++) {
                if (PER * tid + e >= w.b0) sum[e] = 0;
                ahead += sum[e];
            }
            ahead = block_sum(ahead, sh);
            in_list = block_sum(weights(end, (end + THREADS - 1) / THREADS), sh);
            const uint64_t want = wanted(r.top_p, ahead + in_list);
            if (ahead < want) {
                least = end_by_sum(end, ahead, want);
            } else {  // the sum ends in an earlier bin, whose tokens nobody has listed
                const Reach b = bin_that_reaches(sum, want, 1.0f, sh);
                uint64_t c = 0;
                for (int e = 0; e < PER; e++) c += PER * tid + e == b.bin ? count[e] : 0;
                c = block_sum(c, sh);
                if (c > LIST) {
                    mode = ROW_SLOW;
                } else {
                    if (tid == 0) k.n_list = 0;
                    __syncthreads();
                    each(r.x, 0, r.n, [&](float x, int i) {
                        if (x > -INFINITY && r.bin(x) == b.bin) list[atomicAdd(&k.n_list, 1)] = place_of(x, i);
                    });
                    sort_falling(list, (int)c);
                    least = end_by_sum((int)c, b.before, want);
                }
            }
        }
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
    if (tid == 0) take(i, kept(i), whole);
}

// Pieces per row: enough workgroups for the GPU where there are few rows, none shorter than 4096 tokens.
int pieces_of(int n_rows, int n_vocab) {
    int p = (n_vocab + 4095) / 4096;
    (void)n_rows;
    return p < MAX_PIECES ? p : MAX_PIECES;
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
    A.len = ((a->n_vocab + A.pieces - 1) / A.pieces + 3) & ~3;
    A.work = (Work *)a->ws;
    A.sum = (unsigned long long *)(A.work + a->n_rows);
    A.count = (unsigned *)(A.sum + (size_t)a->n_rows * A.pieces * BINS);
    static size_t granted = 0;
    const int rc = sdy_lds_limit((const void *)k_sample_pick, sizeof(Pick), &granted);
    if (rc) return rc;
    const dim3 grid(A.pieces, a->n_rows), block(THREADS);
    hipStream_t st = (hipStream_t)s;
    hipLaunchKernelGGL(k_sample_max, grid, block, 0, st, A);
    hipLaunchKernelGGL(k_sample_bins, grid, block, 0, st, A);
    hipLaunchKernelGGL(k_sample_cut, dim3(a->n_rows), block, 0, st, A);
    hipLaunchKernelGGL(k_sample_list, grid, block, 0, st, A);
    hipLaunchKernelGGL(k_sample_pick, dim3(a->n_rows), block, sizeof(Pick), st, A);
    return sdy_check_launch("sample");
}
