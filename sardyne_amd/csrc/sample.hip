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
// Every kept set is a prefix of the order, so what is looked for is where it ends, without sorting the row. Rows of up to
// 2560 tokens are a workgroup's work in LDS (k_sample_small). A longer row is cut into pieces, a workgroup each, and read
// three times, the second and third from the caches:
//   k_sample_max   each piece's greatest and lowest logit;
//   k_sample_bins  each piece's tokens counted, and their w added, by distance from the greatest logit in 1024 bins;
//   k_sample_cut   one workgroup per row: the bin in which the prefix ends, and what is before it;
//   k_sample_list  that bin's tokens (with a small top_k all up to there);
//   k_sample_pick  one workgroup per row: the prefix's end among these tokens, the pieces' sums, and the token in its piece.
//                  A row whose end lies among more than 4096 tokens (nearly equal logits) is searched digit by digit instead.
#include "sdy_device.h"
#include "sdy_internal.h"
#include "sdy_ops.h"

namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int MAX_VOCAB = 1 << 22;  // a token's place in the order fits 32 + 22 bits
constexpr int BINS = 1024;
constexpr int LIST = 4096;          // tokens that one workgroup holds
// Rows that one workgroup does alone, in one launch (top-k 40 and top-p; alone against in pieces): 2048 tokens 20.7 against
// 22.8 us, 64 such rows 21.6 against 26.1, 1000 rows 47 against 56; 3000 tokens 26.1 against 23.1, 27.1 against 26.5, 60
// against 58.
constexpr int SMALL = 2560;
// Up to so large a top_k the bins' sums are not made: the first top_k tokens are listed themselves (without against with
// sums, 61 rows of 151936: top-k 40 47 against 63 us, 1000 57 against 71).
constexpr int SMALL_K = 1024;
// Pieces of a row (4, 8, 16: one row of 151936 38.8, 33.3, 31.0 us, 61 rows 65, 51, 47, 250 rows 98, 103, 103).
constexpr int MAX_PIECES = 16;
// Up to so many rows 1024 threads to a piece instead of 256 (1 row 27.7 against 31.3 us, 16 32.2 against 35.8, 32 36.7
// against 38.8; 40 43.0 against 41.0, 64 51.9 against 48.3).
constexpr int FEW_ROWS = 32;

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
    unsigned long long sum_of[BINS];       // ROW_COUNT: the bins' sums and counts over the row
    unsigned count_of[BINS];
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
    unsigned long long *sum;   // [n_rows][pieces][BINS]
    unsigned *count;           // [n_rows][pieces][BINS]
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
    SDY_DEV void start(uint64_t place, float low) {
        first = place;
        best = value_at(first);
        none = !(best > -INFINITY);
        alone = none || !(temp > 0.0f);
        inv_t = 1.0 / (double)temp;
        // over the whole of the finite logits, or as far down as a w counts (2^-62 is exp(-43))
        // (at most f32's greatest value: two logits can be farther apart, and are in the last bin then)
        const float range = fminf(fminf(best - low, 43.0f * temp), 0x1.fffffep127f);
        per_bin = range > 0.0f ? (float)BINS / range : 0.0f;
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
        start((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(m >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)m),
              __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(low))));
    }
    SDY_DEV bool sums() const { return !top_k || top_k > SMALL_K; }  // whether the bins' sums are made
    SDY_DEV bool cut() const { return top_k || top_p < 1.0f || min_p > 0.0f; }
    SDY_DEV double weight(float v) const {
        if (v == best) return 1.0;
        if (!(v > -INFINITY) || best == INFINITY) return 0.0;
        return exp(((double)v - (double)best) * inv_t);
    }
    SDY_DEV uint64_t fixed(float v) const { return (uint64_t)(weight(v) * one); }  // w as a whole number of 2^-S
    // the same where min-p leaves the token, else 0
    SDY_DEV uint64_t fixed_kept(uint64_t place) const {
        const double w = weight(value_at(place));
        return place == first || !(w < (double)min_p) ? (uint64_t)(w * one) : 0;
    }
    // never less for a lower logit
    SDY_DEV int bin(float v) const { return v == best ? 0 : (int)fminf((best - v) * per_bin, (float)(BINS - 1)); }
};

// f(logit, index) of the tokens [lo, hi) (lo a multiple of 4), four 16-byte loads in flight where the row allows them
template <int T = THREADS, class F>
SDY_DEV void each(const float *x, int lo, int hi, const F &f) {
    int i = lo;
    if (((uintptr_t)x & 15) == 0) {
        const int end = lo + (hi - lo) / 4 * 4;
        for (int i0 = lo + 4 * (int)threadIdx.x; i0 < end; i0 += 16 * T) {
            float4 v[4];
#pragma unroll
            for (int u = 0; u < 4; u++) v[u] = *reinterpret_cast<const float4 *>(x + (i0 + 4 * u * T < end ? i0 + 4 * u * T : lo));
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int j = i0 + 4 * u * T;
                if (j >= end) continue;
                f(v[u].x, j);
                f(v[u].y, j + 1);
                f(v[u].z, j + 2);
                f(v[u].w, j + 3);
            }
        }
        i = end;
    }
    for (int i0 = i + (int)threadIdx.x; i0 < hi; i0 += 8 * T) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; u++) v[u] = x[i0 + u * T < hi ? i0 + u * T : hi - 1];
#pragma unroll
        for (int u = 0; u < 8; u++)
            if (i0 + u * T < hi) f(v[u], i0 + u * T);
    }
}

// ---- sums over a block of W waves

template <int W>
struct Parts {
    float low[W];
    unsigned long long part[W];
    unsigned long long key, val, run;  // what one thread found
};

// v of the lane that DPP control CTRL names, 0 where there is none (or the row is masked off)
template <int CTRL, int ROWS>
SDY_DEV uint64_t dpp_u64(uint64_t v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, false);
    return (uint64_t)hi << 32 | lo;
}

// Over the wave's lanes up to this one: within rows of 16 lanes by shifts of 1, 2, 4, 8, then the rows' ends passed on.
template <bool MAX>
SDY_DEV uint64_t wave_run(uint64_t v) {
    auto add = [&](uint64_t o) { v = MAX ? (o > v ? o : v) : v + o; };
    add(dpp_u64<0x111, 0xF>(v));
    add(dpp_u64<0x112, 0xF>(v));
    add(dpp_u64<0x114, 0xF>(v));
    add(dpp_u64<0x118, 0xF>(v));
    add(dpp_u64<0x142, 0xA>(v));  // row_bcast 15 to rows 1 and 3
    add(dpp_u64<0x143, 0xC>(v));  // row_bcast 31 to rows 2 and 3
    return v;
}
SDY_DEV uint64_t last_lane(uint64_t v) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), 63) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, 63);
}
SDY_DEV uint64_t wave_sum(uint64_t v) { return last_lane(wave_run<false>(v)); }

template <int W>
SDY_DEV uint64_t block_sum(uint64_t v, Parts<W> &sh) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.part[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t r = 0;
#pragma unroll
    for (int w = 0; w < W; w++) r += sh.part[w];
    return r;
}

template <int W>
SDY_DEV uint64_t block_max(uint64_t v, Parts<W> &sh) {
    v = last_lane(wave_run<true>(v));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.part[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t r = 0;
#pragma unroll
    for (int w = 0; w < W; w++) r = sh.part[w] > r ? sh.part[w] : r;
    return r;
}

// The sum over the threads before this one; *whole the sum over all.
template <int W>
SDY_DEV uint64_t block_scan(uint64_t v, uint64_t *whole, Parts<W> &sh) {
    const uint64_t run = wave_run<false>(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.part[threadIdx.x >> 6] = run;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < W; w++) {
        if (w < (int)(threadIdx.x >> 6)) before += sh.part[w];
        all += sh.part[w];
    }
    *whole = all;
    return before + run - v;
}

// The thread whose v takes the running sum from `before` to `want`: its number in sh.key, what runs before it in sh.run (the
// last thread where all of it is less).
template <int W>
SDY_DEV void reach(uint64_t v, uint64_t before, uint64_t want, Parts<W> &sh) {
    uint64_t whole;
    const uint64_t run = before + block_scan(v, &whole, sh);
    if ((run < want && run + v >= want) || (threadIdx.x == 64 * W - 1 && run + v < want)) sh.key = threadIdx.x, sh.run = run;
    __syncthreads();
}

// The least sum that reaches top_p of the whole
SDY_DEV uint64_t wanted(float top_p, uint64_t whole) {
    const double want = ceil((double)top_p * (double)whole);
    return want > 1.0 ? (uint64_t)want : 1;
}

// u of the whole, in 0 .. whole - 1
SDY_DEV uint64_t share(float u, uint64_t whole) {
    if (!(u > 0.0f)) return 0;
    if (u >= 1.0f) return whole - 1;
    const uint64_t t = (uint64_t)((double)u * (double)whole);
    return t < whole ? t : whole - 1;
}

// ---- among the tokens of one workgroup

constexpr int SUB = THREADS;
struct Lds {
    Parts<WAVES> parts;
    unsigned long long list[LIST];  // places
    union {
        unsigned long long w[LIST];  // their w
        struct {                     // prefix_end's, which has no list
            unsigned long long digit_sum[2048];
            unsigned digit_count[2048];
        };
    };
    unsigned long long sub_sum[SUB], near[64], near_w[64], sums[MAX_PIECES];
    unsigned sub_count[SUB];
    int n;
};

// Of n things with different key(i), in falling order, the one at which the running sum of val(i) from `before` on reaches
// `want`: its key, its val and what runs before it. It exists: before < want <= before and the whole. The keys' range is cut
// into 256 and the piece that holds it again, until 64 things are left; these count each other.
struct Found {
    uint64_t key, val, run;
};
template <class K, class V>
SDY_DEV Found find(int n, const K &key, const V &val, uint64_t before, uint64_t want, Lds &k) {
    const int tid = threadIdx.x;
    uint64_t hi = ~0ull, lo = 0;
    if (n > 64) {
        uint64_t most = 0, least = 0;
        for (int i = tid; i < n; i += THREADS)
            if (val(i)) {
                const uint64_t x = key(i);
                most = x > most ? x : most;
                least = ~x > least ? ~x : least;
            }
        hi = block_max(most, k.parts);
        lo = ~block_max(least, k.parts);
        for (;;) {
            const int bits = 64 - __builtin_clzll((hi - lo) | 1), shift = bits > 8 ? bits - 8 : 0;
            k.sub_sum[tid] = 0;
            k.sub_count[tid] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += THREADS) {
                const uint64_t x = key(i), v = val(i);
                if (v && x >= lo && x <= hi) {
                    atomicAdd(&k.sub_sum[(hi - x) >> shift], (unsigned long long)v);
                    atomicAdd(&k.sub_count[(hi - x) >> shift], 1u);
                }
            }
            __syncthreads();
            reach(k.sub_sum[tid], before, want, k.parts);
            const int d = (int)k.parts.key, c = (int)k.sub_count[d];
            before = k.parts.run;
            hi -= (uint64_t)d << shift;
            const uint64_t l = hi - ((1ull << shift) - 1);
            if (l > lo && l <= hi) lo = l;
            __syncthreads();
            if (c <= 64 || shift == 0) break;
        }
    }
    if (tid == 0) k.n = 0;
    __syncthreads();
    for (int i = tid; i < n; i += THREADS) {
        const uint64_t x = key(i), v = val(i);
        if (v && x >= lo && x <= hi) {
            const int at = atomicAdd(&k.n, 1);
            k.near[at] = x;
            k.near_w[at] = v;
        }
    }
    __syncthreads();
    if (tid < k.n) {
        const uint64_t x = k.near[tid], v = k.near_w[tid];
        uint64_t run = before;
        for (int i = 0; i < k.n; i++) run += k.near[i] > x ? k.near_w[i] : 0;
        if (run < want && run + v >= want) k.parts.key = x, k.parts.val = v, k.parts.run = run;
    }
    __syncthreads();
    const Found f = {k.parts.key, k.parts.val, k.parts.run};
    __syncthreads();
    return f;
}

SDY_DEV void take(const Args &A, int row, int token, uint64_t w, uint64_t whole) {
    A.a.token[row] = token;
    if (A.a.prob) A.a.prob[row] = (float)((double)w / (double)whole);
}

// The token of a row that is alone, or none
SDY_DEV void take_alone(const Args &A, int row, const Row &r) {
    A.a.token[row] = r.none ? -1 : index_at(r.first);
    if (A.a.prob) A.a.prob[row] = r.none ? 0.0f : 1.0f;
}

// The token of a row whose kept ones are all among the n in the list.
SDY_DEV void pick_listed(const Args &A, int row, const Row &r, int n, Lds &k) {
    const int tid = threadIdx.x;
    const float u = A.a.u[row];
    for (int i = tid; i < n; i += THREADS) k.w[i] = r.fixed(value_at(k.list[i]));
    __syncthreads();
    uint64_t least = 0, sum = 0;
    auto place = [&](int i) -> uint64_t { return k.list[i]; };
    if (r.top_k && n > r.top_k)
        least = find(n, place, [](int) -> uint64_t { return 1; }, 0, (uint64_t)r.top_k, k).key;
    if (r.top_p < 1.0f) {
        for (int i = tid; i < n; i += THREADS) sum += k.list[i] >= least ? k.w[i] : 0;
        sum = block_sum(sum, k.parts);
        least = find(n, place, [&](int i) -> uint64_t { return k.list[i] >= least ? k.w[i] : 0; }, 0, wanted(r.top_p, sum), k).key;
        sum = 0;
    }
    for (int i = tid; i < n; i += THREADS) {
        if (k.list[i] < least) k.w[i] = 0;
        else if (r.min_p > 0.0f) k.w[i] = r.fixed_kept(k.list[i]);
        sum += k.w[i];
    }
    sum = block_sum(sum, k.parts);
    // by index now
    const Found f = find(n, [&](int i) -> uint64_t { return k.list[i] & (MAX_VOCAB - 1); }, [&](int i) -> uint64_t { return k.w[i]; }, 0,
                         share(u, sum) + 1, k);
    if (tid == 0) take(A, row, MAX_VOCAB - 1 - (int)f.key, f.val, sum);
}

// Of the tokens [lo, hi) of x the one at which the running sum of kept(logit, index) passes `left` (lo a multiple of 4)
template <class F>
SDY_DEV int narrow(const float *x, int lo, int hi, uint64_t left, const F &kept, Lds &k) {
    while (hi - lo > 1) {
        int per = (hi - lo + THREADS - 1) / THREADS;
        const bool wide = per >= 4 && ((uintptr_t)x & 15) == 0;
        if (wide) per = (per + 3) & ~3;
        const int b = lo + (int)threadIdx.x * per, e = b + per < hi ? b + per : hi;
        uint64_t sum = 0;
        int i = b;
        if (wide) {
#pragma unroll 4
            for (; i + 4 <= e; i += 4) {
                const float4 v = *reinterpret_cast<const float4 *>(x + i);
                sum += kept(v.x, i) + kept(v.y, i + 1) + (kept(v.z, i + 2) + kept(v.w, i + 3));
            }
        }
#pragma unroll 4
        for (; i < e; i++) sum += kept(x[i], i);
        reach(sum, 0, left + 1, k.parts);
        lo = lo + (int)k.parts.key * per < hi ? lo + (int)k.parts.key * per : hi - 1;
        hi = lo + per < hi ? lo + per : hi;
        left -= k.parts.run;
        __syncthreads();
    }
    return lo;
}

// The place of the last token of the shortest prefix, among tokens from place `least` on, that has `want` tokens
// (by_sum false) or a sum of `want` (true): 54 bits, 11 at a time from the top.
SDY_DEV uint64_t prefix_end(const Row &r, uint64_t least, bool by_sum, uint64_t want, Lds &k) {
    uint64_t head = 0, before = 0;
    for (int shift = 44; shift > -11; shift -= 11) {
        const int s = shift < 0 ? 0 : shift, bits = shift < 0 ? 11 + shift : 11;
        __syncthreads();
        for (int i = threadIdx.x; i < 2048; i += THREADS) k.digit_count[i] = 0, k.digit_sum[i] = 0;
        __syncthreads();
        each(r.x, 0, r.n, [&](float v, int i) {
            const uint64_t at = place_of(v, i);
            if (at < least || at >> (s + bits) != head) return;
            const int d = (int)(at >> s) & ((1 << bits) - 1);
            if (by_sum) atomicAdd(&k.digit_sum[d], (unsigned long long)r.fixed(v));
            else atomicAdd(&k.digit_count[d], 1u);
        });
        __syncthreads();
        // the digits from the top, 8 a thread
        const int top = 2047 - 8 * (int)threadIdx.x;
        uint64_t mine = 0;
        for (int e = 0; e < 8; e++) mine += by_sum ? k.digit_sum[top - e] : k.digit_count[top - e];
        uint64_t whole;
        uint64_t run = before + block_scan(mine, &whole, k.parts);
        if (threadIdx.x == 0 && before + whole < want) k.parts.key = 0, k.parts.run = before;  // (fewer than wanted: the last)
        if (run < want && run + mine >= want) {
            int d = top;
            for (;; d--) {
                const uint64_t more = by_sum ? k.digit_sum[d] : k.digit_count[d];
                if (run + more >= want) break;
                run += more;
            }
            k.parts.key = (uint64_t)d;
            k.parts.run = run;
        }
        __syncthreads();
        head = head << bits | k.parts.key;
        before = k.parts.run;
    }
    return head;
}

// ---- the kernels
//
// Times of one row of 151936 logits with top-k and top-p, and of 61 rows of all kinds of parameters (37 MB): together 27 and
// 63 us. One row is bound by its five launches and what each waits for before its work (the row's maximum, the listed bins);
// 61 rows by reading 37 MB (max: 3.5 TB/s), by 64-bit exponentials of rows that need every token's w (bins), and by the
// chains of searches of a workgroup per row (cut, pick). Sorting a row is never needed; a row in one workgroup's hands from
// start to end took 800 us.

// 1000 tokens 15.5 us, 1000 such rows 33: the searches' steps, each a few barriers.
__global__ __launch_bounds__(THREADS) void k_sample_small(Args A) {
    extern __shared__ __align__(16) unsigned char lds_bytes[];
    Lds &k = *reinterpret_cast<Lds *>(lds_bytes);
    const int row = blockIdx.x, tid = threadIdx.x;
    Row r;
    r.params(A, row);
    uint64_t first = 0;
    each(r.x, 0, r.n, [&](float v, int i) {
        const uint64_t at = place_of(v, i);
        k.list[i] = at;
        first = at > first ? at : first;
    });
    r.start(block_max(first, k.parts), 0.0f);
    if (r.alone) {
        if (tid == 0) take_alone(A, row, r);
        return;
    }
    pick_listed(A, row, r, r.n, k);
}

// One row 4.1 us, 61 rows 10.6.
template <int W>
__global__ __launch_bounds__(64 * W) void k_sample_max(Args A) {
    __shared__ Parts<W> sh;
    const int c = blockIdx.x, row = blockIdx.y;
    const float *x = A.a.logits + (size_t)row * A.a.stride;
    const int lo = c * A.len, hi = lo + A.len < A.a.n_vocab ? lo + A.len : A.a.n_vocab;
    uint64_t first = 0;
    float low = INFINITY;
    each<64 * W>(x, lo, hi, [&](float v, int i) {
        const uint64_t at = place_of(v, i);
        first = at > first ? at : first;
        if (v > -INFINITY) low = fminf(low, v);
    });
    for (int off = 32; off >= 1; off >>= 1) low = fminf(low, __shfl_xor(low, off));
    if ((threadIdx.x & 63) == 0) sh.low[threadIdx.x >> 6] = low;
    first = block_max(first, sh);
    if (threadIdx.x == 0) {
        for (int w = 0; w < W; w++) low = fminf(low, sh.low[w]);
        A.work[row].first[c] = first;
        A.work[row].low[c] = low;
    }
}

// One row 3.9 us, 61 rows 13.
template <int W>
__global__ __launch_bounds__(64 * W) void k_sample_bins(Args A) {
    __shared__ Parts<W> sh;
    __shared__ unsigned count[BINS];
    __shared__ unsigned long long sum_of[BINS];
    const int c = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
    Row r;
    r.params(A, row);
    r.maxima(A, row);
    if (r.alone) return;
    const int lo = c * A.len, hi = lo + A.len < r.n ? lo + A.len : r.n;
    if (!r.cut()) {
        uint64_t sum = 0;
        each<64 * W>(r.x, lo, hi, [&](float v, int) { sum += r.fixed(v); });
        sum = block_sum(sum, sh);
        if (tid == 0) A.work[row].sums[c] = sum;
        return;
    }
    const bool sums = r.sums();
    for (int b = tid; b < BINS; b += 64 * W) count[b] = 0, sum_of[b] = 0;
    __syncthreads();
    each<64 * W>(r.x, lo, hi, [&](float v, int) {
        if (!(v > -INFINITY)) return;
        const int b = r.bin(v);
        atomicAdd(&count[b], 1u);
        if (sums) atomicAdd(&sum_of[b], (unsigned long long)r.fixed(v));
    });
    __syncthreads();
    const size_t at = ((size_t)row * A.pieces + c) * BINS;
    for (int b = tid; b < BINS; b += 64 * W) {
        A.count[at + b] = count[b];
        if (sums) A.sum[at + b] = sum_of[b];
    }
}

// A wave per piece, 16 bins a lane; then a bin per thread. One row 7.0 us, 61 rows 9.7.
__global__ __launch_bounds__(BINS) void k_sample_cut(Args A) {
    constexpr int W = BINS / 64, EACH = BINS / 64;
    static_assert(W == MAX_PIECES, "a wave per piece");
    __shared__ Parts<W> sh;
    __shared__ unsigned count_of[BINS], before_n[BINS + 1], listed_of[MAX_PIECES];
    __shared__ unsigned long long sum_of[BINS], before_s[BINS], part_s[W];
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, p = tid >> 6;
    Work &w = A.work[row];
    Row r;
    r.params(A, row);
    const bool sums = r.sums();
    count_of[tid] = 0;
    sum_of[tid] = 0;
    // (on their way before the row's greatest logit is known; a row that needs no cut has left them as they were)
    unsigned n[EACH];
    unsigned long long s[EACH];
    const size_t at = ((size_t)row * A.pieces + p) * BINS + lane;
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        n[e] = p < A.pieces ? A.count[at + 64 * e] : 0;
        s[e] = sums && p < A.pieces ? A.sum[at + 64 * e] : 0;
    }
    r.maxima(A, row);
    if (r.alone || !r.cut()) {
        if (tid == 0) w.mode = r.alone ? ROW_ALONE : ROW_ALL;
        return;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        if (n[e]) atomicAdd(&count_of[64 * e + lane], n[e]);
        if (s[e]) atomicAdd(&sum_of[64 * e + lane], s[e]);
    }
    __syncthreads();
    // the bins' running counts and sums
    const uint64_t count = count_of[tid], sum = sum_of[tid];
    const uint64_t run_n = wave_run<false>(count), run_s = wave_run<false>(sum);
    if (lane == 63) sh.part[p] = run_n, part_s[p] = run_s;
    __syncthreads();
    uint64_t n0 = run_n - count, s0 = run_s - sum, all_n = 0, all_s = 0;
#pragma unroll
    for (int q = 0; q < W; q++) {
        if (q < p) n0 += sh.part[q], s0 += part_s[q];
        all_n += sh.part[q];
        all_s += part_s[q];
    }
    const uint64_t want = r.top_k ? ((uint64_t)r.top_k < all_n ? (uint64_t)r.top_k : all_n) : r.top_p < 1.0f ? wanted(r.top_p, all_s) : ~0ull;
    before_n[tid] = (unsigned)n0;
    before_s[tid] = s0;
    if (r.top_k ? n0 < want && n0 + count >= want : s0 < want && s0 + sum >= want) sh.key = tid;
    if (tid == 0) before_n[BINS] = (unsigned)all_n;
    __syncthreads();
    int b0 = 0, b1 = BINS - 1, mode = ROW_SUM;
    if (r.top_k) {
        b1 = (int)sh.key;
        mode = ROW_TOP;
        if (before_n[b1 + 1] > LIST) {
            b0 = b1;
            mode = sums ? ROW_COUNT : ROW_SLOW;
        }
    } else {
        if (r.top_p < 1.0f) b0 = b1 = (int)sh.key;
        if (r.min_p > 0.0f) {
            // the bins that the border can be in: their arithmetic is in 32 bits
            const float far = r.min_p < 1.0f ? -logf(r.min_p) * r.temp * r.per_bin : 0.0f;
            const int lo = (int)fminf(far * (1.0f - 1e-5f), (float)(BINS - 1));
            // (with min_p 1 all those whose w rounds to 1: 2^-53 T down)
            const int hi = (int)fminf(far * (1.0f + 1e-5f) + 1e-5f + 0x1p-52f * r.temp * r.per_bin, (float)(BINS - 1));
            b0 = r.top_p < 1.0f && b0 < lo ? b0 : lo;
            b1 = hi < b1 ? hi : b1;
        }
    }
    const int listed = (int)(before_n[b1 + 1] - before_n[b0]);
    if (listed > LIST) mode = ROW_SLOW;
    if (tid == 0) {
        w.mode = mode;
        w.n_list = listed;
        w.b0 = b0;
        w.b1 = b1;
        w.before = mode == ROW_COUNT ? before_n[b0] : before_s[b0];
        w.want = want;
    }
    // the piece's sum before the listed bins, and its listed tokens' number
    uint64_t mine = 0, ahead = 0;
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const int b = 64 * e + lane;
        mine += b >= b0 && b <= b1 ? n[e] : 0;
        ahead += b < b0 ? s[e] : 0;
    }
    mine = wave_sum(mine);
    ahead = wave_sum(ahead);
    if (lane == 0) {
        listed_of[p] = (unsigned)mine;
        w.sums[p] = ahead;
    }
    __syncthreads();
    if (tid < A.pieces) {
        unsigned o = 0;
        for (int q = 0; q < tid; q++) o += listed_of[q];
        w.offset[tid] = o;
    }
    if (mode == ROW_COUNT) {  // the pick looks at the bins again
        w.count_of[tid] = (unsigned)count;
        w.sum_of[tid] = sum;
    }
}

// One row 3.1 us, 61 rows 8.4.
template <int W>
__global__ __launch_bounds__(64 * W) void k_sample_list(Args A) {
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
    each<64 * W>(r.x, lo, hi, [&](float v, int i) {
        if (!(v > -INFINITY)) return;
        const int b = r.bin(v);
        if (b >= b0 && b <= b1) w.list[atomicAdd(&next, 1u)] = place_of(v, i);
    });
}

// One row 5.6 us, 61 rows 16 to 19.
__global__ __launch_bounds__(THREADS) void k_sample_pick(Args A) {
    extern __shared__ __align__(16) unsigned char lds_bytes[];
    Lds &k = *reinterpret_cast<Lds *>(lds_bytes);
    const int row = blockIdx.x, tid = threadIdx.x;
    const Work &w = A.work[row];
    int mode = w.mode, n = w.n_list;
    if (mode == ROW_TOP || mode == ROW_SUM || mode == ROW_COUNT)
        for (int i = tid; i < n; i += THREADS) k.list[i] = w.list[i];
    Row r;
    r.params(A, row);
    r.maxima(A, row);
    if (mode == ROW_ALONE) {
        if (tid == 0) take_alone(A, row, r);
        return;
    }
    if (mode == ROW_TOP) {
        __syncthreads();
        pick_listed(A, row, r, n, k);
        return;
    }
    const float u = A.a.u[row];
    uint64_t least = 0;  // the place that the prefix ends at
    auto kept = [&](float x, int i) -> uint64_t {
        const uint64_t at = place_of(x, i);
        return at < least ? 0 : r.fixed_kept(at);
    };
    auto place = [&](int i) -> uint64_t { return k.list[i]; };
    auto w_of = [&](int i) -> uint64_t { return k.w[i]; };
    bool summed = false;  // k.sums: the pieces' sums before the listed tokens, k.w: these tokens' w
    if (mode == ROW_SUM || mode == ROW_ALL) {
        if (tid < A.pieces) k.sums[tid] = w.sums[tid];
        if (mode == ROW_SUM) {
            uint64_t sum = 0, last = ~0ull;
            __syncthreads();
            for (int i = tid; i < n; i += THREADS) {
                sum += k.w[i] = r.fixed(value_at(k.list[i]));
                last = k.list[i] < last ? k.list[i] : last;
            }
            sum = block_sum(sum, k.parts);
            if (r.top_p < 1.0f && w.before + sum >= w.want) least = find(n, place, w_of, w.before, w.want, k).key;
            else if (n) least = ~block_max(~last, k.parts);
        } else {
            n = 0;
        }
        __syncthreads();
        summed = true;
    } else if (mode == ROW_COUNT) {  // many tokens by count: the end of the first top_k is known now, and with it their sum
        int end = w.b0;  // the bin that the prefix ends in, whose tokens are listed
        __syncthreads();
        for (int i = tid; i < n; i += THREADS) k.w[i] = r.fixed(value_at(k.list[i]));
        const uint64_t rest = (uint64_t)r.top_k - w.before;
        if (rest < (uint64_t)n) least = find(n, place, [](int) -> uint64_t { return 1; }, 0, rest, k).key;
        else if (n) {
            uint64_t last = ~0ull;
            for (int i = tid; i < n; i += THREADS) last = k.list[i] < last ? k.list[i] : last;
            least = ~block_max(~last, k.parts);
        }
        if (r.top_p < 1.0f) {
            uint64_t sum = 0, ahead = 0;
            __syncthreads();
            for (int i = tid; i < n; i += THREADS) sum += k.list[i] < least ? (k.w[i] = 0) : k.w[i];
            sum = block_sum(sum, k.parts);
            for (int b = tid; b < w.b0; b += THREADS) ahead += w.sum_of[b];
            ahead = block_sum(ahead, k.parts);
            const uint64_t want = wanted(r.top_p, ahead + sum);
            if (ahead < want) {
                least = find(n, place, w_of, ahead, want, k).key;
            } else {  // the sum ends in an earlier bin, whose tokens nobody has listed
                const Found b = find(w.b0, [](int i) -> uint64_t { return (uint64_t)(BINS - i); }, [&](int i) -> uint64_t { return w.sum_of[i]; }, 0, want, k);
                end = BINS - (int)b.key;
                n = (int)w.count_of[end];
                if (n > LIST) {
                    mode = ROW_SLOW;
                } else {
                    if (tid == 0) k.n = 0;
                    __syncthreads();
                    each(r.x, 0, r.n, [&](float x, int i) {
                        if (x > -INFINITY && r.bin(x) == end) {
                            const int to = atomicAdd(&k.n, 1);
                            k.list[to] = place_of(x, i);
                            k.w[to] = r.fixed(x);
                        }
                    });
                    __syncthreads();
                    least = find(n, place, w_of, b.run, want, k).key;
                }
            }
        }
        // (a min-p can end before the listed bin)
        if (mode == ROW_COUNT && !(r.min_p > 0.0f)) {
            __syncthreads();
            for (int p = tid >> 6; p < A.pieces; p += WAVES) {
                const unsigned long long *of = A.sum + ((size_t)row * A.pieces + p) * BINS;
                uint64_t sum = 0;
#pragma unroll 4
                for (int b = tid & 63; b < end; b += 64) sum += of[b];
                sum = wave_sum(sum);
                if ((tid & 63) == 0) k.sums[p] = sum;
            }
            __syncthreads();
            summed = true;
        }
    }
    if (summed) {
        for (int i = tid; i < n; i += THREADS) {
            const uint64_t v = k.list[i] < least ? 0 : r.min_p > 0.0f ? r.fixed_kept(k.list[i]) : k.w[i];
            if (v) atomicAdd(&k.sums[index_at(k.list[i]) / A.len], (unsigned long long)v);
        }
        __syncthreads();
        uint64_t whole = 0;
        for (int p = 0; p < A.pieces; p++) whole += k.sums[p];
        uint64_t left = share(u, whole);
        int p = 0;
        while (p < A.pieces - 1 && k.sums[p] <= left) left -= k.sums[p++];
        const int lo = p * A.len, i = narrow(r.x, lo, lo + A.len < r.n ? lo + A.len : r.n, left, kept, k);
        if (tid == 0) take(A, row, i, kept(r.x[i], i), whole);
        return;
    }
    if (mode == ROW_SLOW) {
        least = 0;
        if (r.top_k) least = prefix_end(r, 0, false, (uint64_t)r.top_k, k);
        if (r.top_p < 1.0f) {
            uint64_t sum = 0;
            each(r.x, 0, r.n, [&](float v, int i) {
                if (place_of(v, i) >= least) sum += r.fixed(v);
            });
            sum = block_sum(sum, k.parts);
            least = prefix_end(r, least, true, wanted(r.top_p, sum), k);
        }
    }
    uint64_t whole = 0;
    each(r.x, 0, r.n, [&](float x, int i) { whole += kept(x, i); });
    whole = block_sum(whole, k.parts);
    const int i = narrow(r.x, 0, r.n, share(u, whole), kept, k);
    if (tid == 0) take(A, row, i, kept(r.x[i], i), whole);
}

int pieces_of(int n_vocab) {
    const int p = (n_vocab + LIST - 1) / LIST;
    return p < MAX_PIECES ? p : MAX_PIECES;
}

}  // namespace

extern "C" size_t sdy_sample_ws_bytes(int n_rows, int n_vocab) {
    if (n_rows < 1 || n_rows > 65535 || n_vocab < 1 || n_vocab > MAX_VOCAB) return 0;
    if (n_vocab <= SMALL) return 16;
    return (size_t)n_rows * (sizeof(Work) + (size_t)pieces_of(n_vocab) * BINS * 12);
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
    A.pieces = pieces_of(a->n_vocab);
    A.len = ((a->n_vocab + A.pieces - 1) / A.pieces + 3) & ~3;
    A.work = (Work *)a->ws;
    A.sum = (unsigned long long *)(A.work + a->n_rows);
    A.count = (unsigned *)(A.sum + (size_t)a->n_rows * A.pieces * BINS);
    static size_t granted[2];
    const bool small = a->n_vocab <= SMALL;
    const int rc = sdy_lds_limit(small ? (const void *)k_sample_small : (const void *)k_sample_pick, sizeof(Lds), &granted[small]);
    if (rc) return rc;
    const dim3 rows(a->n_rows), grid(A.pieces, a->n_rows), block(THREADS);
    hipStream_t st = (hipStream_t)s;
    if (small) {
        hipLaunchKernelGGL(k_sample_small, rows, block, sizeof(Lds), st, A);
    } else {
        const bool few = a->n_rows <= FEW_ROWS;
        const dim3 wide(1024);
        if (few) {
            hipLaunchKernelGGL(k_sample_max<16>, grid, wide, 0, st, A);
            hipLaunchKernelGGL(k_sample_bins<16>, grid, wide, 0, st, A);
        } else {
            hipLaunchKernelGGL(k_sample_max<4>, grid, block, 0, st, A);
            hipLaunchKernelGGL(k_sample_bins<4>, grid, block, 0, st, A);
        }
        hipLaunchKernelGGL(k_sample_cut, rows, dim3(BINS), 0, st, A);
        if (few) hipLaunchKernelGGL(k_sample_list<16>, grid, wide, 0, st, A);
        else hipLaunchKernelGGL(k_sample_list<4>, grid, block, 0, st, A);
        hipLaunchKernelGGL(k_sample_pick, rows, block, sizeof(Lds), st, A);
    }
    return sdy_check_launch("sample");
}
