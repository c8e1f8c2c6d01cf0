// Attention of a tree of drafted tokens over the cache and over their own ancestors.
//
// Node t of a head takes the scores q_t.k_j / sqrt(head_dim) over every cached position j < n_past and over the drafted
// rows of t and the nodes above it (parent, its parent, ...), one softmax over them, and the weighted sum of the V rows.
// A parent outside [0, t) makes t a root; below -1 it marks a place without a node: its output row stays as it was and no
// node attends to it.
//
//   k_tree_part<HD, KT, RW, KW>  one workgroup per (span of positions, kv head, block of 32 RW rows); a row is a node
//   and one of the query heads that share the kv head, so a K/V tile is read once for all of them. The first spans are the
//   drafted rows, a turn each.
//   RW waves of 32 rows share each tile of 32 positions, KW groups of them take tiles in turn. Per tile a wave computes
//   S^T = K Q^T (a lane holds one row's 16 scores), P = exp2(S - m), and O^T += V^T P. In turn t it multiplies K of tile t + 1
//   while it makes P of tile t, then V of tile t while it splits K of tile t + 2 and V of tile t + 1 into the other buffers.
//   k_tree_merge<HD>  one workgroup per node and head: the spans' (m, l, O) in span order.
//
// Products on the f16 matrix cores at f32's precision: an f32 is the sum of two f16 (22 bits and a sign) once it is scaled by
// a power of two that keeps it well inside f16's range. q, P and an f32 cache's K and V are split so, an f16 cache's values are
// taken as they are; of the split products low x low, at most 2^-22 of the whole, is left out. A row of q goes by its own
// greatest value. A span's K and V go by fixed powers, which suit a greatest value of 2^-5 to 2^10 (K) or 2^-9 to 2^6 (V): its
// low part's least bit is then 2^-24 of it or less; a span outside of that is computed again with its own powers. Powers of
// two go back exactly: K's and q's into the scores' factor, V's into O (ldexp). The running maximum m is kept as a whole
// number, so that its rescales are exact too, and grows only when a score passes it by 2^LAG: P is 2^4 to 2^15 at the greatest
// weight, f16's least bit 2^-28 of it or less.
//
// What bounds it. A full tree over a long cache: the matrix cores. 64 nodes of 32 heads (4 kv heads of 128 dims) over 40000
// f32 positions are 126 GFLOP of f16 products and 164 MB of K and V: 130 to 133 us, k_tree_part 124 of them, 1.02 PFLOP/s (a
// large f16 matrix product of the library reaches 1.28; matrix units busy 61% of the cycles, at about 2.0 GHz). Products and
// other work are written side by side (fix() below) because a wave's own order decides what overlaps: in the compiler's order,
// with four waves to a tile, the same case took 159 us. Few nodes over a short cache: latency. 5 nodes of 16 heads over 700
// positions 13.1 us, k_tree_part 8.2 to 10 (a launch, the chain past -> K -> scores -> O, and code that every launch fetches
// anew, about 40 ns per 64 bytes), k_tree_merge 3.8. Between them both: 61 nodes of 32 heads over 4099 positions 33 us, 12.5
// GFLOP and 28 MB of parts written and read again. With f32 products on the f32 matrix cores (146 TFLOP/s at best) the first
// case would take 290 us.
#include <type_traits>

#include "sdy_attn_dev.h"
#include "sdy_device.h"
#include "sdy_internal.h"
#include "sdy_ops.h"

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int MAX_NODES = 256;
constexpr int KB = 32;         // positions per tile
constexpr int TOP = 13;        // a row of q, and a span computed again, are scaled to a greatest value of 2^TOP .. 2^(TOP + 1)
constexpr int K_SCALE = 5, V_SCALE = 9;  // the powers that K and V are scaled by at first
constexpr float P_BITS = 4;    // P is 2^P_BITS exp2(score - m), of scores up to m + LAG
constexpr float LAG = 11;
constexpr int MAX_PARTS = 512 + MAX_NODES / KB;
constexpr int MAX_PAST = 1 << 28;  // 512 spans of at most 2^30 bytes hold them

struct TreeArgs {
    sdy_attn_tree_args a;
    int rows;       // per kv head: n_tok * (n_head / n_kv_head)
    int n_block;    // row blocks
    int n_draft;    // spans of drafted rows
    int n_span;     // spans of cached positions (the grid's; those in use follow from n_past)
    int least;      // turns of such a span, at least, where there are many
    int granule;    // positions of one turn of a workgroup: 32 KW
    float log_scale;  // log2(e) / sqrt(head_dim)
    float *part;    // [n_draft + n_span][n_kv_head * rows][HD], then the (m, l) [n_draft + n_span][n_kv_head * rows][2]
};

// The rounds (granules) per span and the spans in use for so many positions. One group of waves takes two tiles where there
// are more than 128 of them over the kv heads, half the parts to merge (24 nodes of 16 heads over 2500: 19.7 against 22.8 us with
// one, 32 of 32 heads over 1500 23.1 against 28.0; 5 of 16 heads over 700 13.9 against 13.2, 16 of them 16.3 against 15.9).
SDY_DEV int span_rounds(const TreeArgs &A, int past) {
    const int n = (past + A.granule - 1) / A.granule, per = (n + A.n_span - 1) / A.n_span;
    const int least = (long)n * A.a.n_kv_head > 128 ? A.least : 1;
    return per > least ? per : least;
}
SDY_DEV int spans_used(const TreeArgs &A, int past) {
    const int per = span_rounds(A, past), n = (past + A.granule - 1) / A.granule;
    return (n + per - 1) / per;
}

template <int HD, class KT, int RW, int KW>
struct Lds {
    static constexpr bool F32 = std::is_same<KT, float>::value;
    static constexpr int NP = F32 ? 2 : 1;    // f16 parts of a K or V value
    // f16 of a row: K's rows start 4 banks apart (eight lanes read 16 bytes of a row each), V's 8 (four rows' 32 bytes)
    static constexpr int KS = HD + 8, VS = HD + 16;
    static constexpr int KPLANE = 32 * KS, VPLANE = 32 * VS, TILE = NP * (KPLANE + VPLANE);
    static constexpr size_t tiles = (size_t)KW * 2 * TILE * 2;  // two of each
    static constexpr int ROWS = 32 * RW, OS = HD + 4;
    static constexpr size_t merge = KW > 1 ? (size_t)KW * ROWS * (OS + 2) * 4 : 0;
    static constexpr size_t body = tiles > merge ? tiles : merge;
    // the nodes' masks and their farthest known ancestors; per 32 nodes, those with rows that hold (ok) and that do not (bad)
    static constexpr size_t masks = MAX_NODES * (MAX_NODES / 32) * 4 + MAX_NODES * 2 + 2 * 16 * 4;
    static constexpr size_t flags = 2 * 4;      // the greatest |K| and |V|
    static constexpr size_t bytes = body + masks + flags;
    static_assert(bytes <= 160 * 1024, "fits a CU");
};

// Two f32 as two f16 pairs, hi + lo = x up to 2^-23 of x (while lo is at least f16's least normal)
SDY_DEV void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    float minus = -1.0f;  // (not left as a constant: one mixed multiply-add instead of a conversion and a difference)
    __asm__("" : "+s"(minus));
    const f16x2 h = __builtin_convertvector(f32x2{a, b}, f16x2);
    const f16x2 l = __builtin_convertvector(f32x2{__builtin_fmaf((float)h[0], minus, a), __builtin_fmaf((float)h[1], minus, b)}, f16x2);
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, l);
}

// max(m, |a|, |b|) in one instruction (fmaxf makes its operands canonical first)
SDY_DEV float max3_abs(float m, uint32_t a, uint32_t b) {
    __asm__("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(m) : "v"(a), "v"(b));
    return m;
}

// The power of two that brings a greatest |value| (one of at least 2^-100) to 2^TOP .. 2^(TOP + 1)
SDY_DEV int power_for(float most) {
    const int e = (int)(__float_as_uint(most) >> 23) - 127;
    return TOP - (e > -100 ? e : -100);
}
SDY_DEV float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// Rows of K and V on their way to LDS: thread tg of a group of 64 RW holds chunks of CE consecutive elements of one row.
template <int HD, class KT, int RW>
struct Stage {
    static constexpr bool F32 = std::is_same<KT, float>::value;
    static constexpr int LPR = 2 * RW;                              // lanes of a row
    static constexpr int CE = HD / 8 >= LPR ? 8 : 4;                // elements of a chunk
    static constexpr int NC = HD / CE / LPR;                        // chunks of a lane
    static constexpr int W = CE * (int)sizeof(KT) / 4;              // words of a chunk
    static_assert(NC >= 1 && HD == NC * CE * LPR, "a row's chunks divide over its lanes");
    uint32_t r[NC][W];
    SDY_DEV void load(__amdgpu_buffer_rsrc_t rs, uint32_t key, int tg) {
        const uint32_t o = (key + (uint32_t)(tg / LPR)) * (uint32_t)(HD * sizeof(KT)) + (uint32_t)(tg % LPR) * (CE * sizeof(KT));
#pragma unroll
        for (int i = 0; i < NC; i++) {
            const uint32_t at = o + (uint32_t)(i * LPR * CE * sizeof(KT));
            if constexpr (W >= 4) {
#pragma unroll
                for (int x = 0; x < W; x += 4) {
                    const auto u = __builtin_amdgcn_raw_buffer_load_b128(rs, at + 4 * x, 0, 0);
                    for (int w = 0; w < 4; w++) r[i][x + w] = u[w];
                }
            } else {
                const auto u = __builtin_amdgcn_raw_buffer_load_b64(rs, at, 0, 0);
                for (int w = 0; w < 2; w++) r[i][w] = u[w];
            }
        }
    }
    // 0, or NaN where this thread's values have an infinity or a NaN
    SDY_DEV float zeros() const {
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; i++)
#pragma unroll
            for (int w = 0; w < W; w++) {
                if constexpr (F32) z = __builtin_fmaf(__uint_as_float(r[i][w]), 0.0f, z);
                else z = __builtin_fmaf(sdy_h2f((uint16_t)r[i][w]), 0.0f, __builtin_fmaf(sdy_h2f((uint16_t)(r[i][w] >> 16)), 0.0f, z));
            }
        return z;
    }
    SDY_DEV void clear() {
#pragma unroll
        for (int i = 0; i < NC; i++)
#pragma unroll
            for (int w = 0; w < W; w++) r[i][w] = 0;
    }
    static constexpr int PAIRS = NC * CE / 2;  // pairs of values
    uint32_t part[F32 ? 2 : 1][PAIRS];
    // the greatest of m and an f32 pair's |values|
    SDY_DEV float most_of(int j, float m) const {
        if constexpr (F32) return max3_abs(m, r[2 * j / CE][2 * j % CE], r[2 * j / CE][2 * j % CE + 1]);
        else return m;
    }
    // pair j's parts (f32: of the values times sc)
    SDY_DEV void split(int j, float sc) {
        const int i = 2 * j / CE, w = 2 * j % CE;
        if constexpr (F32) split2(__uint_as_float(r[i][w]) * sc, __uint_as_float(r[i][w + 1]) * sc, part[0][j], part[1][j]);
        else part[0][j] = r[i][w / 2];
    }
    // all parts to the planes at dst, rows RS apart
    template <int RS>
    SDY_DEV void store(uint16_t *dst, int tg) const {
        uint16_t *d = dst + (tg / LPR) * RS + (tg % LPR) * CE;
#pragma unroll
        for (int i = 0; i < NC; i++)
#pragma unroll
            for (int p = 0; p < (F32 ? 2 : 1); p++) {
                uint16_t *to = d + p * 32 * RS + i * LPR * CE;
                const uint32_t *x = part[p] + i * CE / 2;
                if constexpr (CE == 8) *reinterpret_cast<u32x4 *>(to) = u32x4{x[0], x[1], x[2], x[3]};
                else *reinterpret_cast<u32x2 *>(to) = u32x2{x[0], x[1]};
            }
    }
};

// Which nodes each node sees, as bits: mask[t] starts as t itself, then takes that of the farthest node known above it and
// that one's farthest in turn, doubling the distance. The first 256 threads do (up to 64 nodes, in the first wave's registers: 5
// nodes over 700 positions 13.7 -> 12.9 us, 24 16.6 -> 16.4, 61 20.8 -> 20.6); p0 is the parent of node tid.
SDY_DEV void ancestor_masks(int p0, int n, uint32_t (*mask)[MAX_NODES / 32], int16_t *up) {
    constexpr int W = MAX_NODES / 32;
    const int tid = threadIdx.x, words = (n + 31) / 32;
    if (n <= 64) {  // one wave, in registers
        if (tid < 64) {
            uint64_t sees = p0 >= -1 ? 1ull << tid : 0;
            int p = p0 < 0 || p0 >= tid ? -1 : p0;
            if (__shfl(p0, p & 63) < -1) p = -1;  // under an empty place: a root
            for (int reach = 1; reach < n; reach *= 2) {
                const uint64_t s = __shfl((unsigned long long)sees, p & 63);
                const int far = __shfl(p, p & 63);
                if (p >= 0) sees |= s, p = far;
            }
#pragma unroll
            for (int w = 0; w < W; w++) mask[tid][w] = w == 0 ? (uint32_t)sees : w == 1 ? (uint32_t)(sees >> 32) : 0u;
        }
        __syncthreads();
        return;
    }
    const bool mine = tid < MAX_NODES;
    if (mine) {
        up[tid] = (int16_t)(p0 < -1 ? -2 : p0 < 0 || p0 >= tid ? -1 : p0);
#pragma unroll
        for (int w = 0; w < W; w++) mask[tid][w] = p0 >= -1 && w == tid / 32 ? 1u << (tid % 32) : 0u;
    }
    __syncthreads();
    int p = mine ? up[tid] : -1;
    if (p >= 0 && up[p] < -1) p = -1;  // under an empty place: a root
    __syncthreads();
    if (mine) up[tid] = (int16_t)p;
    __syncthreads();
    for (int reach = 1; reach < n; reach *= 2) {
        uint32_t add[W];
        int far = -1;
        if (p >= 0) {
            far = up[p];
            for (int w = 0; w < words; w++) add[w] = mask[p][w];
        }
        __syncthreads();
        if (p >= 0) {
            for (int w = 0; w < words; w++) mask[tid][w] |= add[w];
            up[tid] = (int16_t)far;
            p = far;
        }
        __syncthreads();
    }
}

// The work of one span: all of its tiles, (m, l, O) in registers.
template <int HD, class KT, int RW, int KW, bool DRAFT>
struct Span {
    using L = Lds<HD, KT, RW, KW>;
    using St = Stage<HD, KT, RW>;
    static constexpr bool F32 = L::F32;
    static constexpr int NP = L::NP, KS = L::KS, VS = L::VS, ND = HD / 32, NS = HD / 16;
    // given
    uint16_t *tiles;
    const uint32_t *sees;        // DRAFT: this row's nodes
    const uint32_t *ok, *bad;    // DRAFT: rows that hold and that do not, per 32 nodes
    unsigned *greatest;
    __amdgpu_buffer_rsrc_t rk, rv;
    int n_keys, rounds, kw, tg, tid, lane, hh, ql;
    bool live;                   // whether this wave has rows (one without only brings tiles)
    float log_scale;             // log2(e) / sqrt(HD), over the power that q is scaled by
    f16x8 qh[NS], qlo[NS];
    // made
    f32x16 o[ND];
    float m, l;  // m whole
    int pk, pv;  // the powers that K and V are scaled by

    SDY_DEV uint32_t at_round(int it) const { return (uint32_t)((it * KW + kw) * KB); }  // the group's first position in the span
    SDY_DEV void drafted(St &st, int it) const {
        if constexpr (DRAFT) {
            const uint32_t t = at_round(it) / KB;
            if (!((ok[t] & ~bad[t]) >> (tg / St::LPR) & 1)) st.clear();
        }
    }
    SDY_DEV const uint16_t *k_row(int it) const { return tiles + (it & 1) * NP * L::KPLANE + ql * KS + 8 * hh; }
    SDY_DEV static f16x8 frag(const uint16_t *p) { return *reinterpret_cast<const f16x8 *>(p); }
    SDY_DEV static f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    // nothing moves across: products and other work stay side by side as they are written
    SDY_DEV static void fix() { __builtin_amdgcn_sched_barrier(0); }
    // what a tile's row does not see; register r of the scores is position 8 (r / 4) + 4 hh + r % 4 of the tile
    SDY_DEV void masked(f32x16 &s, int it) {
        const int k0 = (int)at_round(it);
        if (!DRAFT && k0 + KB <= n_keys) return;
        __asm__ volatile("");  // (a branch: not worth a select per score)
        uint32_t bits = k0 >= n_keys ? 0u : n_keys - k0 >= KB ? ~0u : (1u << (n_keys - k0)) - 1;
        if constexpr (DRAFT) {
            bits = k0 < n_keys && sees ? sees[k0 / KB] : 0u;
            if (bits & bad[k0 / KB]) l = NAN;
        }
        bits >>= 4 * hh;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const uint32_t see = (uint32_t)__builtin_amdgcn_sbfe((int)bits, 8 * (r >> 2) + (r & 3), 1);
            s[r] = __uint_as_float((__float_as_uint(s[r]) & see) | (0xFF800000u & ~see));
        }
    }
    // One pass; the greatest |K| and |V| that this thread met.
    SDY_DEV void pass(float &greatest_k, float &greatest_v) {
        St sk, sv;
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] = f32x16{};
        m = -INFINITY;
        l = 0.0f;
        greatest_k = greatest_v = 0.0f;
        // (never 0, which would make a masked score NaN: with q and K below 2^-100 every score is 0 all the same)
        const float factor = fmaxf(ldexpf(log_scale, -pk), 0x1p-126f), fk = pow2(pk), fv = pow2(pv);
        // K and V of turn `it` into their buffers, the next ones on their way
        auto put_k = [&](int it) {
            sk.template store<KS>(tiles + (it & 1) * NP * L::KPLANE, tg);
            sk.load(rk, at_round(it + 1), tg);
        };
        auto put_v = [&](int it) {
            sv.template store<VS>(tiles + 2 * NP * L::KPLANE + (it & 1) * NP * L::VPLANE, tg);
            sv.load(rv, at_round(it + 1), tg);
        };
        constexpr int PAIRS = St::PAIRS;
        __syncthreads();
        sk.load(rk, at_round(0), tg);
        sv.load(rv, at_round(0), tg);
#pragma unroll 1
        for (int it = 0; it < 2 && it < rounds; it++) {  // (the scores of a turn that is none are masked, whatever K is)
            drafted(sk, it);
#pragma unroll
            for (int j = 0; j < PAIRS; j++) greatest_k = sk.most_of(j, greatest_k), sk.split(j, fk);
            put_k(it);
        }
        drafted(sv, 0);
#pragma unroll
        for (int j = 0; j < PAIRS; j++) greatest_v = sv.most_of(j, greatest_v), sv.split(j, fv);
        put_v(0);
        __syncthreads();
        f32x16 s = f32x16{};
        if (live) {
            const uint16_t *kr = k_row(0);
#pragma unroll
            for (int i = 0; i < NS; i++) {
                const f16x8 k = frag(kr + 16 * i);
                s = mfma(k, qlo[i], s);
                if constexpr (F32) s = mfma(frag(kr + L::KPLANE + 16 * i), qh[i], s);
                s = mfma(k, qh[i], s);
            }
        }
        masked(s, 0);
        float mt = s[0];  // the row's greatest score of the tile
#pragma unroll
        for (int r = 1; r < 16; r++) mt = fmaxf(mt, s[r]);
#pragma unroll 1
        for (int it = 0; it < rounds; it++) {
            __syncthreads();
            // a row whose scores pass its maximum too far: all that it has, down by the difference of two whole numbers
            mt = fmaxf(mt, __shfl_xor(mt, 32)) * factor;
            if (__ballot(mt > m + LAG || (mt > -INFINITY && m == -INFINITY))) {
                const float up_to = mt > m + LAG || m == -INFINITY ? ceilf(mt) : m;
                const int down = m == -INFINITY ? -300 : (int)fmaxf(m - up_to, -300.0f);
                m = up_to;
                l = ldexpf(l, down);
                if (it > 0) {
#pragma unroll
                    for (int d = 0; d < ND; d++)
#pragma unroll
                        for (int e = 0; e < 16; e++) o[d][e] = ldexpf(o[d][e], down);
                }
            }
            const float mu = P_BITS - (m == -INFINITY ? 0.0f : m);  // nothing seen yet: every weight is 0
            // S of turn it + 1, a step of 16 dims at a time; beside it P of turn `it`, in 8 pairs
            f32x16 next = f32x16{};
            u32x4 ph[2] = {}, pl[2] = {};
            if (live) {
                const uint16_t *kr = k_row(it + 1);
                f16x8 k = frag(kr), k2 = frag(kr + (NP - 1) * L::KPLANE);
                constexpr int EACH = NS < 8 ? 8 / NS : 1, EVERY = NS > 8 ? NS / 8 : 1;
                float x[EACH], y[EACH];
                fix();
#pragma unroll
                for (int i = 0; i < NS; i++) {
                    const int i1 = i + 1 < NS ? i + 1 : i;
                    const f16x8 kn = frag(kr + 16 * i1), kn2 = frag(kr + (NP - 1) * L::KPLANE + 16 * i1);
                    const bool on = i % EVERY == 0;
                    const int j0 = i / EVERY * EACH;
                    next = mfma(k, qlo[i], next);
                    fix();
                    if (on)
#pragma unroll
                        for (int e = 0; e < EACH; e++) {
                            x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * (j0 + e)], factor, mu));
                            y[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * (j0 + e) + 1], factor, mu));
                            __asm__ volatile("" : "+v"(x[e]), "+v"(y[e]));  // (made here, not where it is used)
                        }
                    fix();
                    if constexpr (F32) next = mfma(k2, qh[i], next);
                    fix();
                    if (on)
#pragma unroll
                        for (int e = 0; e < EACH; e++) {
                            l += x[e] + y[e];
                            uint32_t h0, l0;
                            split2(x[e], y[e], h0, l0);
                            __asm__ volatile("" : "+v"(h0), "+v"(l0));
                            ph[(j0 + e) / 4][(j0 + e) % 4] = h0;
                            pl[(j0 + e) / 4][(j0 + e) % 4] = l0;
                        }
                    fix();
                    next = mfma(k, qh[i], next);
                    k = kn;
                    k2 = kn2;
                }
                fix();
            }
            masked(next, it + 1);
            drafted(sk, it + 2);
            drafted(sv, it + 1);
            // O, 32 dims and 16 positions a step: u: positions 16 u + 4 hh .. + 3 and 16 u + 8 + 4 hh .. + 3 of the tile, the
            // scores' registers 8 u ..; beside it the greatest of the next scores, K of turn it + 2 and V of turn it + 1
            {
                const uint16_t *const vt = tiles + 2 * NP * L::KPLANE + (it & 1) * NP * L::VPLANE + (4 * hh + ((lane & 15) >> 2)) * VS +
                                           16 * ((lane >> 4) & 1) + 4 * (lane & 3);
                // V^T by transposing reads: 16 lanes give the addresses of 4 rows x 16 dims (4 each) and get a dim's 4 rows
                auto vread = [&](int plane, int step) {
                    const uint16_t *at = vt + plane * L::VPLANE + 16 * (step / ND) * VS + 32 * (step % ND);
                    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)at);
                    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(at + 8 * VS));
                    return __builtin_bit_cast(f16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
                };
                constexpr int STEPS = 2 * ND, EACH = (2 * PAIRS + STEPS - 1) / STEPS, MORE = 16 / STEPS;
                f16x8 v = vread(0, 0), v2 = vread(NP - 1, 0);
                mt = next[0];
                fix();
#pragma unroll
                for (int step = 0; step < STEPS; step++) {
                    const int u = step / ND, d = step % ND, s1 = step + 1 < STEPS ? step + 1 : step;
                    const f16x8 vn = vread(0, s1), vn2 = vread(NP - 1, s1);
                    o[d] = mfma(v, __builtin_bit_cast(f16x8, pl[u]), o[d]);
                    fix();
                    auto work = [&](int e) {
                        const int j = EACH * step + e;
                        if (j < PAIRS) {
                            greatest_k = sk.most_of(j, greatest_k);
                            sk.split(j, fk);
                        } else if (j < 2 * PAIRS) {
                            const int i = j - PAIRS;
                            greatest_v = sv.most_of(i, greatest_v);
                            sv.split(i, fv);
                        }
                    };
#pragma unroll
                    for (int e = 0; e < EACH / 2; e++) work(e);
                    fix();
                    if constexpr (F32) o[d] = mfma(v2, __builtin_bit_cast(f16x8, ph[u]), o[d]);
                    fix();
#pragma unroll
                    for (int e = EACH / 2; e < EACH; e++) work(e);
#pragma unroll
                    for (int r = 0; r < MORE; r++) mt = fmaxf(mt, next[MORE * step + r]);
                    fix();
                    o[d] = mfma(v, __builtin_bit_cast(f16x8, ph[u]), o[d]);
                    v = vn;
                    v2 = vn2;
                }
                fix();
            }
            s = next;
            put_k(it + 2);
            put_v(it + 1);
        }
    }
    SDY_DEV void run() {
        pk = F32 ? K_SCALE : 0;
        pv = F32 ? V_SCALE : 0;
        for (;;) {
            float gk, gv;
            pass(gk, gv);
            if constexpr (!F32) return;
            // K or V beyond their powers, or so small that the low parts lack bits: once more, with the span's own
            if (pk != K_SCALE || pv != V_SCALE) return;
            if (tid < 2) greatest[tid] = 0;
            __syncthreads();
            for (int off = 32; off >= 1; off >>= 1) {
                gk = fmaxf(gk, __shfl_xor(gk, off));
                gv = fmaxf(gv, __shfl_xor(gv, off));
            }
            if (lane == 0) {
                atomicMax(&greatest[0], __float_as_uint(gk));
                atomicMax(&greatest[1], __float_as_uint(gv));
            }
            __syncthreads();
            gk = __uint_as_float(greatest[0]);
            gv = __uint_as_float(greatest[1]);
            const bool fits_k = gk == 0.0f || (gk >= pow2(-K_SCALE) && gk <= pow2(15 - K_SCALE));
            const bool fits_v = gv == 0.0f || (gv >= pow2(-V_SCALE) && gv <= pow2(15 - V_SCALE));
            if (fits_k && fits_v) return;
            if (!fits_k) pk = power_for(gk);
            if (!fits_v) pv = power_for(gv);
        }
    }
};

template <int HD, class KT, int RW, int KW>
__global__ __launch_bounds__(64 * RW * KW, 1) void k_tree_part(TreeArgs A) {
    using L = Lds<HD, KT, RW, KW>;
    using St = Stage<HD, KT, RW>;
    constexpr bool F32 = L::F32;
    constexpr int ND = HD / 32, NS = HD / 16, GROUP = 64 * RW, THREADS = GROUP * KW;
    static_assert(THREADS >= MAX_NODES, "a thread per node");
    extern __shared__ __align__(16) unsigned char lds_bytes[];
    const sdy_attn_tree_args &a = A.a;
    // all row blocks of one span and kv head on one XCD (workgroups are dealt to the 8 in turn): its L2 holds the tile
    const int pairs = (A.n_draft + A.n_span) * a.n_kv_head;
    const int id = (int)blockIdx.x, pair = (id / 8 / A.n_block) * 8 + id % 8, block = id / 8 % A.n_block;
    if (pair >= pairs) return;
    const int part = pair / a.n_kv_head, g = pair - part * a.n_kv_head;
    const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5, ql = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), rw = wave / KW, kw = wave % KW, tg = rw * 64 + lane;
    const bool draft = part < A.n_draft;
    const int rep = a.n_head / a.n_kv_head;
    const int row = (block * RW + rw) * 32 + ql;
    const int past = *a.n_past;
    const int node = row < A.rows ? row / rep : 0;
    const int p0 = draft && tid < a.n_tok ? a.parent[tid] : -2;

    // the row's queries: step i holds dims 16 i + 8 hh .. + 7
    f16x8 qh[NS], qlo[NS];
    float log_scale;
    {
        const float *q = a.q + (size_t)node * a.q_stride + (size_t)(g * rep + (row < A.rows ? row - node * rep : 0)) * HD + 8 * hh;
        float most = 0.0f;
        float4 v[2 * NS];
#pragma unroll
        for (int i = 0; i < NS; i++) {
            v[2 * i] = *reinterpret_cast<const float4 *>(q + 16 * i);
            v[2 * i + 1] = *reinterpret_cast<const float4 *>(q + 16 * i + 4);
        }
#pragma unroll
        for (int i = 0; i < 2 * NS; i++) {
            most = max3_abs(most, __float_as_uint(v[i].x), __float_as_uint(v[i].y));
            most = max3_abs(most, __float_as_uint(v[i].z), __float_as_uint(v[i].w));
        }
        most = fmaxf(most, __shfl_xor(most, 32));
        const int eq = power_for(most);
        const float sc = pow2(eq);
        log_scale = ldexpf(A.log_scale, -eq);
#pragma unroll
        for (int i = 0; i < NS; i++) {
            u32x4 h, l;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float4 x = v[2 * i + e];
                uint32_t h0, l0, h1, l1;
                split2(x.x * sc, x.y * sc, h0, l0);
                split2(x.z * sc, x.w * sc, h1, l1);
                h[2 * e] = h0, h[2 * e + 1] = h1, l[2 * e] = l0, l[2 * e + 1] = l1;
            }
            qh[i] = __builtin_bit_cast(f16x8, h);
            qlo[i] = __builtin_bit_cast(f16x8, l);
        }
    }

    if (past < 0 || past > a.max_past) return;
    int lo = part * A.granule, hi = lo + A.granule < a.n_tok ? lo + A.granule : a.n_tok;
    if (draft) {
        const int last = (block + 1) * 32 * RW < A.rows ? (block + 1) * 32 * RW - 1 : A.rows - 1;
        if (lo > last / rep) return;  // none of the block's nodes sees a later one, nor does the merge look
    } else {
        const int per = span_rounds(A, past) * A.granule;
        const long l0 = (long)(part - A.n_draft) * per, h0 = l0 + per;
        if (l0 >= past) return;  // the merge does not look at it
        lo = (int)l0;
        hi = h0 < past ? (int)h0 : past;
    }
    const long from = ((long)g * (draft ? a.draft_stride : a.head_stride) + (long)lo * HD) * (long)sizeof(KT);
    const int n_keys = hi - lo, size = n_keys * (int)(HD * sizeof(KT));  // (a span's bytes fit 31 bits: the host sees to it)
    // positions past the span's end read as zeros and are masked
    const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void *)((const char *)(draft ? a.k_draft : a.k_cache) + from), (short)0, size, 0x00020000);
    const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void *)((const char *)(draft ? a.v_draft : a.v_cache) + from), (short)0, size, 0x00020000);
    const int rounds = (n_keys + KB * KW - 1) / (KB * KW);

    uint32_t(*const mask)[MAX_NODES / 32] = reinterpret_cast<uint32_t(*)[MAX_NODES / 32]>(lds_bytes + L::body);
    int16_t *const up = reinterpret_cast<int16_t *>(mask + MAX_NODES);
    uint32_t *const ok = reinterpret_cast<uint32_t *>(up + MAX_NODES), *const bad = ok + 16;

    f32x16 o[ND];
    float m, l;
    int pv;
    auto span = [&](auto w) {
        w.tiles = reinterpret_cast<uint16_t *>(lds_bytes) + kw * 2 * L::TILE;
        const int tile = draft ? lo / KB : 0;
        w.sees = row < A.rows ? mask[node] + tile : nullptr;
        w.ok = ok + tile;
        w.bad = bad + tile;
        w.greatest = bad + 16;
        w.rk = rk;
        w.rv = rv;
        w.n_keys = n_keys;
        w.rounds = rounds;
        w.kw = kw;
        w.tg = tg;
        w.tid = tid;
        w.lane = lane;
        w.hh = hh;
        w.ql = ql;
        w.live = (block * RW + rw) * 32 < A.rows;
        w.log_scale = log_scale;
#pragma unroll
        for (int i = 0; i < NS; i++) w.qh[i] = qh[i], w.qlo[i] = qlo[i];
        w.run();
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] = w.o[d];
        m = w.m;
        l = w.l;
        pv = w.pv;
    };
    if (draft) {
        // which nodes see which, and rows that are left out: an empty place's, and those with an infinity or a NaN (NaN for
        // the nodes that see them, nothing for the others)
        St sk, sv;
        sk.load(rk, (uint32_t)(kw * KB), tg);
        sv.load(rv, (uint32_t)(kw * KB), tg);
        if (tid < 32) ok[tid] = 0;
        ancestor_masks(p0, a.n_tok, mask, up);
        const float z = sk.zeros() + sv.zeros();
        const int t = lo + kw * KB + tg / St::LPR;
        if (t < a.n_tok && (mask[t][t / 32] >> (t % 32) & 1)) atomicOr(z == 0.0f ? &ok[t / 32] : &bad[t / 32], 1u << (t % 32));
        span(Span<HD, KT, RW, KW, true>());
    } else {
        span(Span<HD, KT, RW, KW, false>());
    }

    const long all = (long)a.n_kv_head * A.rows;
    float *const po = A.part + ((long)part * all + (long)g * A.rows) * HD;
    float *const pm = A.part + (long)(A.n_draft + A.n_span) * all * HD + 2 * ((long)part * all + (long)g * A.rows);
    float *const om = reinterpret_cast<float *>(lds_bytes), *const ml = om + KW * L::ROWS * L::OS;
    if constexpr (KW > 1) __syncthreads();  // (the tiles are read no more)
    l += __shfl_xor(l, 32);
    const int lr = rw * 32 + ql;
    float *const to = KW == 1 ? po + (long)row * HD : om + (kw * L::ROWS + lr) * L::OS;
    if (KW > 1 || row < A.rows) {
        const float back = F32 ? pow2(-pv) : 1.0f;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                *reinterpret_cast<float4 *>(to + 32 * d + 8 * e + 4 * hh) =
                    make_float4(o[d][4 * e] * back, o[d][4 * e + 1] * back, o[d][4 * e + 2] * back, o[d][4 * e + 3] * back);
        if (hh == 0) *reinterpret_cast<float2 *>(KW == 1 ? pm + 2 * row : ml + 2 * (kw * L::ROWS + lr)) = make_float2(m, l);
    }
    if constexpr (KW > 1) {
        // the groups' (m, l, O) in group order
        constexpr int ROWS = L::ROWS, OS = L::OS;
        __syncthreads();
        for (int i = tid; i < ROWS * HD / 4; i += THREADS) {
            const int r = i / (HD / 4), c = 4 * (i - r * (HD / 4)), gr = block * ROWS + r;
            if (gr >= A.rows) continue;
            float M = -INFINITY, ls = 0.0f;
#pragma unroll
            for (int w = 0; w < KW; w++) M = fmaxf(M, ml[2 * (w * ROWS + r)]);
            const float mu = M == -INFINITY ? 0.0f : M;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < KW; w++) {
                const float x = __builtin_amdgcn_exp2f(ml[2 * (w * ROWS + r)] - mu);
                const float4 y = *reinterpret_cast<const float4 *>(om + (w * ROWS + r) * OS + c);
                ls += ml[2 * (w * ROWS + r) + 1] * x;
                sum.x += y.x * x, sum.y += y.y * x, sum.z += y.z * x, sum.w += y.w * x;
            }
            *reinterpret_cast<float4 *>(po + (long)gr * HD + c) = sum;
            if (c == 0) *reinterpret_cast<float2 *>(pm + 2 * gr) = make_float2(M, ls);
        }
    }
}

// The parts of one node and head in part order: 256 / (HD / 4) groups of lanes take parts in turn. Bound by reading them: 64
// nodes of 32 heads, 32 parts each, 34 MB (just written, so from the caches) 9.2 us, 3.7 TB/s; few nodes 3.4 us.
template <int HD>
__global__ __launch_bounds__(256) void k_tree_merge(TreeArgs A) {
    constexpr int LN = HD / 4, NG = 256 / LN;
    __shared__ float2 ml[MAX_PARTS];
    __shared__ float red[4];
    __shared__ float4 sums[NG][LN];
    __shared__ float ls[NG];
    const sdy_attn_tree_args &a = A.a;
    const int past = *a.n_past, tid = threadIdx.x;
    const int t = blockIdx.x, h = blockIdx.y;
    if (past < 0 || past > a.max_past || a.parent[t] < -1) return;
    // the drafted spans up to the node's own, and those of the cache
    const int nd = t / A.granule + 1, n = nd + spans_used(A, past), rep = a.n_head / a.n_kv_head, g = h / rep;
    auto at = [&](int p) { return (long)(p < nd ? p : p - nd + A.n_draft); };
    const long all = (long)a.n_kv_head * A.rows, row = (long)g * A.rows + (long)t * rep + (h - g * rep);
    const float2 *pm = reinterpret_cast<const float2 *>(A.part + (long)(A.n_draft + A.n_span) * all * HD) + row;
    float M = -INFINITY;
    for (int p = tid; p < n; p += 256) {
        ml[p] = pm[at(p) * all];
        M = fmaxf(M, ml[p].x);
    }
    for (int off = 32; off >= 1; off >>= 1) M = fmaxf(M, __shfl_xor(M, off));
    if ((tid & 63) == 0) red[tid >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const int grp = tid / LN, ln = tid - grp * LN;
    const float4 *po = reinterpret_cast<const float4 *>(A.part + row * HD) + ln;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float lsum = 0.0f;
#pragma unroll 4
    for (int p = grp; p < n; p += NG) {
        const float4 y = po[at(p) * all * LN];
        const float x = __builtin_amdgcn_exp2f(ml[p].x - M);
        lsum += ml[p].y * x;
        sum.x += y.x * x, sum.y += y.y * x, sum.z += y.z * x, sum.w += y.w * x;
    }
    sums[grp][ln] = sum;
    if (ln == 0) ls[grp] = lsum;
    __syncthreads();
    if (grp == 0) {
        lsum = 0.0f;
        sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < NG; i++) {
            const float4 y = sums[i][ln];
            lsum += ls[i];
            sum.x += y.x, sum.y += y.y, sum.z += y.z, sum.w += y.w;
        }
        reinterpret_cast<float4 *>(a.out + (size_t)t * a.out_stride + (size_t)h * HD)[ln] =
            make_float4(sum.x / lsum, sum.y / lsum, sum.z / lsum, sum.w / lsum);
    }
}

// How the work is split, from the sizes alone.
struct Plan {
    int rw, kw, rows, n_block, n_draft, n_span;
};
Plan plan_of(int n_tok, int n_head, int n_kv_head, int hd, int max_past, bool f16) {
    Plan p;
    p.rows = n_tok * (n_head / n_kv_head);
    // Eight waves as one group of 256 rows or as two of 128 that take tiles in turn. The one group brings a tile in half the
    // time, and needs no merge: it wins where a workgroup has few tiles, and with f32's longer products. The two have work
    // for waves that would have no rows, and products of one group beside the other work of the other. `work`: tiles of a
    // workgroup, in blocks of 128 rows. us, one group against two, 2 or 4 kv heads of 128 dims:
    //   f16   40 rows over 700 11.6 : 12.9, over 33001 22.8 : 20.8; 128 rows over 700 15.2 : 17.1, over 4099 20.8 : 21.2, over
    //         33001 38.3 : 35.9; 256 rows over 700 20.4 : 19.0, over 4099 29.7 : 24.7, over 33001 54.3 : 50.0
    //   f32   40 rows over 700 13.9 : 16.0, over 33001 29.4 : 31.9; 128 rows over 4099 23.9 : 26.3; 512 rows over 4099 37.4 :
    //         36.2, over 33001 116 : 128; 32 rows of 8 kv heads over 33001 62 : 57
    //   64 dims  32 rows of 8 kv heads over 33001 f32 42 : 30, f16 34 : 23; 488 rows over 700 16.3 : 15.3, 14.7 : 13.7
    const long work = ((long)max_past + KB - 1) / KB * n_kv_head * ((p.rows + 127) / 128) / 256;
    const bool two = f16 || hd == 64 ? p.rows > 192 || work >= 2 : p.rows <= 64 && work >= 24;
    p.rw = hd == 256 || two ? 4 : 8;
    p.kw = hd == 256 ? 1 : 8 / p.rw;
    const int block = 32 * p.rw;
    p.n_block = (p.rows + block - 1) / block;
    const int granule = KB * p.kw;
    p.n_draft = (n_tok + granule - 1) / granule;
    const long pairs = (long)n_kv_head * p.n_block, rounds = ((long)max_past + granule - 1) / granule;
    long n = (256 - pairs * p.n_draft) / pairs;
    if (n < 128 / pairs) n = 128 / pairs;
    if (n > rounds) n = rounds;
    if (n > 512) n = 512;
    // a span's bytes (at most 2^31 - 1 for a buffer resource)
    const long least = (rounds * granule * hd * 4 + (1l << 30) - 1) >> 30;
    if (n < least) n = least;
    p.n_span = (int)(n < 1 ? 1 : n);
    return p;
}

template <int HD, class KT, int RW, int KW>
int launch_part(const TreeArgs &A, hipStream_t st) {
    static size_t granted = 0;
    const void *fn = (const void *)k_tree_part<HD, KT, RW, KW>;
    const int rc = sdy_lds_limit(fn, Lds<HD, KT, RW, KW>::bytes, &granted);
    if (rc) return rc;
    SDY_NOTE_KERNEL((k_tree_part<HD, KT, RW, KW>));
    const long pairs = (long)(A.n_draft + A.n_span) * A.a.n_kv_head;
    hipLaunchKernelGGL((k_tree_part<HD, KT, RW, KW>), dim3((unsigned)((pairs + 7) / 8 * 8 * A.n_block)), dim3(64 * RW * KW),
                       (Lds<HD, KT, RW, KW>::bytes), st, A);
    return sdy_check_launch("attn_tree");
}

template <int HD, class KT>
int launch_rows(const TreeArgs &A, const Plan &p, hipStream_t st) {
    if constexpr (HD == 256) return launch_part<HD, KT, 4, 1>(A, st);
    else return p.rw == 8 ? launch_part<HD, KT, 8, 1>(A, st) : launch_part<HD, KT, 4, 2>(A, st);
}

template <int HD>
int launch_tree(const TreeArgs &A, const Plan &p, hipStream_t st) {
    const int rc = A.a.kv_type == SDY_KV_F16 ? launch_rows<HD, uint16_t>(A, p, st) : launch_rows<HD, float>(A, p, st);
    if (rc) return rc;
    hipLaunchKernelGGL(k_tree_merge<HD>, dim3(A.a.n_tok, A.a.n_head), dim3(256), 0, st, A);
    return sdy_check_launch("attn_tree merge");
}

}  // namespace

extern "C" int sdy_attn_tree_ok(int n_tok, int n_head, int n_kv_head, int hd) {
    return n_tok >= 1 && n_tok <= MAX_NODES && n_head >= 1 && n_head <= 65535 && n_kv_head >= 1 && n_head % n_kv_head == 0 &&
           (hd == 64 || hd == 128 || hd == 256);
}

extern "C" size_t sdy_attn_tree_floats(int n_tok, int n_head, int n_kv_head, int hd, int max_past) {
    if (!sdy_attn_tree_ok(n_tok, n_head, n_kv_head, hd) || max_past < 0 || max_past > MAX_PAST) return 0;
    size_t most = 0;  // of the two types
    for (int f16 = 0; f16 < 2; f16++) {
        const Plan p = plan_of(n_tok, n_head, n_kv_head, hd, max_past, f16);
        const size_t n = (size_t)(p.n_draft + p.n_span) * n_kv_head * p.rows * (hd + 2);
        most = n > most ? n : most;
    }
    return most;
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
    if (a->max_past < 0 || a->max_past > MAX_PAST || (a->max_past > 0 && (!a->k_cache || !a->v_cache)))
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
    const Plan p = plan_of(a->n_tok, a->n_head, a->n_kv_head, a->hd, a->max_past, elt == 2);
    TreeArgs A;
    A.a = *a;
    A.rows = p.rows;
    A.n_block = p.n_block;
    A.n_span = p.n_span;
    A.granule = KB * p.kw;
    A.n_draft = p.n_draft;
    A.least = p.kw == 1 ? 2 : 1;
    A.log_scale = (float)(1.4426950408889634074 / sqrt((double)a->hd));
    A.part = a->part;
    hipStream_t st = (hipStream_t)s;
    return a->hd == 64 ? launch_tree<64>(A, p, st) : a->hd == 128 ? launch_tree<128>(A, p, st) : launch_tree<256>(A, p, st);
}
