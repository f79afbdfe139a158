// Decode attention of B hypotheses that share a prompt: o[b, h] = sum_t w v / sum_t w, w = exp(scale q . k - max), over
// the prompt's cache (the prefix, one for all) and the hypothesis's own slots (the suffix). A slot of the suffix is
// looked up through a table once a beam search has reordered the hypotheses, so no cache is ever copied.
//
// Both products run on the matrix cores (v_mfma_f32_16x16x32): S^T = K Q^T has a query row per lane column and four
// consecutive slots per lane, which is how the next product, O^T = V^T P^T, wants P if its k index runs over the slots in
// the order 4 quad + (0..3), 16 + 4 quad + (0..3): the weights stay in their lanes. The softmax is in log2 units with a
// running maximum that moves only when a score exceeds it by more than 2^kSlack, so the exchange between the quads and
// the rescaling of O run in few steps. Scores, statistics and sums are fp32. int8 caches run on fp16 operands, in which the
// codes are exact; K's scale goes to the scores, V's scale to P.
//
// P's rounding. Plain caches: to their type, fp16 2^-11 relative, or 2^-32 of the largest weight where that is more, bf16 2^-8;
// the sum is of the rounded weights, so what they have in common cancels, and the result is 1.0 to 1.3 times as far off as by
// its own rounding to the type. In two 16-bit parts, with a product of V for each, it would be 1.0 times, for 82 us instead
// of 73 (32 hypotheses x 65536 slots, 8 KV heads): not taken. int8: the scales are in P, nothing cancels, and a result in fp16
// was up to 1.6 times as far off. There P has two parts of fp16, 22 bits: 1.0 times, for 97.8 us instead of 86.5 (128 rows x
// 65536 slots and 8 heads), 74.5 instead of 67.0 (64 rows), 19.4 instead of 19.1 (5 hypotheses x 30001). With bf16
// activations one part of fp16 does: 1.0 times.
//
// Launches: direct_kernel alone for small caches; else part_kernel for the suffixes and short prefixes, wide_kernel for
// long prefixes of many query rows and join_kernel, which adds the splits up. All read the lengths on the device; a
// kernel that has nothing to do for them returns at once.
#include <algorithm>

#include "kv8.h"

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kStep = 32;        // slots a wave takes at a time: the k index of one MFMA of P V
constexpr int kBlockStep = kStep * kWaves;
constexpr int kTileRows = 16;    // query rows of one MFMA tile
constexpr int kTileSlots = 2 * kStep;  // slots of one LDS tile of the wide kernel
constexpr int kMaxSplits = 128;
constexpr int kBlocks = 512;     // blocks of part_kernel that the card holds at a time: two per CU

typedef __bf16 b8_t __attribute__((ext_vector_type(8)));

struct AttnArgs {
    const uint16_t* q;
    uint16_t* o;
    const void *kc, *vc, *ks, *vs;
    const float *kcs, *vcs, *kss, *vss;
    const int64_t *plen, *spos;
    const int32_t* src;
    float* po;   // [B * NH][nsp + nss][128]
    float2* ml;  // [B * NH][nsp + nss]: running maximum (log2), sum
    float scale;
    int B, NH, NKV, S, T, rows, nspos, src_ld, nsp, nss;
    int nsp_narrow, nsp_wide;  // splits of a short and of a long prefix (wide 0: the narrow kernel takes them all)
    int groups, groups_wide;   // row groups of 16, and of a wide block's rows
    int prefix_blocks;
    int wide_min;  // prefix slots from which the wide kernel takes it, where nsp_wide
};

RK_DEV int prefix_len(const AttnArgs& a) {
    return a.kc ? (int)max<int64_t>(min<int64_t>(a.plen[0], a.S), 0) : 0;
}
RK_DEV int suffix_len(const AttnArgs& a, int b) {
    if (!a.ks) return 0;
    const int64_t t = a.spos[a.nspos > 1 ? b : 0];
    return t < 0 ? 0 : (int)min<int64_t>(t, a.T - 1) + 1;
}
RK_DEV bool is_wide(const AttnArgs& a, int n) { return a.nsp_wide > 0 && n >= a.wide_min; }
// Splits that take part of n slots, kBlockStep (narrow) or kTileSlots (wide) at a time in turn: neighbouring blocks read
// neighbouring slots at any time.
RK_DEV int active(int n, int splits, int quantum) { return min(splits, (int)(((long long)n + quantum - 1) / quantum)); }
RK_DEV int prefix_splits(const AttnArgs& a, int n) {
    return is_wide(a, n) ? active(n, a.nsp_wide, kTileSlots) : active(n, a.nsp_narrow, kBlockStep);
}
RK_DEV int suffix_splits(const AttnArgs& a, int n) { return active(n, a.nss, kBlockStep); }

template <bool BF16>
RK_DEV f4_t mfma(u4_t x, u4_t y, f4_t c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, x), __builtin_bit_cast(b8_t, y), c, 0, 0,
                                                       0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, x), __builtin_bit_cast(h8_t, y), c, 0, 0,
                                                      0);
}

// two fp32 as two rounded 16-bit values in a word
template <bool BF16>
RK_DEV uint32_t pack2(float x, float y) {
    if constexpr (BF16) {
        typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, b2_t{(__bf16)x, (__bf16)y});
    } else {
        return as_u32(h2_t{(_Float16)x, (_Float16)y});
    }
}

// Two int8 codes, in bytes 0 and 2 of w (the others 0), as fp16: 0x6400 + (code + 128) is 1024 + 128 + code exactly.
RK_DEV uint32_t codes2_to_h2(uint32_t w) {
    return as_u32(as_h2(w ^ 0x64806480u) - h2_t{(_Float16)1152.0f, (_Float16)1152.0f});
}
// four codes in a word as two words of fp16
RK_DEV u2_t codes4_to_h4(uint32_t w) {
    return u2_t{codes2_to_h2(perm(0u, w, 0x0c010c00u)), codes2_to_h2(perm(0u, w, 0x0c030c02u))};
}

// The weights of 8 slots as they meet V; TWO (int8 with fp16 activations): hi + lo. (An infinite V, which codes do not have,
// would meet a lo of 0.)
template <bool TWO>
struct Weights {
    u4_t hi;
};
template <>
struct Weights<true> {
    u4_t hi, lo;
};

// A wave's state for RT tiles of 16 query rows; lane (col, quad) = (lane & 15, lane >> 4): query row col of each tile.
template <int RT>
struct State {
    u4_t q[RT][4];       // B operand of K Q: the row's dims in K's order
    float qs[RT];        // |scale| * log2(e) (int8 with bf16: times what the fp16 copy of q was divided by)
    float m[RT];         // running maximum in log2 units, kLift below (at most kLift + kSlack below the true one)
    f4_t l[RT];          // sum of weights in l[.][0]; int8: of the quad's weights
    f4_t acc[RT][8];     // sum of weights * V, dim 8 (4 quad + e) + d in acc[.][d][e]
    float cap;           // int8: a power of two that no V scale so far exceeds; acc is in units of cap / 2^kHead
};
constexpr float kSlack = 8.0f;
constexpr int kHead = 7;
// What the maximum's weight is lifted by: a plain fp16 cache's weights meet V in fp16, which has no more than 2^-25 below
// 1. Lifted, they reach from 2^(kSlack + 7) = 2^15 down to 2^-32 of the maximum's weight. int8 has kHead for that.
template <bool BF16, bool Q8>
constexpr float kLift = BF16 || Q8 ? 0.0f : 7.0f;
constexpr float kLowest = -3.402823466e38f;  // "no maximum yet": exp2(-inf - kLowest) is 0, not NaN

// The state before the first slot. qrow: this lane's query row of tile r, its 128 values. CODES: K's order of dims is 64
// (c / 2) + 16 quad + 8 (c & 1) (16 codes to a load), else 32 c + 8 quad, for operand c. The scale's sign goes to q, so
// that the largest product is the largest score.
template <bool BF16, bool Q8, bool CODES = Q8, int RT, class QRow>
RK_DEV void start(State<RT>& s, float scale, QRow qrow) {
    const int quad = (threadIdx.x & 63) >> 4;
    const float c = fabsf(scale) * 1.4426950408889634f;
    const uint32_t sign = scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const uint16_t* q = qrow(r);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            s.q[r][i] = *reinterpret_cast<const u4_t*>(q + (CODES ? 64 * (i >> 1) + 16 * quad + 8 * (i & 1)
                                                                  : 32 * i + 8 * quad));
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s.q[r][i] ^= sign;
        s.qs[r] = c;
        if constexpr (BF16 && Q8) {
            // fp16 copies of the row over a power of two that brings its largest value to [2^10, 2^11): what falls
            // below fp16's subnormals is less than 2^-34 of that
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    top = max(top, max(s.q[r][i][e] & 0x7fffu, (s.q[r][i][e] >> 16) & 0x7fffu));
            top = max(top, xor_lanes<16>(top));
            top = max(top, xor_lanes<32>(top));
            const int e = max((int)(top >> 7), 30);
            const float f = __builtin_bit_cast(float, (uint32_t)(264 - e) << 23);
            s.qs[r] = c * __builtin_bit_cast(float, (uint32_t)(e - 10) << 23);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[8];
                widen8<true>(s.q[r][i], v);
#pragma unroll
                for (int x = 0; x < 4; ++x) s.q[r][i][x] = pack2<false>(v[2 * x] * f, v[2 * x + 1] * f);
            }
        }
        s.m[r] = kLowest;
        s.l[r] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < 8; ++d) s.acc[r][d] = f4_t{0.f, 0.f, 0.f, 0.f};
    }
    s.cap = 0x1p-117f;
}

// int8: V's scales vw (0 for what is no slot) become what P is multiplied by, scale * 2^kHead / cap: P stays within fp16,
// and precise for scales down to 2^-21 of the largest.
template <int RT>
RK_DEV void scale_weights(float (&vw)[8], State<RT>& s) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(vw[i]));
    if (__ballot(top > s.cap)) {  // rare after the first step: a larger scale than any before
        top = max_xor<32>(max_xor<16>(top));  // the lanes of a quad hold the same slots
        // the power of two above it, kept where its reciprocal is a normal number too
        const uint32_t e = min((__builtin_bit_cast(uint32_t, top) >> 23) + 1u, 252u);
        const float cap = __builtin_bit_cast(float, max(e, 10u) << 23);
        const float f = s.cap / cap;  // both powers of two
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int d = 0; d < 8; ++d) s.acc[r][d] *= f;
        s.cap = cap;
    }
    const float inv = (float)(1 << kHead) / s.cap;
#pragma unroll
    for (int i = 0; i < 8; ++i) vw[i] *= inv;
}

// The weights of tile r's query rows for the quad's eight slots, from their dot products; the running maximum, the sum
// and, when the maximum moves, acc follow. A score is the rounded product fl(t qs) in the maximum and in the exponent
// alike; fused into the subtraction, the highest score's exponent would be its product's rounding error, half a step of the
// maximum (32 at 2^29), and no longer 0. ok: bit i set where slot i is one. The sum is of the rounded weights, those
// that meet V, by one more product with ones (the VALU is the busier unit); int8's weights meet V with its scales in them,
// there it is of the fp32 ones.
template <bool BF16, bool Q8, bool TWO, bool MASK, int RT>
RK_DEV Weights<TWO> weights(const f4_t (&sc)[2], const float (&ks)[8], const float (&vw)[8], uint32_t ok, State<RT>& s, int r) {
#pragma clang fp contract(off)
    float t[8];
    float top = kLowest;  // as it is, no product of it: a lane without a slot is below any score
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        t[i] = sc[i >> 2][i & 3];
        if constexpr (Q8) t[i] *= ks[i];
        t[i] *= s.qs[r];
        if constexpr (MASK) t[i] = ok >> i & 1 ? t[i] : -INFINITY;
        top = fmaxf(top, t[i]);
    }
    constexpr float lift = kLift<BF16, Q8>;
    // some row's maximum moved by more than 2^kSlack (their difference: s.m + kSlack may round up to the next score)
    if (__ballot(top - s.m[r] > kSlack + lift)) {
        top = max_xor<32>(max_xor<16>(top));
        const float mn = fmaxf(s.m[r], top - lift), f = __builtin_amdgcn_exp2f(s.m[r] - mn);
        s.m[r] = mn;
        s.l[r] *= f;
#pragma unroll
        for (int d = 0; d < 8; ++d) s.acc[r][d] *= f;
    }
    // A bound for the compiler: without it the work of several tiles is interleaved, and blocks of 128 rows spill 120 bytes (128
    // fp16 rows x 65536 slots, 8 heads: 101 us instead of 98).
    if constexpr (Q8) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = __builtin_amdgcn_exp2f(t[i] - s.m[r]);
    Weights<TWO> w;
    if constexpr (Q8) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += t[i];
        s.l[r][0] += sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = t[2 * i] * vw[2 * i], y = t[2 * i + 1] * vw[2 * i + 1];
            w.hi[i] = pack2<false>(x, y);
            if constexpr (TWO)
                w.lo[i] = pack2<false>(__builtin_fmaf((float)as_h2(w.hi[i]).x, -1.0f, x),
                                       __builtin_fmaf((float)as_h2(w.hi[i]).y, -1.0f, y));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) w.hi[i] = pack2<BF16>(t[2 * i], t[2 * i + 1]);
        const uint32_t one = BF16 ? 0x3f803f80u : 0x3c003c00u;
        s.l[r] = mfma<BF16>(u4_t{one, one, one, one}, w.hi, s.l[r]);
    }
    return w;
}

// the sum of weights of tile r's row col, in every lane
template <bool Q8, int RT>
RK_DEV float total(const State<RT>& s, int r) {
    return Q8 ? sum_xor<32>(sum_xor<16>(s.l[r][0])) : s.l[r][0];
}

// ======================================================================= the suffixes, and prefixes that are not wide
// Where a wave's slots lie: K / V rows of 128 values, the scales of an int8 cache beside them.
struct Slots {
    const void *k, *v;
    const float *ks, *vs;
    size_t row0;         // row of slot 0 (prefix; suffix without a table)
    const int32_t* src;  // the hypothesis's table, or NULL
    int rows;            // its entries are below this
    size_t row_stride;   // rows from one table entry to the next
};

// One step's K and V as they come from memory or LDS:
//   k[j]  slot 16 j + col of the step; plain: dims 32 c + 8 quad .. + 7 in k[j][c]; int8: dims 64 c + 16 quad .. + 15
//   v[i]  slot 16 (i / 4) + 4 quad + i % 4, dims 8 col .. + 7: whole rows are read together
template <bool Q8>
struct Step {
    u4_t k[2][Q8 ? 2 : 4];
    u4_t v[8];
    float ks[8], vs[8];  // int8: the scales of v's slots
    uint32_t ok;         // bit i: v[i] is a slot
};

template <bool Q8, bool SUFFIX>
RK_DEV void load_step(const Slots& at, int s0, int end, Step<Q8>& st) {
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int last = end - 1 - s0;  // slots past the end read the last one
    constexpr int kRow = kHeadDim * (Q8 ? 1 : 2), kV = Q8 ? 8 : 16;  // bytes of a row, of a lane's piece of a V row
    st.ok = 0;
    if constexpr (SUFFIX) {
        size_t krow[2], vrow[8];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int t = s0 + min(16 * j + col, last);
            int w = at.src ? at.src[t] : 0;
            w = w >= 0 && w < at.rows ? w : 0;
            krow[j] = at.row0 + w * at.row_stride + t;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int off = 16 * (i / 4) + 4 * quad + i % 4, t = s0 + min(off, last);
            int w = at.src ? at.src[t] : 0;
            const bool in = w >= 0 && w < at.rows;
            w = in ? w : 0;
            vrow[i] = at.row0 + w * at.row_stride + t;
            st.ok |= (in && off <= last ? 1u : 0u) << i;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < (Q8 ? 2 : 4); ++c)
                st.k[j][c] = *reinterpret_cast<const u4_t*>((const char*)at.k + krow[j] * kRow + 64 * c + 16 * quad);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const char* v = (const char*)at.v + vrow[i] * kRow + kV * col;
            if constexpr (Q8) {
                const u2_t c = *reinterpret_cast<const u2_t*>(v);
                st.v[i][0] = c[0];
                st.v[i][1] = c[1];
                st.ks[i] = at.ks[vrow[i]];
                st.vs[i] = at.vs[vrow[i]];
            } else {
                st.v[i] = *reinterpret_cast<const u4_t*>(v);
            }
        }
    } else {
        // a wave-uniform base and small lane offsets
        const char* kb = (const char*)at.k + (at.row0 + s0) * kRow;
        const char* vb = (const char*)at.v + (at.row0 + s0) * kRow;
        const uint32_t kl = 16 * quad, vl = kV * col;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t r = min(16 * j + col, last);
#pragma unroll
            for (int c = 0; c < (Q8 ? 2 : 4); ++c)
                st.k[j][c] = *reinterpret_cast<const u4_t*>(kb + (r * kRow + kl) + 64 * c);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int off = 16 * (i / 4) + 4 * quad + i % 4;
            const uint32_t r = min(off, last);
            st.ok |= (off <= last ? 1u : 0u) << i;
            if constexpr (Q8) {
                const u2_t c = *reinterpret_cast<const u2_t*>(vb + (r * kRow + vl));
                st.v[i][0] = c[0];
                st.v[i][1] = c[1];
                st.ks[i] = at.ks[at.row0 + s0 + r];
                st.vs[i] = at.vs[at.row0 + s0 + r];
            } else {
                st.v[i] = *reinterpret_cast<const u4_t*>(vb + (r * kRow + vl));
            }
        }
    }
}

// The dot products of RT tiles of query rows with a step's K: slot 16 j + 4 quad + e of row col in sc[.][j][e].
template <bool BF16, bool Q8, int RT>
RK_DEV void products(const Step<Q8>& st, const State<RT>& s, f4_t (&sc)[RT][2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int r = 0; r < RT; ++r) sc[r][j] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            u4_t k;
            if constexpr (Q8) {
                const u2_t lo = codes4_to_h4(st.k[j][c >> 1][2 * (c & 1)]),
                           hi = codes4_to_h4(st.k[j][c >> 1][2 * (c & 1) + 1]);
                k = u4_t{lo[0], lo[1], hi[0], hi[1]};
            } else {
                k = st.k[j][c];
            }
#pragma unroll
            for (int r = 0; r < RT; ++r) sc[r][j] = mfma<BF16 && !Q8>(k, s.q[r][c], sc[r][j]);
        }
    }
}

// Their softmax: the weights w of each tile.
template <bool BF16, bool Q8, bool MASK, class Loaded, bool TWO, int RT>
RK_DEV void softmax(const Loaded& st, const f4_t (&sc)[RT][2], State<RT>& s, Weights<TWO> (&w)[RT]) {
    float vw[8];
    if constexpr (Q8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) vw[i] = !MASK || (st.ok >> i & 1) ? st.vs[i] : 0.f;
        scale_weights(vw, s);
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) w[r] = weights<BF16 && !Q8, Q8, TWO, MASK>(sc[r], st.ks, vw, st.ok, s, r);
}

// The weights' products with the step's V, transposed to the A operand (row = dim, k = slot): dim 8 col + d of the
// eight slots at a time.
template <bool BF16, bool Q8, bool MASK, bool TWO, int RT>
RK_DEV void add_values(const Step<Q8>& st, const Weights<TWO> (&w)[RT], State<RT>& s) {
#pragma unroll
    for (int d = 0; d < 8; ++d) {
        u4_t vt;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            if constexpr (Q8) {
                const uint32_t b = d & 3;
                vt[p] = codes2_to_h2(perm(st.v[2 * p + 1][d >> 2], st.v[2 * p][d >> 2],
                                          0x0c000c00u | ((4 + b) << 16) | b));
            } else {
                uint32_t lo = st.v[2 * p][d >> 1], hi = st.v[2 * p + 1][d >> 1];
                if constexpr (MASK) {  // 0 times whatever lies there may be NaN
                    lo = st.ok & (1u << (2 * p)) ? lo : 0u;
                    hi = st.ok & (2u << (2 * p)) ? hi : 0u;
                }
                vt[p] = perm(hi, lo, d & 1 ? 0x07060302u : 0x05040100u);
            }
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            if constexpr (TWO) s.acc[r][d] = mfma<BF16 && !Q8>(vt, w[r].lo, s.acc[r][d]);
            s.acc[r][d] = mfma<BF16 && !Q8>(vt, w[r].hi, s.acc[r][d]);
        }
    }
}

template <bool BF16, bool Q8, bool MASK>
RK_DEV void take(const Step<Q8>& st, State<1>& s) {
    f4_t sc[1][2];
    Weights<!BF16 && Q8> w[1];
    products<BF16>(st, s, sc);
    softmax<BF16, Q8, MASK>(st, sc, s, w);
    add_values<BF16, Q8, MASK>(st, w, s);
}

// A wave's steps: slots first + i stride .. + kStep - 1, below end.
template <bool BF16, bool Q8, bool SUFFIX>
RK_DEV void take_steps(const Slots& at, int first, int stride, int end, State<1>& s) {
    if (first >= end) return;
    // two steps' registers in turn; only a wave's last step can be a partial one
    Step<Q8> x, y;
    const int n = (end - 1 - first) / stride + 1;
    load_step<Q8, SUFFIX>(at, first, end, x);
    int i = 0;
    for (; i + 2 < n; i += 2) {
        load_step<Q8, SUFFIX>(at, first + (i + 1) * stride, end, y);
        __builtin_amdgcn_sched_barrier(0);
        take<BF16, Q8, SUFFIX>(x, s);
        load_step<Q8, SUFFIX>(at, first + (i + 2) * stride, end, x);
        __builtin_amdgcn_sched_barrier(0);
        take<BF16, Q8, SUFFIX>(y, s);
    }
    if (i + 1 < n) {
        load_step<Q8, SUFFIX>(at, first + (i + 1) * stride, end, y);
        __builtin_amdgcn_sched_barrier(0);
        take<BF16, Q8, SUFFIX>(x, s);
        x = y;
    }
    take<BF16, Q8, true>(x, s);
}

// Where a block's W waves meet.
template <int W>
struct Meet {
    f4_t acc[W][8][64];
    float m[W][kTileRows], l[W][kTileRows], cap[W];
};
template <bool Q8, int W>
RK_DEV void hand_over(const State<1>& s, Meet<W>& meet, int wave) {
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const float l = total<Q8>(s, 0);
    if (quad == 0) {
        meet.m[wave][col] = s.m[0];
        meet.l[wave][col] = l;
    }
    if (lane == 0) meet.cap[wave] = Q8 ? s.cap * (1.0f / (1 << kHead)) : 1.0f;
#pragma unroll
    for (int d = 0; d < 8; ++d) meet.acc[wave][d][lane] = s.acc[0][d];
}
// The sum of the waves for dims 32 quad + 8 e .. + 7 of row i: acc[d][lane][e] is dim 8 (4 quad + e) + d.
template <int W>
RK_DEV void meet_all(const Meet<W>& meet, int i, int quad, int e, float& M, float& L, float (&o)[8]) {
    M = kLowest;
    L = 0.f;
#pragma unroll
    for (int d = 0; d < 8; ++d) o[d] = 0.f;
#pragma unroll
    for (int g = 0; g < W; ++g) M = fmaxf(M, meet.m[g][i]);
#pragma unroll
    for (int g = 0; g < W; ++g) {
        const float f = __builtin_amdgcn_exp2f(meet.m[g][i] - M), fc = f * meet.cap[g];
        L += f * meet.l[g][i];
#pragma unroll
        for (int d = 0; d < 8; ++d) o[d] += fc * meet.acc[g][d][16 * quad + i][e];
    }
}

// Slots begin + (0 .. kBlockStep - 1) + i stride below end of `at` for up to 16 query rows, a step for each wave. qrow(i):
// the query row i, as a row of q; out(i): its place in the workspace.
template <bool BF16, bool Q8, bool SUFFIX, class QRow, class Out>
RK_DEV void strip(const AttnArgs& a, const Slots& at, int begin, int stride, int end, int nrows, Meet<kWaves>& meet,
                  QRow qrow, Out out) {
    const int lane = threadIdx.x & 63, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    State<1> s;
    start<BF16, Q8>(s, a.scale, [&](int) { return a.q + qrow(min(col, nrows - 1)) * kHeadDim; });
    take_steps<BF16, Q8, SUFFIX>(at, begin + wave * kStep, stride, end, s);
    hand_over<Q8>(s, meet, wave);
    __syncthreads();
    const int i = lane >> 2, e = lane & 3;
    if (i >= nrows) return;
    float M, L, o[8];
    meet_all(meet, i, wave, e, M, L, o);
    const size_t p = out(i);
    f4_t* dst = reinterpret_cast<f4_t*>(a.po + p * kHeadDim + 32 * wave + 8 * e);
    dst[0] = f4_t{o[0], o[1], o[2], o[3]};
    dst[1] = f4_t{o[4], o[5], o[6], o[7]};
    if (wave == 0 && e == 0) a.ml[p] = float2{M, L};
}

// the suffix of hypothesis b, KV head g
RK_DEV Slots suffix_slots(const AttnArgs& a, int b, int g) {
    const size_t per = (size_t)a.NKV * a.T;
    return {a.ks, a.vs, a.kss, a.vss, (a.src ? 0 : b * per) + (size_t)g * a.T,
            a.src ? a.src + (size_t)b * a.src_ld : nullptr, a.rows, a.src ? per : 0};
}

// Small caches, in one launch and without a workspace: a block takes all slots of one hypothesis and KV head, its eight
// waves shared out between prefix and suffix by their lengths, and writes the result. A step costs a wave about 2 us of
// memory latency, and a CU holds one such block. So it pays for one step per wave and two blocks per CU; for half as many to
// as many blocks as CUs, where part_kernel has few blocks to a hypothesis, for three, at 128 of them about even. In a graph,
// part_kernel and join_kernel / this, 4 query heads per KV head, plain, then both caches int8:
//   one step   4 hypotheses and 4 KV heads x (34 + 9) slots 7.3 / 5.7 us, 8.3 / 6.9; with 8 KV heads 32 x (100 + 20) 11.0 /
//              6.2, 11.8 / 7.2; 64 x (190 + 60) 16.7 / 12.6, 17.4 / 13.6; but 68 x (34 + 9) 15.2 / 13.4, 16.9 / 17.6, and
//              128 x (190 + 60) of one head 16.2 / 24.3, 18.1 / 27.7
//   three      with 8 KV heads 16 x (200 + 80) 8.9 / 7.9, 9.2 / 9.1, x (500 + 260) 11.9 / 12.1, 11.2 / 12.8, x (700 + 68)
//              11.5 / 12.5, 11.0 / 12.8, x (100 + 660) 15.4 / 12.2, 15.9 / 12.8; 18 x (500 + 260) 14.6 / 12.2, 14.7 / 12.8,
//              x (700 + 68) 12.6 / 12.5, 11.8 / 12.7, x (100 + 660) 13.3 / 12.3, 14.2 / 12.8; 32 x (500 + 260) 17.5 / 12.6,
//              17.5 / 13.3, x (100 + 660) 19.7 / 12.7, 20.2 / 13.4; 34 x (500 + 260) 20.5 / 22.9, 20.4 / 23.7. It loses where
//              part_kernel takes a long prefix in full groups of 16 rows: 32 x (700 + 68) of one head per KV head 10.2 / 13.7,
//              10.3 / 14.8
// An eager call saves a launch besides.
constexpr int kDirectWaves = 8;
constexpr int kDirectSlots = kDirectWaves * kStep;
RK_DEV int direct_waves(int n1, int n2) {  // the prefix's: its share of the steps n1 + n2, but one at least for either
    const int w = (kDirectWaves * n1 + (n1 + n2) / 2) / max(n1 + n2, 1);
    return n1 && n2 ? min(max(w, 1), kDirectWaves - 1) : w;
}
template <bool BF16, bool P8, bool S8>
__global__ __launch_bounds__(64 * kDirectWaves, 2) void direct_kernel(AttnArgs a) {
    __shared__ __align__(16) Meet<kDirectWaves> meet;
    const int REP = a.NH / a.NKV, b = blockIdx.x / a.NKV, g = blockIdx.x % a.NKV;
    const int lane = threadIdx.x & 63, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint16_t* q = a.q + ((size_t)b * a.NH + g * REP + min(col, REP - 1)) * kHeadDim;
    const int np = prefix_len(a), ns = suffix_len(a, b);
    const int wp = direct_waves((np + kStep - 1) / kStep, (ns + kStep - 1) / kStep);
    State<1> s;
    if (wave < wp) {
        const Slots at{a.kc, a.vc, a.kcs, a.vcs, (size_t)g * a.S, nullptr, 0, 0};
        start<BF16, P8>(s, a.scale, [&](int) { return q; });
        take_steps<BF16, P8, false>(at, wave * kStep, wp * kStep, np, s);
        hand_over<P8>(s, meet, wave);
    } else {
        start<BF16, S8>(s, a.scale, [&](int) { return q; });
        take_steps<BF16, S8, true>(suffix_slots(a, b, g), (wave - wp) * kStep, (kDirectWaves - wp) * kStep, ns, s);
        hand_over<S8>(s, meet, wave);
    }
    __syncthreads();
    const int i = lane >> 2, e = lane & 3;
    if (wave >= 4 || i >= REP) return;
    float M, L, o[8];
    meet_all(meet, i, wave, e, M, L, o);
#pragma unroll
    for (int d = 0; d < 8; ++d) o[d] = L == 0.f ? 0.f : o[d] / L;
    *reinterpret_cast<u4_t*>(a.o + ((size_t)b * a.NH + g * REP + i) * kHeadDim + 32 * wave + 8 * e) = narrow8<BF16>(o);
}

// Blocks [0, prefix_blocks): (split, KV head, group of 16 query rows) of the prefix, the groups of a split side by side
// (they read the same slots); then (hypothesis, KV head, split) of the suffixes, whose NH / NKV rows fill part of a tile.
template <bool BF16, bool P8, bool S8>
__global__ __launch_bounds__(kThreads, 2) void part_kernel(AttnArgs a) {
    __shared__ __align__(16) Meet<kWaves> meet;
    const int REP = a.NH / a.NKV, nsplit = a.nsp + a.nss;
    if ((int)blockIdx.x < a.prefix_blocks) {
        const int rg = blockIdx.x % a.groups, x = blockIdx.x / a.groups;
        const int g = x % a.NKV, split = x / a.NKV;
        const int n = prefix_len(a), splits = prefix_splits(a, n);
        if (is_wide(a, n) || split >= splits) return;
        const int row0 = rg * kTileRows, nrows = min(a.B * REP - row0, kTileRows);
        const Slots at{a.kc, a.vc, a.kcs, a.vcs, (size_t)g * a.S, nullptr, 0, 0};
        auto qrow = [&](int i) { return (size_t)((row0 + i) / REP) * a.NH + g * REP + (row0 + i) % REP; };
        strip<BF16, P8, false>(a, at, split * kBlockStep, splits * kBlockStep, n, nrows, meet, qrow,
                               [&](int i) { return qrow(i) * nsplit + split; });
    } else {
        const int x = blockIdx.x - a.prefix_blocks, split = x % a.nss, g = x / a.nss % a.NKV, b = x / a.nss / a.NKV;
        const int n = suffix_len(a, b), splits = suffix_splits(a, n);
        if (split >= splits) return;
        auto qrow = [&](int i) { return (size_t)b * a.NH + g * REP + i; };
        strip<BF16, S8, true>(a, suffix_slots(a, b, g), split * kBlockStep, splits * kBlockStep, n, REP, meet, qrow,
                              [&](int i) { return qrow(i) * nsplit + a.nsp + split; });
    }
}

// ============================================================================== long prefixes of more than 16 query rows
// A block takes 16 RT RW query rows of a KV head over one split of the prefix: RW waves with rows of their own for each
// half of the slots. Those come in tiles of 64 by global_load_lds into a ring of kRing (plain) or kRing8 (int8) LDS
// buffers, one block to a CU, more on their way than registers could hold; each tile is read from memory once for all
// the block's rows. 16-byte chunk c of a row of 256 bytes is stored at chunk c ^ (row & 15), so that the K operands (16
// rows, one chunk) touch every bank equally often. An int8 tile is stored as it comes and converted once for all the
// block's waves, by one half of them K, by the other V, into two pairs of tiles of fp16 that are laid out like plain ones
// (8 heads x 65536 slots, one product with V per weight, 128 rows: 85 us, 91 with each wave converting what it reads; 64
// rows 68 and 71).
constexpr int kRing = 4, kRing8 = 5;

template <bool Q8>
struct Tile {
    static constexpr int kRow = Q8 ? kHeadDim : 2 * kHeadDim;
    static constexpr int kPart = kTileSlots * kRow;             // bytes of K, and of V
    static constexpr int kScales = Q8 ? 2 * 4 * kTileSlots : 0; // K's, V's
    static constexpr int kBytes = 2 * kPart + kScales;
    static constexpr int kCount = Q8 ? kRing8 : kRing;
    static constexpr int kPlain = 2 * kHeadDim * kTileSlots;    // bytes of a plain K or V tile
    static constexpr int kLds = kCount * kBytes + (Q8 ? 4 * kPlain : 0);
};

// Waits and barriers of the ring. To the compiler the builtins are no memory operations: the fences (no instruction) keep
// LDS reads and copies on their side of them.
RK_DEV void fence() { asm volatile("" ::: "memory"); }
template <int N>
RK_DEV void wait_copies() {  // s_waitcnt vmcnt(N) alone (bits [3:0] and [15:14]; expcnt and lgkmcnt at their maxima)
    fence();
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
    fence();
}
RK_DEV void wait_lds() {  // lgkmcnt(0) alone
    fence();
    __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4) | (0 << 8));
    fence();
}
RK_DEV void barrier() {
    fence();
    __builtin_amdgcn_s_barrier();
    fence();
}

template <bool BF16, bool Q8, int RT, int RW>
__global__ __launch_bounds__(128 * RW, RW > 2 ? 2 : 1) void wide_kernel(AttnArgs a) {
    using TL = Tile<Q8>;
    constexpr int kW = 2 * RW, kRows = kTileRows * RT * RW;
    constexpr int kCopies = 2 * TL::kPart / 1024 / kW;  // 1 KiB copies of a wave per tile
    constexpr int kPerTile = kCopies + (Q8 ? 1 : 0);
    extern __shared__ __align__(16) char ring[];
    __shared__ float s_m[RW][RT][kTileRows], s_l[RW][RT][kTileRows], s_cap[2][RW];
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rw = wave % RW, half = wave / RW;
    // blocks are dealt to the eight XCDs in turn: the row groups of a split, eight apart, share an L2
    const int rest = blockIdx.x >> 3, rg = rest % a.groups_wide, item = (rest / a.groups_wide) * 8 + (blockIdx.x & 7);
    const int g = item % a.NKV, split = item / a.NKV;
    const int REP = a.NH / a.NKV, nsplit = a.nsp + a.nss;
    const int row0 = rg * kRows, nrows = min(a.B * REP - row0, kRows);
    auto qrow = [&](int i) { return (size_t)((row0 + i) / REP) * a.NH + g * REP + (row0 + i) % REP; };
    // q first, beside the length, and all of it before the first copy: the wait for a load that is still pending at the
    // loop would be one for the copies, too
    State<RT> s;
    start<BF16, Q8, false>(s, a.scale, [&](int r) {
        return a.q + qrow(min((rw * RT + r) * kTileRows + col, nrows - 1)) * kHeadDim;
    });
    const int end = prefix_len(a), splits = prefix_splits(a, end), stride = splits * kTileSlots;
    if (!is_wide(a, end) || split >= splits) return;
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) asm volatile("" : "+v"(s.q[r][c]));
    const char* kb = (const char*)a.kc + (size_t)g * a.S * TL::kRow;
    const char* vb = (const char*)a.vc + (size_t)g * a.S * TL::kRow;
    // int8: even waves copy K's scales, odd ones V's (some of them the same ones, so that every wave's count is the same)
    const float* sb = Q8 ? (wave & 1 ? a.vcs : a.kcs) + (size_t)g * a.S : nullptr;

    // one tile's copies; slots past the end copy the last one
    auto issue = [&](int t0, int slot) {
        char* dst = ring + slot * TL::kBytes;
        const int base = min(t0, end - 1);
        const uint32_t last = end - 1 - base;
        auto source = [&](int j) {  // of the tile's copy j: K's first
            constexpr int kPer = TL::kPart / 1024, kChunks = TL::kRow / 16, kR = 64 / kChunks;
            const int jj = j < kPer ? j : j - kPer;
            const uint32_t r = kR * jj + lane / kChunks, c = (lane % kChunks) ^ (Q8 ? 0 : r & 15);
            const char* from = (j < kPer ? kb : vb) + (size_t)base * TL::kRow + (min(r, last) * TL::kRow + 16 * c);
            return reinterpret_cast<const uint4*>(from);
        };
        // (the operands as variables of their own types: dependent ones keep the host pass from making the launch stub)
        // nontemporal, unless another block reads the same slots (65536 slots and 8 heads, copies alone: 41 us against 44)
        if (a.groups_wide == 1) {
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const uint4* from = source(wave + kW * i);
                uint4* to = reinterpret_cast<uint4*>(dst + 1024 * (wave + kW * i));
                __builtin_amdgcn_global_load_lds(from, to, 16, 0, 2);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const uint4* from = source(wave + kW * i);
                uint4* to = reinterpret_cast<uint4*>(dst + 1024 * (wave + kW * i));
                __builtin_amdgcn_global_load_lds(from, to, 16, 0, 0);
            }
        }
        if constexpr (Q8)
            __builtin_amdgcn_global_load_lds(
                reinterpret_cast<const uint32_t*>(sb + base + min((uint32_t)lane, last)),
                reinterpret_cast<uint32_t*>(dst + 2 * TL::kPart + 4 * kTileSlots * (wave & 1)), 4, 0, 0);
    };

    const int begin = split * kTileSlots, tiles = (end - 1 - begin) / stride + 1;
#pragma unroll
    for (int i = 0; i < TL::kCount; ++i) issue(begin + i * stride, i);

    // lane offsets in a plain tile: K's operand c of slot col (^ 64 c), V's piece of the slots 4 quad + i
    constexpr int kRow = 2 * kHeadDim;
    const int krow = kStep * half + col, koff = krow * kRow + ((quad ^ (krow & 15)) << 4);
    int voff[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = kStep * half + 4 * quad + i;
        voff[i] = r * kRow + ((col ^ (r & 15)) << 4);
    }
    auto tile_at = [&](int i) { return ring + (uint32_t)i % TL::kCount * TL::kBytes; };
    char* conv = ring + TL::kCount * TL::kBytes;
    auto k_at = [&](int i) -> const char* { return Q8 ? conv + (i & 1) * TL::kPlain : tile_at(i); };
    auto v_at = [&](int i) -> const char* { return Q8 ? conv + (2 + (i & 1)) * TL::kPlain : tile_at(i) + TL::kPart; };
    Step<false> st;
    auto read_k = [&](int i) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                st.k[j][c] = *reinterpret_cast<const u4_t*>(k_at(i) + (koff ^ (c << 6)) + 16 * j * kRow);
    };
    auto read_v = [&](int i) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            st.v[e] = *reinterpret_cast<const u4_t*>(v_at(i) + voff[e & 3] + 16 * (e >> 2) * kRow);
    };
    // int8: this half's part of tile i (half 0: K, half 1: V) as fp16; ends before the next barrier
    auto convert = [&](int i) {
        if constexpr (Q8) {
            static_assert(kW == 8, "256 threads, two pieces of 16 codes each");
            const char* from = tile_at(i) + half * TL::kPart;
            char* to = conv + (2 * half + (i & 1)) * TL::kPlain;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int p = (threadIdx.x & 255) + 256 * e, r = p >> 3, c = 2 * (p & 7);
                const u4_t w = *reinterpret_cast<const u4_t*>(from + 16 * p);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const u2_t lo = codes4_to_h4(w[2 * x]), hi = codes4_to_h4(w[2 * x + 1]);
                    u4_t* dst = reinterpret_cast<u4_t*>(to + r * kRow + (((c + x) ^ (r & 15)) << 4));
                    *dst = u4_t{lo[0], lo[1], hi[0], hi[1]};
                }
            }
        }
    };
    auto converted = [&] {
        if constexpr (Q8) wait_lds();
    };
    // The two waves of a SIMD, one of each half, work in opposite phases: while one multiplies (the last tile's weights
    // with its V, then q with this tile's K) the other is in its softmax, so that the matrix cores and the VALU are both
    // busy (in step, both waves waited for the same unit: 41 us of arithmetic for 65536 slots and 8 heads, as long as the
    // copies take). Phase 2 i: half 0 multiplies for tile i, phase 2 i + 1: half 1 does. A barrier ends each phase; in
    // front of that of phase 2 i each wave's copies of tile i + 1 have landed, whose K is read from phase 2 i + 1 on. The
    // last reads of tile i (V's, by half 1) end in phase 2 i + 2; its buffer is filled again from phase 2 i + 3 on.
    // int8: K of tile i is converted in phase 2 i - 2, V in phase 2 i - 1; so the copies have to have landed a phase
    // earlier, in front of phase 2 i that of tile i + 1.
    constexpr bool kB = BF16 && !Q8;  // int8 runs on fp16 operands
    f4_t sc[RT][2];
    Weights<!BF16 && Q8> w[RT];
    auto refill = [&](int i) {  // in phase 2 i + 1
        if (i > 0) issue(begin + (i - 1 + TL::kCount) * stride, (uint32_t)(i - 1) % TL::kCount);
    };
    auto multiply = [&](int i) {
        convert(i + 1);
        read_v(i);
        products<kB>(st, s, sc);
        converted();
    };
    auto weigh = [&](int i, auto masked) {
        constexpr bool MASK = decltype(masked)::value;
        st.ok = 0xff;
        if constexpr (MASK) {
            st.ok = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                st.ok |= (begin + i * stride + kStep * half + 16 * (e >> 2) + 4 * quad + (e & 3) < end ? 1u : 0u) << e;
        }
        if constexpr (Q8) {
            const float* scales = reinterpret_cast<const float*>(tile_at(i) + 2 * TL::kPart) + kStep * half + 4 * quad;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const f4_t x = *reinterpret_cast<const f4_t*>(scales + 16 * j);
                const f4_t y = *reinterpret_cast<const f4_t*>(scales + kTileSlots + 16 * j);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    st.ks[4 * j + e] = x[e];
                    st.vs[4 * j + e] = y[e];
                }
            }
        }
        if constexpr (!Q8) read_k(i + 1);
        softmax<BF16, Q8, MASK>(st, sc, s, w);
        wait_lds();  // V's and K's reads have ended before the barrier
    };
    auto landed = [&] { wait_copies<(TL::kCount - 3) * kPerTile>(); };
    auto phase = [&] {
        if constexpr (Q8) __builtin_amdgcn_sched_barrier(0);
        barrier();
    };
    wait_copies<(TL::kCount - (Q8 ? 2 : 1)) * kPerTile>();
    phase();
    if constexpr (Q8) {
        convert(0);
        converted();
        phase();
    }
    read_k(0);
    if (half == 0) {
        multiply(0);
        if constexpr (!Q8) landed();
        phase();
        for (int i = 0; i + 1 < tiles; ++i) {
            refill(i);
            weigh(i, std::false_type());
            if constexpr (Q8) landed();
            phase();
            if constexpr (Q8) read_k(i + 1);
            add_values<kB, false, false>(st, w, s);
            multiply(i + 1);
            if constexpr (!Q8) landed();
            phase();
        }
        weigh(tiles - 1, std::true_type());
        phase();
        phase();
    } else {
        if constexpr (!Q8) landed();
        phase();
        multiply(0);
        if constexpr (Q8) landed();
        phase();
        for (int i = 0; i + 1 < tiles; ++i) {
            weigh(i, std::false_type());
            if constexpr (!Q8) landed();
            phase();
            refill(i + 1);
            if constexpr (Q8) read_k(i + 1);
            add_values<kB, false, false>(st, w, s);
            multiply(i + 1);
            if constexpr (Q8) landed();
            phase();
        }
        weigh(tiles - 1, std::true_type());
        phase();
    }
    add_values<kB, false, true>(st, w, s);
    wait_copies<0>();  // the copies past the last tile have landed too, before other data takes their place
    __syncthreads();
    f4_t* sums = reinterpret_cast<f4_t*>(ring) + rw * RT * 8 * 64 + lane;
    f4_t* rows = reinterpret_cast<f4_t*>(ring) + (RW * RT + wave) * 8 * 64;  // this wave's 16 rows of 128
    static_assert((RW * RT + kW) * 8 * 64 * 16 <= TL::kLds, "both in the ring");
    const float unit = Q8 ? s.cap * (1.0f / (1 << kHead)) : 1.0f;
    float l[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) l[r] = total<Q8>(s, r);
    // each half hands over one of two tiles and writes the other (of one tile: half 1 hands it over)
#pragma unroll
    for (int r = 0; r < RT; ++r)
        if (RT == 1 ? half == 1 : half != r) {
            if (quad == 0) {
                s_m[rw][r][col] = s.m[r];
                s_l[rw][r][col] = l[r];
            }
#pragma unroll
            for (int d = 0; d < 8; ++d) sums[(r * 8 + d) * 64] = s.acc[r][d];
        }
    if (lane == 0) s_cap[half][rw] = unit;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int row = (rw * RT + r) * kTileRows + col;
        if (RT == 1 ? half == 1 : half != r) continue;
        const float m1 = s_m[rw][r][col], M = fmaxf(s.m[r], m1);
        const float f0 = __builtin_amdgcn_exp2f(s.m[r] - M), f1 = __builtin_amdgcn_exp2f(m1 - M);
        const float c0 = f0 * unit, c1 = f1 * s_cap[half ^ 1][rw];
        f4_t o[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) o[d] = c0 * s.acc[r][d] + c1 * sums[(r * 8 + d) * 64];
        // through LDS (chunk c of row i at chunk c ^ i), so that a store is two whole rows
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // acc[d][e] is dim 8 (4 quad + e) + d
            rows[col * 32 + ((8 * quad + 2 * e) ^ col)] = f4_t{o[0][e], o[1][e], o[2][e], o[3][e]};
            rows[col * 32 + ((8 * quad + 2 * e + 1) ^ col)] = f4_t{o[4][e], o[5][e], o[6][e], o[7][e]};
        }
        if (quad == 0 && row < nrows)
            a.ml[qrow(row) * nsplit + split] = float2{M, f0 * l[r] + f1 * s_l[rw][r][col]};
        fence();  // LDS serves a wave's accesses in order
        __builtin_amdgcn_wave_barrier();
        fence();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int x = 2 * i + (lane >> 5), to = (rw * RT + r) * kTileRows + x;
            const f4_t v = rows[x * 32 + ((lane & 31) ^ x)];
            if (to < nrows)
                reinterpret_cast<f4_t*>(a.po + (qrow(to) * nsplit + split) * kHeadDim)[lane & 31] = v;
        }
    }
}

// =========================================================================================================== the join
// Block = row b * NH + h: the sum of its splits' (m, l, acc), each weighted by 2^(m - max m). Zeros where no slot had
// any weight. A split per 32 threads, 4 dims each.
constexpr int kJoinThreads = 256;
constexpr int kJoinGroups = kJoinThreads / 32;
// Partial sums in flight per thread, so that a row's latency is one for up to 64 splits: 5 hypotheses x 30001 int8 slots
// and 16 heads, 60 splits, 5.0 us one at a time, 4.6 with 4, 3.9 with 8.
constexpr int kJoinLoads = 8;
template <bool BF16>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(AttnArgs a) {
    __shared__ __align__(16) float s_o[kJoinGroups][kHeadDim];
    __shared__ float s_l[kJoinGroups];
    const int row = blockIdx.x, b = row / a.NH, lane = threadIdx.x & 63, grp = threadIdx.x >> 5;
    const int np = prefix_len(a), ns = suffix_len(a, b);
    const int cp = prefix_splits(a, np), cs = suffix_splits(a, ns);
    const int n = cp + cs;
    const float2* ml = a.ml + (size_t)row * (a.nsp + a.nss);
    const f4_t* po = reinterpret_cast<const f4_t*>(a.po) + (size_t)row * (a.nsp + a.nss) * 32 + (threadIdx.x & 31);
    auto at = [&](int i) { return i < cp ? i : a.nsp + i - cp; };
    f4_t o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    if (n > 0) {
        float M = kLowest;
        for (int j = lane; j < n; j += 64) M = fmaxf(M, ml[at(j)].x);
        for (int first = 0; first < n; first += kJoinGroups * kJoinLoads) {
            const int i = first + grp;
            f4_t v[kJoinLoads];
            float2 x[kJoinLoads];
#pragma unroll
            for (int u = 0; u < kJoinLoads; ++u) {
                const int j = at(min(i + u * kJoinGroups, n - 1));
                v[u] = po[32 * (size_t)j];
                x[u] = ml[j];
            }
            if (first == 0) M = wave_max(M);
#pragma unroll
            for (int u = 0; u < kJoinLoads; ++u) {
                if (i + u * kJoinGroups >= n) break;
                const float w = __builtin_amdgcn_exp2f(x[u].x - M);
                l += w * x[u].y;
                o += w * v[u];
            }
        }
    }
    *reinterpret_cast<f4_t*>(&s_o[grp][4 * (threadIdx.x & 31)]) = o;
    if ((threadIdx.x & 31) == 0) s_l[grp] = l;
    __syncthreads();
    if (threadIdx.x >= kHeadDim) return;
    float O = 0.f, L = 0.f;
#pragma unroll
    for (int g = 0; g < kJoinGroups; ++g) {
        O += s_o[g][threadIdx.x];
        L += s_l[g];
    }
    const float r = L == 0.f ? 0.f : O / L;
    a.o[(size_t)row * kHeadDim + threadIdx.x] = BF16 ? f32_to_bf16_bits(r) : f32_to_f16_bits(r);
}

// A long prefix goes to the wide kernel, which reads it once, from so much work on (slots x KV heads x groups of 16 rows)
// that reading it once per group from L2 takes longer than the wide kernel's extra launch and its larger start. In a
// graph, part_kernel against wide_kernel, 8 KV heads, plain: 20 rows x 10000 slots 19.7 / 19.5 us, x 30000 41 / 31; 64 x
// 4096 18.2 / 19.9, x 10000 31 / 22.0; 128 x 2500 22.0 / 22.4, x 30000 138 / 45. int8 (half the bytes, but codes
// to convert and scales to apply), bf16 and fp16 activations: 32 x 30000 27 / 40, 28 / 42; 48 x 65536 66 / 68, 66 / 73; 64 x
// 30000 44 / 43, 44 / 45, x 65536 83 / 69, 84 / 75; 80 x 30000 53 / 50, 53 / 56; 128 x 10000 34 / 35, 35 / 37, x 20000
// 56 / 47, 56 / 51.
constexpr long long kWideWork = 3 << 16, kWideWork8 = 1 << 20;
constexpr long long kWideMin = 1024;  // and none shorter, whatever the number of heads
constexpr int kWideRows = kTileRows, kWideRows8 = 3 * kTileRows;  // for more rows than these
// The blocks' sizes, 32, 64 or 128 rows: the larger one of two, with as many more splits, where a split is long enough
// to outweigh their partial sums, from about 12 tiles on: 64 rows as 32 / 64, x 10000 22.6 / 25.8 us, x 20000 29.2 /
// 31.4, x 65536 69 / 59; 128 rows as 64 / 128, x 10000 26 / 33, x 30000 44 / 45, x 65536 80 / 70.
constexpr long long kSplitTiles = 12;

struct Plan {
    int rt, rw, groups, groups_wide, nsp_narrow, nsp_wide, nsp, nss, wide_min;
    size_t ml, bytes;
};
Plan plan(int B, int NH, int NKV, int S, int T, bool p8) {
    Plan p;
    const long long rows = (long long)B * (NH / NKV);
    // `target` blocks over `others` of them per split
    auto splits = [](long long others, int target, int n, int quantum) {
        const long long s = std::min<long long>(kMaxSplits, std::max<long long>(1, target / others));
        return n ? (int)std::min<long long>(s, ((long long)n + quantum - 1) / quantum) : 0;
    };
    p.groups = (int)((rows + kTileRows - 1) / kTileRows);
    p.nss = splits((long long)NKV * B, kBlocks, T, kBlockStep);
    // a few suffix blocks leave the prefix the rest of the 512, so that none waits for a whole prefix block to end:
    // 5 hypotheses x 10000 int8 slots, 8 KV heads, 14.7 -> 13.1 us, x 30001 20.2 -> 19.1; with 192 of them the prefix
    // would be the longer for it (8 x 60000: 33.2 -> 38.0)
    const long long left = kBlocks - (long long)NKV * B * p.nss;
    p.nsp_narrow = splits(NKV * (long long)p.groups, left >= kBlocks * 7 / 8 ? (int)left : kBlocks, S, kBlockStep);
    // the wide kernel's splits: no more than an XCD's 32 CUs hold at a time of the row groups of every eighth of them
    auto wide = [&](int block_rows) {
        p.groups_wide = (int)((rows + block_rows - 1) / block_rows);
        p.nsp_wide = splits(NKV, 8 * std::max(32 / p.groups_wide, 1), S, kTileSlots);
        return S >= kSplitTiles * kTileSlots * p.nsp_wide;
    };
    p.rt = p.rw = p.groups_wide = p.nsp_wide = p.wide_min = 0;
    const long long per_slot = NKV * (long long)p.groups;
    const long long min_slots = std::max(((p8 ? kWideWork8 : kWideWork) + per_slot - 1) / per_slot, kWideMin);
    if (rows > (p8 ? kWideRows8 : kWideRows) && S >= min_slots) {
        p.wide_min = (int)min_slots;
        p.rt = rows > 64 && wide(128) ? 2 : 1;
        p.rw = p8 || rows > 64 || (rows > 32 && wide(64)) ? 4 : 2;
        wide(kTileRows * p.rt * p.rw);
    }
    p.nsp = std::max(p.nsp_narrow, p.nsp_wide);
    const size_t n = (size_t)B * NH * (p.nsp + p.nss);
    p.ml = n * kHeadDim * sizeof(float);
    p.bytes = p.ml + n * sizeof(float2);
    return p;
}

bool heads_ok(int NH, int NKV) {
    if (NKV <= 0 || NH <= 0 || NH % NKV) return false;
    const int r = NH / NKV;
    return r == 1 || r == 2 || r == 4 || r == 8;
}

template <bool Q8, int RT, int RW>
void launch_wide(const AttnArgs& a, bool bf, unsigned blocks, hipStream_t s) {
    auto k = bf ? wide_kernel<true, Q8, RT, RW> : wide_kernel<false, Q8, RT, RW>;
    hipLaunchKernelGGL(k, dim3(blocks), dim3(128 * RW), Tile<Q8>::kLds, s, a);
}

}  // namespace

extern "C" {

size_t rk_beam_attn_ws_bytes(int B, int NH, int NKV, int S, int T) {
    if (B <= 0 || !heads_ok(NH, NKV) || S < 0 || T < 0 || (S == 0 && T == 0)) return 0;
    return std::max(plan(B, NH, NKV, S, T, false).bytes, plan(B, NH, NKV, S, T, true).bytes);
}

int rk_beam_attn(const rk_beam_attn_params* p, rk_stream_t stream) {
    if (!p || !p->q || !p->o || !p->ws || (!p->kc && !p->ks)) return RK_ERR_NULL;
    if (p->kc && (!p->vc || !p->plen || (!p->kc_scale != !p->vc_scale))) return RK_ERR_NULL;
    if (p->ks && (!p->vs || !p->spos || (!p->ks_scale != !p->vs_scale))) return RK_ERR_NULL;
    const int S = p->kc ? p->S : 0, T = p->ks ? p->T : 0;
    if (p->HD != kHeadDim || p->B <= 0 || p->B > 65535 || !heads_ok(p->NH, p->NKV) || p->NKV > 65535 ||
        (p->kc && S <= 0) || (p->ks && (T <= 0 || p->rows <= 0 || (p->nspos != 1 && p->nspos != p->B))))
        return RK_ERR_SHAPE;
    if (p->ks && (p->src ? p->src_ld < T : p->rows < p->B)) return RK_ERR_SHAPE;
    const bool bf = p->dt == RK_BF16, p8 = p->kc && p->kc_scale, s8 = p->ks && p->ks_scale;
    if (p->ws_bytes < rk_beam_attn_ws_bytes(p->B, p->NH, p->NKV, S, T)) return RK_ERR_SHAPE;
    const Plan pl = plan(p->B, p->NH, p->NKV, S, T, p8);
    if (p->dt != RK_F16 && p->dt != RK_BF16) return RK_ERR_DTYPE;
    if (((uintptr_t)p->q | (uintptr_t)p->o | (uintptr_t)p->kc | (uintptr_t)p->vc | (uintptr_t)p->ks |
         (uintptr_t)p->vs | (uintptr_t)p->ws) & 15)
        return RK_ERR_ALIGN;
    AttnArgs a;
    a.q = (const uint16_t*)p->q; a.o = (uint16_t*)p->o;
    a.kc = p->kc; a.vc = p->vc; a.ks = p->ks; a.vs = p->vs;
    a.kcs = p->kc_scale; a.vcs = p->vc_scale; a.kss = p->ks_scale; a.vss = p->vs_scale;
    a.plen = p->plen; a.spos = p->spos; a.src = p->src;
    a.po = (float*)p->ws; a.ml = (float2*)((char*)p->ws + pl.ml);
    a.scale = p->scale; a.B = p->B; a.NH = p->NH; a.NKV = p->NKV; a.S = S; a.T = T;
    a.rows = p->rows; a.nspos = p->nspos; a.src_ld = p->src_ld;
    a.nsp = pl.nsp; a.nss = pl.nss; a.nsp_narrow = pl.nsp_narrow; a.nsp_wide = pl.nsp_wide;
    a.groups = pl.groups; a.groups_wide = pl.groups_wide;
    const long long prefix_blocks = (long long)pl.nsp_narrow * p->NKV * pl.groups;
    const long long blocks = prefix_blocks + (long long)p->B * p->NKV * pl.nss;
    const long long wide_blocks = ((long long)pl.nsp_wide * p->NKV + 7) / 8 * 8 * pl.groups_wide;
    if (blocks * kThreads > kMaxLaunch || wide_blocks * 512 > kMaxLaunch ||
        (long long)p->B * p->NH * kJoinThreads > kMaxLaunch)
        return RK_ERR_SHAPE;
    a.prefix_blocks = (int)prefix_blocks;
    a.wide_min = pl.wide_min;
    const hipStream_t s = (hipStream_t)stream;
    const long long direct_blocks = (long long)p->B * p->NKV;
    const int steps = direct_blocks > 512 ? 0 : direct_blocks >= 128 && direct_blocks <= 256 ? 3 : 1;
    if ((long long)S + T <= steps * kDirectSlots) {
        auto k = bf ? (p8 ? (s8 ? direct_kernel<true, true, true> : direct_kernel<true, true, false>)
                          : (s8 ? direct_kernel<true, false, true> : direct_kernel<true, false, false>))
                    : (p8 ? (s8 ? direct_kernel<false, true, true> : direct_kernel<false, true, false>)
                          : (s8 ? direct_kernel<false, false, true> : direct_kernel<false, false, false>));
        hipLaunchKernelGGL(k, dim3((unsigned)direct_blocks), dim3(64 * kDirectWaves), 0, s, a);
        return hipGetLastError() == hipSuccess ? RK_OK : RK_ERR_LAUNCH;
    }
    if (pl.nsp_wide) {
        const unsigned n = (unsigned)wide_blocks;
        if (pl.rw == 2) launch_wide<false, 1, 2>(a, bf, n, s);
        else if (p8) pl.rt == 1 ? launch_wide<true, 1, 4>(a, bf, n, s) : launch_wide<true, 2, 4>(a, bf, n, s);
        else pl.rt == 1 ? launch_wide<false, 1, 4>(a, bf, n, s) : launch_wide<false, 2, 4>(a, bf, n, s);
        if (hipGetLastError() != hipSuccess) return RK_ERR_LAUNCH;
    }
    auto k = bf ? (p8 ? (s8 ? part_kernel<true, true, true> : part_kernel<true, true, false>)
                      : (s8 ? part_kernel<true, false, true> : part_kernel<true, false, false>))
                : (p8 ? (s8 ? part_kernel<false, true, true> : part_kernel<false, true, false>)
                      : (s8 ? part_kernel<false, false, true> : part_kernel<false, false, false>));
    hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(kThreads), 0, s, a);
    if (hipGetLastError() != hipSuccess) return RK_ERR_LAUNCH;
    auto j = bf ? join_kernel<true> : join_kernel<false>;
    hipLaunchKernelGGL(j, dim3((unsigned)(p->B * p->NH)), dim3(kJoinThreads), 0, s, a);
    return hipGetLastError() == hipSuccess ? RK_OK : RK_ERR_LAUNCH;
}

int rk_beam_attn_params_size(void) { return (int)sizeof(rk_beam_attn_params); }

}  // extern "C"
