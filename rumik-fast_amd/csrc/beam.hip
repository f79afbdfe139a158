// One decode step's glue for B hypotheses of one prompt: everything after the fused projection (rk_beam_post) and a
// beam search's selection with the reordering of its states (rk_beam_pick). No counterpart in the reference, which
// decodes one sequence.
#include <algorithm>

#include "kv8.h"

namespace {

bool act_dt_ok(int dt) { return dt == RK_F16 || dt == RK_BF16; }

// =============================================================================================== rows after w_in
// Row b of y = [q | k | v | gate | up] at suffix slot t = spos[b] and position plen + t. A 16-lane group per (row, head):
// 8 values (4 RoPE pairs) per lane, so that a head is one coalesced 256-byte access and its int8 scale a maximum over
// the group; then the MLP channels, 8 per thread. Bound by launch latency at a few rows (0.3 MB at 4), by memory at
// many. VEC: rows 16-byte aligned (y, act, inter and ldy multiples of 8); else 2-byte accesses.
constexpr int kPostThreads = 256;
constexpr int kPostGroups = kPostThreads / kRowLanes;

struct PostArgs {
    const uint16_t* y;
    const int64_t* spos;
    const int64_t* plen;
    const uint16_t *cos_t, *sin_t;
    void *ks, *vs;
    float *kss, *vss;
    uint16_t *q, *act;
    int ldy, nspos, P, B, NH, NKV, T, inter, rope, head_blocks, act_blocks_per_row;
};

template <bool VEC>
RK_DEV u4_t load8(const uint16_t* s) {
    if constexpr (VEC) return *reinterpret_cast<const u4_t*>(s);
    u4_t v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (uint32_t)s[2 * e] | ((uint32_t)s[2 * e + 1] << 16);
    return v;
}

template <bool BF16, bool Q8, bool VEC>
__global__ __launch_bounds__(kPostThreads) void post_kernel(PostArgs a) {
    const int heads = a.NH + 2 * a.NKV;
    if ((int)blockIdx.x < a.head_blocks) {
        const int lane = threadIdx.x % kRowLanes;
        const int item = blockIdx.x * kPostGroups + threadIdx.x / kRowLanes;
        if (item >= a.B * heads) return;
        const int b = item / heads, h = item % heads;
        const int64_t t = a.spos[a.nspos > 1 ? b : 0], p0 = a.plen ? a.plen[0] : 0;
        // no slot or no table row for this position: the row's q, k and v are not written
        if (t < 0 || t >= a.T || (a.rope && (p0 < 0 || p0 >= a.P || p0 + t >= a.P))) return;
        u4_t x = load8<VEC>(a.y + (size_t)b * a.ldy + (size_t)h * kHeadDim + 8 * lane);
        if (a.rope && h < a.NH + a.NKV) {
            const size_t at = (size_t)(p0 + t) * kHeadDim + 8 * lane;
            float v[8], c[8], s[8];
            widen8<BF16>(x, v);
            widen8<BF16>(load8<VEC>(a.cos_t + at), c);
            widen8<BF16>(load8<VEC>(a.sin_t + at), s);
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float xe = v[e], xo = v[e + 1];
                v[e] = __builtin_fmaf(xe, c[e], -(xo * s[e]));
                v[e + 1] = __builtin_fmaf(xo, c[e], xe * s[e]);
                // rounded to fp32 and then to the type, as rk_post does: not one fused rounding (v_fma_mixlo_f16)
                asm("" : "+v"(v[e]), "+v"(v[e + 1]));
            }
            x = narrow8<BF16>(v);
        }
        if (h < a.NH) {
            *reinterpret_cast<u4_t*>(a.q + ((size_t)b * a.NH + h) * kHeadDim + 8 * lane) = x;
            return;
        }
        const bool is_v = h >= a.NH + a.NKV;
        const size_t row = ((size_t)b * a.NKV + (h - a.NH - (is_v ? a.NKV : 0))) * a.T + (size_t)t;
        void* cache = is_v ? a.vs : a.ks;
        if constexpr (Q8) {
            // the values a plain cache would hold (rounded to the activations' type), quantised
            float scale;
            const u2_t codes = quantize_row8<BF16>(x, scale);
            *reinterpret_cast<u2_t*>((int8_t*)cache + row * kHeadDim + 8 * lane) = codes;
            if (lane == 0) (is_v ? a.vss : a.kss)[row] = scale;
        } else {
            *reinterpret_cast<u4_t*>((uint16_t*)cache + row * kHeadDim + 8 * lane) = x;
        }
        return;
    }
    const int blk = blockIdx.x - a.head_blocks;
    const int b = blk / a.act_blocks_per_row;
    const int i = ((blk % a.act_blocks_per_row) * kPostThreads + threadIdx.x) * 8;
    if (i >= a.inter) return;
    const uint16_t* gp = a.y + (size_t)b * a.ldy + (size_t)heads * kHeadDim + i;
    uint16_t* out = a.act + (size_t)b * a.inter + i;
    if (VEC || i + 8 <= a.inter) {
        float g[8], u[8];
        widen8<BF16>(load8<VEC>(gp), g);
        widen8<BF16>(load8<VEC>(gp + a.inter), u);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = g[e] / (1.0f + __expf(-g[e])) * u[e];
        const u4_t r = narrow8<BF16>(g);
        if constexpr (VEC) {
            *reinterpret_cast<u4_t*>(out) = r;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) out[e] = (uint16_t)(r[e / 2] >> (16 * (e & 1)));
        }
    } else {
        for (int e = 0; i + e < a.inter; ++e) {
            const float g = load_act(gp, BF16 ? RK_BF16 : RK_F16, e);
            const float u = load_act(gp, BF16 ? RK_BF16 : RK_F16, a.inter + e);
            store_act(out, BF16 ? RK_BF16 : RK_F16, e, g / (1.0f + __expf(-g)) * u);
        }
    }
}

// ============================================================================================ beam search selection
// The value of token v for hypothesis b: score[b] + (x - m) - log(sum exp(x - m)), m its row's maximum. For an ended
// hypothesis the one candidate is (its own score, end_idx). Kept: the B best by value, the lower (hypothesis, token)
// first where equal. Two launches, joined by a workspace:
//   select  a block per up to 8192 logits of a row: their best kKeep in order (value, then lower index), their maximum
//           and sum of exponentials. Also copies what the second launch reads of the states, which may be updated in
//           place.
//   merge   every block picks the B best of all lists (the same work in each) and reorders its own columns of the tables;
//           block 0 writes the scalars.
// Both find the B best without sorting everything: of the maxima of 64 groups (of logits; of lists) the B-th largest is a
// bound that at least B candidates reach and few more do (about 64 ln 2 = 44 for B = 32); those are gathered in LDS and
// sorted by one wave, 64 to a sorting network. (A wave's maximum 32 times over for each 1024 logits, and every candidate
// ranked against all: 41 us instead of 12 for 8 x 16385, 271 instead of 18 for 32 x 131101.) Where few hypotheses lead,
// or all agree on the tokens, the merge's bound by lists lets through all of their candidates; a second bound, of groups
// of those, leaves a sort's worth or little more (32 x 131072 logits whose best ones are neighbours: 315 us when found one
// after the other, 17 so). What finds them one after the other is left for more candidates than LDS takes: equal ones (32 rows
// of 131072 equal logits: 418 us) and, in select, a row's best logits that all lie in few of the 64 groups but in more than
// one: at 2 to B - 1 residues of the index modulo 64 (8 x 16385: 30 us, 12 for random logits; 32 x 131072: 109, 19).
// Ordering key of a logit: (sortable(x) << 32) | (0xffffffff - index): a larger key is a larger logit, then a lower index.
constexpr int kKeep = 32;       // hypotheses at most, so candidates kept per list
// Logits of a lane: of 8, 10, 12 and 16 the fewest were the fastest (4 x 4096 9.3, 9.4, 9.6, 9.8 us; 32 x 131101 18.3, 18.3,
// 18.6, 19.5) but where a few blocks more than the card holds make a second round (32 x 151936: 20.6, 18.6, 18.9, 19.6).
constexpr int kPerLane = 8;
constexpr int kPiece = 64 * kPerLane;  // logits of a wave
constexpr int kPickWaves = 16;  // waves of a select block at most, a power of two
constexpr int kGather = 256;    // candidates that are gathered; more take the slow way
constexpr int kMergeThreads = 1024;
constexpr int kMergeWaves = kMergeThreads / 64;
constexpr int kMergeLists = 1024;  // lists that reach the bound
constexpr int kMergeGather = 2048; // their candidates that do
constexpr int kMergeCols = 128; // table columns per merge block
constexpr int kMergeRows = kKeep / (kMergeThreads / kMergeCols);  // rows of a thread
constexpr uint64_t kNone = 0;   // below every key of a logit: sortable(-NaN) alone would give it

RK_DEV uint32_t sortable(float x) {  // unsigned order of the values; -0 is 0
    const int32_t b = __builtin_bit_cast(int32_t, x + 0.0f);
    return (uint32_t)(b ^ ((b >> 31) & 0x7fffffff)) ^ 0x80000000u;
}
RK_DEV uint64_t logit_key(float x, uint32_t i) { return ((uint64_t)sortable(x) << 32) | (0xffffffffu - i); }
RK_DEV float key_logit(uint64_t k) {
    const int32_t b = (int32_t)((uint32_t)(k >> 32) ^ 0x80000000u);
    return __builtin_bit_cast(float, b ^ ((b >> 31) & 0x7fffffff));
}
RK_DEV int key_index(uint64_t k) { return (int)(0xffffffffu - (uint32_t)k); }

template <int M>
RK_DEV uint64_t xor64(uint64_t v) {
    return ((uint64_t)xor_lanes<M>((uint32_t)(v >> 32)) << 32) | xor_lanes<M>((uint32_t)v);
}
template <class T>
RK_DEV T shfl_xor(T v, int m) {  // m a power of two below 64, a constant once the callers' loops are unrolled
    if constexpr (sizeof(T) == 4) {
        switch (m) {
            case 1: return xor_lanes<1>(v);
            case 2: return xor_lanes<2>(v);
            case 4: return xor_lanes<4>(v);
            case 8: return xor_lanes<8>(v);
            case 16: return xor_lanes<16>(v);
            default: return xor_lanes<32>(v);
        }
    } else {
        switch (m) {
            case 1: return xor64<1>(v);
            case 2: return xor64<2>(v);
            case 4: return xor64<4>(v);
            case 8: return xor64<8>(v);
            case 16: return xor64<16>(v);
            default: return xor64<32>(v);
        }
    }
}

// the wave's 64 keys (one per lane) sorted, the largest in lane 0
template <class T>
RK_DEV T sort64(T x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) {
            const T o = shfl_xor(x, j);
            const bool keep_max = ((lane & j) == 0) == ((lane & k) == 0);
            x = keep_max == (o > x) ? o : x;
        }
    return x;
}

RK_DEV uint64_t wave_max64(uint64_t v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const uint64_t o = shfl_xor(v, m);
        v = o > v ? o : v;
    }
    return v;
}

struct PickState {
    const float* score;
    const uint8_t* done;
    const int64_t *lens, *step, *hist;
    const int32_t* src;
    float* score_out;
    uint8_t* done_out;
    int64_t *lens_out, *step_out, *hist_out;
    int32_t* src_out;
};

struct PickArgs {
    const void* logits;
    const int64_t* ids;
    PickState st;
    int64_t* tok;
    int32_t* parent;
    // workspace
    uint64_t* lists;  // [B][blocks][kKeep]
    float* sums;      // [B][blocks][2]: maximum, sum of exp(x - maximum)
    float* w_score;   // [B] copies
    int64_t* w_lens;  // [B]
    int64_t* w_step;  // [1]
    uint8_t* w_done;  // [B]
    long long ldl;
    int ldt, B, V, T, end_idx, min_new, blocks;  // blocks of select per row
};

// fp32 of the element at p: what T = 0 (fp16), 1 (bf16), 2 (fp32) is
template <int T>
RK_DEV float load_logit(const void* p, size_t i) { return load_act(p, T, i); }

template <int DT>
__global__ __launch_bounds__(64 * kPickWaves) void pick_select_kernel(PickArgs a) {
    __shared__ uint32_t s_group[64], s_bound;
    __shared__ uint64_t s_gather[kGather], s_best[kPickWaves];
    __shared__ float s_m[kPickWaves], s_sum[kPickWaves];
    __shared__ int s_count;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int b = blockIdx.x / a.blocks, blk = blockIdx.x % a.blocks;
    const int64_t step = a.st.step[0];
    const bool ended = a.st.done[b];
    // an index may pass 2^31 in the last block
    const uint32_t v0 = ((uint32_t)blk * waves + wave) * kPiece + lane;
    const size_t row = (size_t)b * a.ldl;
    float x[kPerLane];
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) x[i] = load_logit<DT>(a.logits, row + min(v0 + 64 * i, (uint32_t)a.V - 1));
    if (blockIdx.x == 0 && (int)threadIdx.x < a.B) {
        a.w_score[threadIdx.x] = a.st.score[threadIdx.x];
        a.w_lens[threadIdx.x] = a.st.lens[threadIdx.x];
        a.w_done[threadIdx.x] = a.st.done[threadIdx.x];
        if (threadIdx.x == 0) a.w_step[0] = step;
    }
    static_assert(kKeep <= 64, "a thread per hypothesis in a block of one wave");
    if (ended) return;  // the whole block
    if (threadIdx.x == 0) s_count = 0;
    if (wave == 0) s_group[lane] = 0;
    __syncthreads();
    const uint32_t mask = step < a.min_new ? (uint32_t)a.end_idx : ~0u;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        const uint32_t v = v0 + 64 * i;
        // no NaN, nothing beyond the largest finite value, no end token during the first min_new steps
        if (!(x[i] == x[i]) || v == mask || v >= (uint32_t)a.V) x[i] = -INFINITY;
        x[i] = fminf(x[i], 3.402823466e38f);
        top = fmaxf(top, x[i]);
    }
    atomicMax(&s_group[lane], sortable(top));  // a group: every 64th logit of the block, so that neighbours are apart
    __syncthreads();
    if (wave == 0) {  // -inf never is a candidate
        const uint32_t best = sort64(s_group[lane]);
        if (lane == a.B - 1) s_bound = max(best, sortable(-INFINITY) + 1u);
    }
    const float m = wave_max(top);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) sum += m == -INFINITY ? 0.f : __expf(x[i] - m);
    sum = wave_sum(sum);
    if (lane == 0) {
        s_m[wave] = m;
        s_sum[wave] = sum;
    }
    __syncthreads();
    const uint32_t bound = s_bound;
    if (__ballot(sortable(top) >= bound)) {
#pragma unroll
        for (int i = 0; i < kPerLane; ++i)
            if (sortable(x[i]) >= bound) {
                const int at = atomicAdd(&s_count, 1);  // in any order: they are sorted below
                if (at < kGather) s_gather[at] = logit_key(x[i], v0 + 64 * i);
            }
    }
    __syncthreads();
    const int count = s_count;
    uint64_t key = kNone;
    if (count <= kGather) {
        if (wave > 0) return;
        key = sort64(lane < count ? s_gather[lane] : kNone);
        for (int c = 64; c < count; c += 32) {  // the best 32 so far and the next 32
            if (lane >= 32) key = c + lane - 32 < count ? s_gather[c + lane - 32] : kNone;
            key = sort64(key);
        }
    } else {  // the block's largest key, again and again
        uint64_t below = ~0ull;
        for (int k = 0; k < a.B; ++k) {
            uint64_t next = kNone;
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) {
                const uint64_t y = sortable(x[i]) >= bound ? logit_key(x[i], v0 + 64 * i) : kNone;
                if (y < below && y > next) next = y;
            }
            next = wave_max64(next);
            __syncthreads();
            if (lane == 0) s_best[wave] = next;
            __syncthreads();
            below = kNone;
            for (int w = 0; w < waves; ++w) below = s_best[w] > below ? s_best[w] : below;
            if (lane == k) key = below;
        }
        if (wave > 0) return;
    }
    if (lane < kKeep) a.lists[(size_t)blockIdx.x * kKeep + lane] = key;
    const float wm = lane < waves ? s_m[lane] : -INFINITY;
    const float M = wave_max(wm);
    const float total = wave_sum(wm == -INFINITY ? 0.f : s_sum[lane] * __expf(wm - M));
    if (lane == 0) {
        a.sums[2 * (size_t)blockIdx.x] = M;
        a.sums[2 * (size_t)blockIdx.x + 1] = total;
    }
}

// A candidate of the merge: its value (as an unsigned order, 0: none) and (hypothesis << 32 | token), the lower first where
// values are equal.
struct Cand {
    uint64_t v, at;
};
RK_DEV bool before(const Cand& x, const Cand& y) { return x.v > y.v || (x.v == y.v && x.at < y.at); }
RK_DEV uint64_t value_order(double v) {  // unsigned order of the values; -inf is none
    if (v == -INFINITY) return 0;
    const int64_t k = __builtin_bit_cast(int64_t, v + 0.0);
    return (uint64_t)(k ^ ((k >> 63) & 0x7fffffffffffffffLL)) ^ 0x8000000000000000ull;
}
RK_DEV double order_value(uint64_t u) {
    const int64_t k = (int64_t)(u ^ 0x8000000000000000ull);
    return __builtin_bit_cast(double, k ^ ((k >> 63) & 0x7fffffffffffffffLL));
}
RK_DEV Cand shfl_xor_cand(const Cand& c, int m) { return {shfl_xor(c.v, m), shfl_xor(c.at, m)}; }
RK_DEV Cand sort64(Cand x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) {
            const Cand o = shfl_xor_cand(x, j);
            const bool keep_first = ((lane & j) == 0) == ((lane & k) == 0);
            if (keep_first == before(o, x)) x = o;
        }
    return x;
}

// One of 64 groups for item x of a row, such that the same x in many rows, and many x of a row, fall into many groups:
// the fractional parts of x and row times powers of 1 / 1.3247, the plane's counterpart of golden-ratio hashing.
RK_DEV int spread(uint32_t x, uint32_t row) { return (x * 0x91E10DA5u + row * 0xC13FA9A9u) >> 26; }

__global__ __launch_bounds__(kMergeThreads) void pick_merge_kernel(PickArgs a) {
    __shared__ double s_base[kKeep];
    __shared__ float s_max[kKeep];
    __shared__ bool s_ended[kKeep];
    __shared__ uint64_t s_group[64], s_bound;
    __shared__ int s_list[kMergeLists], s_lists;
    __shared__ Cand s_gather[kMergeGather], s_few[kGather], s_best[kMergeWaves];
    __shared__ int s_count, s_again, s_parent[kKeep];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int lists = a.B * a.blocks;
    const bool few = lists * a.B <= 64;  // all candidates at once
    const int64_t step = a.w_step[0];
    // the first loads beside the step's: a list's best per thread, or all candidates
    const int first = few ? min(lane / a.B, lists - 1) * kKeep + lane % a.B : min((int)threadIdx.x, lists - 1) * kKeep;
    const uint64_t head = a.lists[first];
    const int c0 = blockIdx.x * kMergeCols;
    constexpr int kRows = kKeep / kMergeWaves;  // a wave's rows: wave, wave + kMergeWaves
    float2 part[kRows];
    float score[kRows];
    bool ended[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const int b = min(wave + kMergeWaves * r, a.B - 1);
        part[r] = reinterpret_cast<const float2*>(a.sums)[(size_t)b * a.blocks + min(lane, a.blocks - 1)];
        score[r] = a.w_score[b];
        ended[r] = a.w_done[b];
    }
    if (step < 0 || step >= a.T) return;  // no column for this step: nothing is written
    if (blockIdx.x > 0 && c0 >= step) return;  // no column to reorder
    if (threadIdx.x < 64) s_group[threadIdx.x] = 0;
    if (threadIdx.x == 0) s_count = s_lists = s_again = 0;
    // a row's offset, its score - log(sum)
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const int b = wave + kMergeWaves * r;
        if (b >= a.B) break;
        const float2* sums = reinterpret_cast<const float2*>(a.sums) + (size_t)b * a.blocks;
        float m = -INFINITY, sum = 0.f;
        if (!ended[r]) {
            for (int p = lane; p < a.blocks; p += 64) {
                const float2 o = p == lane ? part[r] : sums[p];
                const float M = fmaxf(m, o.x);
                if (M != -INFINITY) sum = sum * __expf(m - M) + o.y * __expf(o.x - M);
                m = M;
            }
            const float M = wave_max(m);
            sum = wave_sum(m == -INFINITY ? 0.f : sum * __expf(m - M));
            m = M;
        }
        if (lane == 0) {
            s_ended[b] = ended[r];
            s_max[b] = m;
            s_base[b] = score[r] != score[r] ? -INFINITY
                                             : ended[r] ? (double)score[r] : (double)score[r] - log((double)sum);
        }
    }
    __syncthreads();
    // candidate `rank` of list l; an ended row's first one is the row itself
    auto candidate = [&](int l, int rank, uint64_t key) {
        const int b = l / a.blocks;
        const double base = s_base[b];
        if (s_ended[b]) return Cand{rank == 0 && l % a.blocks == 0 ? value_order(base) : 0,
                                    ((uint64_t)b << 32) | (uint32_t)a.end_idx};
        const bool is = key != kNone && base > -INFINITY;
        return Cand{is ? value_order(base + ((double)key_logit(key) - (double)s_max[b])) : 0,
                    ((uint64_t)b << 32) | (uint32_t)key_index(key)};
    };
    const Cand none = {0, ~0ull - lane};
    Cand best = none;
    if (few) {
        if (wave == 0) best = sort64(lane < lists * a.B ? candidate(lane / a.B, lane % a.B, head) : none);
    } else {
        // the B-th largest of 64 groups of the lists' best values; hypotheses often agree on the tokens, so on the lists
        for (int l = threadIdx.x; l < lists; l += kMergeThreads) {
            const uint64_t v = candidate(l, 0, l < kMergeThreads ? head : a.lists[(size_t)l * kKeep]).v;
            const int group = lists <= 64 ? l : spread(l % a.blocks, l / a.blocks);
            if (v) atomicMax((unsigned long long*)&s_group[group], (unsigned long long)v);
        }
        __syncthreads();
        if (wave == 0) {
            const uint64_t g = sort64(s_group[lane]);
            if (lane == a.B - 1) s_bound = g > 1 ? g : 1;
        }
        __syncthreads();
        const uint64_t bound = s_bound;
        // the lists that reach it, then their candidates that do
        for (int l = threadIdx.x; l < lists; l += kMergeThreads)
            if (candidate(l, 0, l < kMergeThreads ? head : a.lists[(size_t)l * kKeep]).v >= bound) {
                const int at = atomicAdd(&s_lists, 1);
                if (at < kMergeLists) s_list[at] = l;
            }
        __syncthreads();
        const int reach = s_lists;
        if (reach <= kMergeLists)
            for (int i = threadIdx.x / kKeep; i < reach; i += kMergeThreads / kKeep) {
                const int l = s_list[i], rank = threadIdx.x % kKeep;
                const Cand c = candidate(l, rank, a.lists[(size_t)l * kKeep + rank]);
                if (c.v >= bound) {
                    const int at = atomicAdd(&s_count, 1);  // in any order: they are sorted below
                    if (at < kMergeGather) s_gather[at] = c;
                }
            }
        __syncthreads();
        int count = reach <= kMergeLists ? s_count : kMergeGather + 1;
        bool again = count > 64 && count <= kMergeGather;
        if (again) {  // more than one sort takes, as where few hypotheses lead: a bound of 64 groups of these
            if (threadIdx.x < 64) s_group[threadIdx.x] = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < count; i += kMergeThreads) {
                const Cand c = s_gather[i];
                atomicMax((unsigned long long*)&s_group[spread((uint32_t)c.at, (uint32_t)(c.at >> 32))],
                          (unsigned long long)c.v);
            }
            __syncthreads();
            if (wave == 0) {
                const uint64_t g = sort64(s_group[lane]);
                if (lane == a.B - 1) s_bound = g > 1 ? g : 1;
            }
            __syncthreads();
            for (int i = threadIdx.x; i < count; i += kMergeThreads)
                if (s_gather[i].v >= s_bound) {
                    const int at = atomicAdd(&s_again, 1);
                    if (at < kGather) s_few[at] = s_gather[i];
                }
            __syncthreads();
            again = s_again <= kGather;
        }
        if (count <= kMergeGather) {
            if (wave == 0) {
                const Cand* from = again ? s_few : s_gather;
                if (again) count = s_again;
                best = sort64(lane < count ? from[lane] : none);
                for (int c = 64; c < count; c += 32) {  // the best 32 so far and the next 32
                    if (lane >= 32) best = c + lane - 32 < count ? from[c + lane - 32] : none;
                    best = sort64(best);
                }
            }
        } else {  // more than that: the best of all that come after the last one, again and again
            Cand last = {~0ull, 0};
            for (int k = 0; k < a.B; ++k) {
                Cand next = none;
                for (int i = threadIdx.x; i < lists * kKeep; i += kMergeThreads) {
                    const Cand c = candidate(i / kKeep, i % kKeep, a.lists[i]);
                    if (c.v && before(last, c) && before(c, next)) next = c;
                }
#pragma unroll
                for (int m = 1; m < 64; m <<= 1) {
                    const Cand o = shfl_xor_cand(next, m);
                    if (before(o, next)) next = o;
                }
                __syncthreads();
                if (lane == 0) s_best[wave] = next;
                __syncthreads();
                next = s_best[0];
                for (int w = 1; w < kMergeWaves; ++w)
                    if (before(s_best[w], next)) next = s_best[w];
                last = next;
                if (lane == k) best = next;
            }
        }
    }
    if ((int)threadIdx.x < a.B) {
        const int k = threadIdx.x;
        const bool live = best.v != 0;  // fewer candidates than hypotheses: the others end here
        const int p = live ? (int)(best.at >> 32) : k;
        s_parent[k] = p;
        if (blockIdx.x == 0) {
            const bool was = !live || a.w_done[p];
            const int c = live ? (int)(uint32_t)best.at : a.end_idx;
            const int64_t id = a.ids ? a.ids[c] : c;
            a.st.score_out[k] = live ? fmaxf((float)order_value(best.v), -3.402823466e38f) : -INFINITY;
            a.st.done_out[k] = was || c == a.end_idx;
            a.st.lens_out[k] = a.w_lens[p] + (was ? 0 : 1);
            a.tok[k] = id;
            a.parent[k] = p;
            a.st.hist_out[(size_t)k * a.T + step] = id;
            a.st.src_out[(size_t)k * a.T + step] = k;
            if (k == 0) a.st.step_out[0] = step + 1;
        }
    }
    __syncthreads();
    // the columns before this step: a block's old entries are all read before its new ones are written
    const int t = c0 + threadIdx.x % kMergeCols, k0 = threadIdx.x / kMergeCols * kMergeRows;
    const bool in = t < step && t < a.T;
    int64_t h[kMergeRows];
    int32_t s[kMergeRows];
#pragma unroll
    for (int k = 0; k < kMergeRows; ++k)
        if (in && k0 + k < a.B) {
            h[k] = a.st.hist[(size_t)s_parent[k0 + k] * a.T + t];
            s[k] = a.st.src[(size_t)s_parent[k0 + k] * a.T + t];
        }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kMergeRows; ++k)
        if (in && k0 + k < a.B) {
            a.st.hist_out[(size_t)(k0 + k) * a.T + t] = h[k];
            a.st.src_out[(size_t)(k0 + k) * a.T + t] = s[k];
        }
}

struct PickPlan {
    int blocks, waves;  // of select: blocks per row, waves in each
    size_t lists, sums, lens, step, score, done, bytes;
};
PickPlan pick_plan(int B, int V) {
    PickPlan w;
    const int pieces = (V - 1) / kPiece + 1;
    w.waves = 1;
    while (w.waves < pieces && w.waves < kPickWaves) w.waves *= 2;
    w.blocks = (pieces - 1) / w.waves + 1;
    const size_t n = (size_t)B * w.blocks;
    w.lists = 0;
    w.lens = n * kKeep * sizeof(uint64_t);
    w.step = w.lens + (size_t)B * sizeof(int64_t);
    w.sums = w.step + sizeof(int64_t);
    w.score = w.sums + 2 * n * sizeof(float);
    w.done = w.score + (size_t)B * sizeof(float);
    w.bytes = (w.done + (size_t)B + 15) & ~(size_t)15;
    return w;
}

}  // namespace

extern "C" {

int rk_beam_post(const void* y, int ldy, const int64_t* spos, int nspos, const int64_t* plen, const void* cos_t,
                 const void* sin_t, int P, void* ks, float* ks_scale, void* vs, float* vs_scale, void* q, void* act,
                 int dt, int B, int NH, int NKV, int HD, int T, int inter, int rope, rk_stream_t stream) {
    if (!y || !spos || !ks || !vs || !q || !act || (rope && (!cos_t || !sin_t)) || (!ks_scale != !vs_scale))
        return RK_ERR_NULL;
    const long long row = (long long)(NH + 2LL * NKV) * HD + 2LL * inter;
    if (HD != kHeadDim || B <= 0 || NH <= 0 || NKV <= 0 || NH % NKV || T <= 0 || inter <= 0 || ldy < row ||
        (nspos != 1 && nspos != B) || (rope && P <= 0))
        return RK_ERR_SHAPE;
    if (!act_dt_ok(dt)) return RK_ERR_DTYPE;
    // q and the caches take whole 16-byte rows; y, the tables and act may lie anywhere a 16-bit value may
    if (((uintptr_t)ks | (uintptr_t)vs | (uintptr_t)q) & 15) return RK_ERR_ALIGN;
    if ((((uintptr_t)y | (uintptr_t)cos_t | (uintptr_t)sin_t | (uintptr_t)act) & 1) ||
        (((uintptr_t)ks_scale | (uintptr_t)vs_scale) & 3))
        return RK_ERR_ALIGN;
    const long long items = (long long)B * (NH + 2LL * NKV);
    const long long per_row = (inter + 8LL * kPostThreads - 1) / (8LL * kPostThreads);
    const long long head_blocks = (items + kPostGroups - 1) / kPostGroups;
    if (items > 0x7fffffffLL || (head_blocks + per_row * B) * kPostThreads > kMaxLaunch) return RK_ERR_SHAPE;
    PostArgs a;
    a.y = (const uint16_t*)y; a.spos = spos; a.plen = plen;
    a.cos_t = (const uint16_t*)cos_t; a.sin_t = (const uint16_t*)sin_t;
    a.ks = ks; a.vs = vs; a.kss = ks_scale; a.vss = vs_scale; a.q = (uint16_t*)q; a.act = (uint16_t*)act;
    a.ldy = ldy; a.nspos = nspos; a.P = P; a.B = B; a.NH = NH; a.NKV = NKV; a.T = T; a.inter = inter; a.rope = rope;
    a.head_blocks = (int)head_blocks; a.act_blocks_per_row = (int)per_row;
    const bool vec = !(((uintptr_t)y | (uintptr_t)cos_t | (uintptr_t)sin_t | (uintptr_t)act) & 15) && ldy % 8 == 0 &&
                     inter % 8 == 0;
    const bool bf = dt == RK_BF16, q8 = ks_scale != nullptr;
    auto k = bf ? (q8 ? (vec ? post_kernel<true, true, true> : post_kernel<true, true, false>)
                      : (vec ? post_kernel<true, false, true> : post_kernel<true, false, false>))
                : (q8 ? (vec ? post_kernel<false, true, true> : post_kernel<false, true, false>)
                      : (vec ? post_kernel<false, false, true> : post_kernel<false, false, false>));
    hipLaunchKernelGGL(k, dim3((unsigned)(head_blocks + per_row * B)), dim3(kPostThreads), 0, (hipStream_t)stream, a);
    return hipGetLastError() == hipSuccess ? RK_OK : RK_ERR_LAUNCH;
}

size_t rk_beam_pick_ws_bytes(int B, int V) {
    if (B <= 0 || B > kKeep || V <= 0) return 0;
    return pick_plan(B, V).bytes;
}

int rk_beam_pick(const rk_beam_pick_params* p, rk_stream_t stream) {
    if (!p || !p->logits || !p->score || !p->done || !p->lens || !p->step || !p->hist || !p->src || !p->score_out ||
        !p->done_out || !p->lens_out || !p->step_out || !p->hist_out || !p->src_out || !p->tok || !p->parent || !p->ws)
        return RK_ERR_NULL;
    if (p->B <= 0 || p->B > kKeep || p->V <= 0 || p->T <= 0 || p->T > (1 << 29) || p->ldl < p->V || p->end_idx < 0 ||
        p->end_idx >= p->V)
        return RK_ERR_SHAPE;
    const PickPlan w = pick_plan(p->B, p->V);
    if (p->ws_bytes < w.bytes) return RK_ERR_SHAPE;
    if (p->logits_dtype != RK_F16 && p->logits_dtype != RK_BF16 && p->logits_dtype != RK_F32) return RK_ERR_DTYPE;
    if ((uintptr_t)p->ws & 15) return RK_ERR_ALIGN;
    PickArgs a;
    a.logits = p->logits; a.ids = p->ids; a.tok = p->tok; a.parent = p->parent;
    a.st = {p->score, p->done, p->lens, p->step, p->hist, p->src,
            p->score_out, p->done_out, p->lens_out, p->step_out, p->hist_out, p->src_out};
    char* ws = (char*)p->ws;
    a.lists = (uint64_t*)(ws + w.lists);
    a.sums = (float*)(ws + w.sums);
    a.w_score = (float*)(ws + w.score);
    a.w_lens = (int64_t*)(ws + w.lens);
    a.w_step = (int64_t*)(ws + w.step);
    a.w_done = (uint8_t*)(ws + w.done);
    a.ldl = p->ldl; a.ldt = p->logits_dtype; a.B = p->B; a.V = p->V; a.T = p->T; a.end_idx = p->end_idx;
    a.min_new = p->min_new; a.blocks = w.blocks;
    if ((long long)w.blocks * a.B * 64 * w.waves > kMaxLaunch) return RK_ERR_SHAPE;
    auto k = a.ldt == RK_F16 ? pick_select_kernel<RK_F16>
                             : a.ldt == RK_BF16 ? pick_select_kernel<RK_BF16> : pick_select_kernel<RK_F32>;
    hipLaunchKernelGGL(k, dim3(w.blocks * a.B), dim3(64 * w.waves), 0, (hipStream_t)stream, a);
    if (hipGetLastError() != hipSuccess) return RK_ERR_LAUNCH;
    hipLaunchKernelGGL(pick_merge_kernel, dim3((a.T - 1) / kMergeCols + 1), dim3(kMergeThreads), 0,
                       (hipStream_t)stream, a);
    return hipGetLastError() == hipSuccess ? RK_OK : RK_ERR_LAUNCH;
}

int rk_beam_pick_params_size(void) { return (int)sizeof(rk_beam_pick_params); }

}  // extern "C"
