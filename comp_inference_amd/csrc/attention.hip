// Attention over the paged key/value cache (layout and matrix operands: paged.h).
//
//   out[i, h] = sum_j w_j v[j, g],  w = softmax over the visible keys j of scale * q[i, h] . k[j, g],  g = h / group
//   query i of a sequence stands at position p = length - new tokens + i; key j is visible when j <= p and
//   (no window, or p - j < window, or j < sinks)
//
// One pass over the keys with a running maximum and sum per row (both, and the output, in 32 bits; weights are rounded to
// bf16 for the matrix instruction, off by at most 2^-8 of themselves each, while their sum takes them unrounded).  The
// query heads that share a kv head are rows of one product: row r of a sequence's kv head is (token r / group, head
// r % group).
//
// S^T = K Q^T puts queries into columns, so a lane holds 16 scores of ONE row and maximum and sum are lane arithmetic plus
// one exchange between lane halves, and P^T is the operand of O^T = V^T P^T as it stands.
//
// Two kernels:
//   attend_split_kernel   for few rows (single tokens): bound by reading the cache.  A tile is up to 32 rows; the blocks of
//                         keys of all (sequence, tile, head) items form one list that is cut into equal shares, one per
//                         workgroup, wherever the cut falls, so a batch of very different lengths fills the chip evenly.
//                         An item that was cut is joined by attend_join_kernel.  Measured, 32 heads over 8 of 128 (a
//                         copy on the same card moves 4.9 TB/s, read and written): one token each of 4 documents of 60
//                         to 131 thousand tokens, 1.6 GB: 270 us, 5.8 TB/s; of 64 ragged chats under a window of 4096,
//                         1.0 GB: 187 us, 5.4 TB/s; of 48 ragged chats in 4 bits, 0.86 GB: 181 us, 4.7 TB/s.
//   attend_rows_kernel    for many rows (prompts): bound by the matrix and vector units.  Eight wavefronts of 32 rows share
//                         the keys and values of a step of 64 tokens through the LDS, in two groups that take turns at the
//                         matrix unit.  Measured, the same heads: a prompt of 8192 tokens 545 us, 1.01 PFLOP/s (a large
//                         library product reaches 1.20), vector unit busy 42 % and matrix unit 46 % of the time; the last
//                         1500 tokens each of two sequences of up to 16384 in 4 bits 926 us, 0.63 PFLOP/s, 48 and 26 %:
//                         the vector unit has the steps and middles to apply as well; ragged prompts under a window of
//                         1000, 12 heads of 64, 111 us, 48 and 23 %.
#include "paged.h"

namespace ci {

struct AttendArgs {
    KvView cache;
    KvBatch batch;
    const uint16_t *q;
    uint16_t *out;
    float *lse;  // or nullptr: ln of the sum of exp(scores), [row, head]
    int64_t q_row, q_head, o_row, o_head, l_row;
    uint32_t group;  // query heads of a kv head
    double per_group;  // 1 / group
    float scale_log2;  // scale * log2(e): the kernel works on powers of two
    int32_t window, sinks;  // window 0: none
    float *work;            // partial sums of cut items
    uint32_t whole;         // 1: every item in one workgroup (no shares)
};

constexpr float kNone = -__builtin_inff();
constexpr uint32_t kUnit = 4;  // blocks of a unit of work: one per wavefront

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// (one instruction for three operands, and none to quiet a NaN first: a NaN among scores is carried by their weights)
__device__ __forceinline__ float most(float x, float y) { return __builtin_elementwise_maximum(x, y); }

__device__ __forceinline__ float other_half(float x) {  // the value of lane ^ 32
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}
__device__ __forceinline__ float lane_xor(float x, int d) {
    return __int_as_float(__shfl(__float_as_int(x), (int)(threadIdx.x & 63) ^ d, 64));
}
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }
__device__ __forceinline__ float max_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// row / group, exact: the quotient of row + 1/2 is at least 1 / (2 group) >= 2^-17 away from the next whole number, and the
// product is off by less than 2^-20 (rows are below 2^31).
__device__ __forceinline__ uint32_t token_of(const AttendArgs &a, uint32_t row) {
    return (uint32_t)(((double)row + 0.5) * a.per_group);
}
__device__ __forceinline__ uint32_t rows_of(const AttendArgs &a, const SeqInfo &s) { return (uint32_t)s.n * a.group; }

// Rows [r0, r1) of a sequence, and the blocks of keys some of them see: [0, s1) and [w0, w0 + nb - s1).
struct Span {
    int32_t p_lo, p_hi;  // positions of the first and last row
    uint32_t s1, w0, nb;
    __device__ __forceinline__ uint32_t block(uint32_t i) const { return i < s1 ? i : i - s1 + w0; }
};

__device__ __forceinline__ Span span_of(const AttendArgs &a, const SeqInfo &s, uint32_t r0, uint32_t r1) {
    Span x;
    x.p_lo = s.len - s.n + (int32_t)token_of(a, r0);
    x.p_hi = s.len - s.n + (int32_t)token_of(a, r1 - 1);
    const uint32_t end = x.p_hi < 0 ? 0 : (uint32_t)x.p_hi / kKvBlock + 1;
    x.s1 = x.w0 = 0;
    if (a.window) {
        x.w0 = x.p_lo - a.window + 1 > 0 ? (uint32_t)(x.p_lo - a.window + 1) / kKvBlock : 0;
        x.s1 = min(((uint32_t)a.sinks + kKvBlock - 1) / kKvBlock, end);
        if (x.s1 >= x.w0) x.s1 = x.w0 = 0;
    }
    x.nb = x.s1 + end - x.w0;
    return x;
}

__device__ __forceinline__ int32_t position_of(const AttendArgs &a, const SeqInfo &s, uint32_t row) {
    return s.len - s.n + (int32_t)token_of(a, row);
}

// Whether every row of the span sees every key of the block that starts at kb.
__device__ __forceinline__ bool all_visible(const AttendArgs &a, const Span &x, int32_t kb) {
    return kb + 31 <= x.p_lo && (!a.window || kb + 31 < a.sinks || kb > x.p_hi - a.window);
}
// Bits a .. b - 1 of a word (any a, b).
__device__ __forceinline__ uint32_t bits(int32_t a, int32_t b) {
    const uint32_t below_b = b >= 32 ? 0xFFFFFFFFu : b <= 0 ? 0u : (1u << b) - 1;
    const uint32_t below_a = a >= 32 ? 0xFFFFFFFFu : a <= 0 ? 0u : (1u << a) - 1;
    return below_b & ~below_a;
}
// The keys of the block at kb (a bit each) that some row at positions p_lo .. p_hi sees.
__device__ __forceinline__ uint32_t seen_keys(const AttendArgs &a, int32_t p_lo, int32_t p_hi, int32_t kb) {
    if (!a.window) return bits(0, p_hi + 1 - kb);
    return bits(p_lo - a.window + 1 - kb, p_hi + 1 - kb) | bits(0, min(a.sinks, p_hi + 1) - kb);
}


// One over a row's sum of weights.  The largest weight is at least one, so a sum of zero is that of a row that sees no key,
// which gets zeros, or of one whose scores are all minus infinity, which is no number.
__device__ __forceinline__ float inverse_sum(const AttendArgs &a, uint32_t seq, const SeqInfo &s, uint32_t row, float l) {
    if (l > 0.0f || l != l) return 1.0f / l;
    const Span x = span_of(a, s, row, row + 1);
    for (uint32_t i = x.nb; i > 0; --i)  // (its own key's page is the last)
        if (page_of(a.batch, a.cache, seq, x.block(i - 1)) != kNoPage) return __builtin_nanf("");
    return 0.0f;
}

// ---- matrix operands ------------------------------------------------------------------------------------------------
__device__ __forceinline__ f32x16_p mfma(u32x4 x, u32x4 y, f32x16_p c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_p, x), __builtin_bit_cast(bf16x8_p, y), c, 0, 0, 0);
}
// Eight codes as bf16 numbers 128 + code: 0x4300 is 128 with seven fraction bits, the last four of which are the code.  The
// mask is kept in a vector register: with two constants the and-or would be two instructions (and three a pair, shift
// included, instead of two).
struct CodeMask {
    uint32_t low_nibbles = 0x000F000Fu;
    __device__ __forceinline__ CodeMask() { asm volatile("" : "+v"(low_nibbles)); }
    __device__ __forceinline__ u32x4 to_bf16(uint32_t w) const {
        u32x4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = (w >> (4 * j) & low_nibbles) | 0x43004300u;
        return r;
    }
};
__device__ __forceinline__ f32x16_p splat16(float x) {
    f32x16_p r;
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = x;
    return r;
}

template <int D>
struct Queries {
    u32x4 f[D / 16];
    float sum;  // of all D channels
};

// Column `row` (of the rows of one kv head) as operand of S^T; columns at or beyond `rows` are zero.
template <int D>
__device__ __forceinline__ Queries<D> load_queries(const AttendArgs &a, const SeqInfo &s, uint32_t head, uint32_t row, uint32_t rows) {
    Queries<D> q;
    const uint32_t h = (threadIdx.x >> 5) & 1;
    const bool there = row < rows;
    const uint32_t tok = there ? token_of(a, row) : 0, g = there ? row - tok * a.group : 0;
    const uint16_t *src = a.q + (int64_t)(s.row + (int32_t)tok) * a.q_row + (int64_t)(head * a.group + g) * a.q_head;
    q.sum = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
        q.f[i] = u32x4{0, 0, 0, 0};
        if (there) q.f[i] = *reinterpret_cast<const u32x4 *>(src + 16 * i + 8 * h);
#pragma unroll
        for (int w = 0; w < 4; ++w) q.sum += bf16_lo(q.f[i][w]) + bf16_hi(q.f[i][w]);
    }
    q.sum += other_half(q.sum);
    return q;
}

// ---- few rows -------------------------------------------------------------------------------------------------------
// RP columns of the 32 are rows; the columns c, c + RP, c + 2 RP .. hold the same row.  Every one of them gets all 32 scores
// of a block in the product, and works on 32 / RP of them only: column c + j RP takes elements [j NV, (j + 1) NV) of its
// lane and puts zeros for the others into P^T, so O^T's columns are sums over disjoint sets of keys, each with a running
// maximum of its own, joined once per item.  With four rows (a token of a model with four query heads per kv head) a lane
// does the exponential of 2 scores per block instead of 16.
template <int RP>
struct Cols {
    static constexpr int NJ = 32 / RP, NV = 16 / NJ;
    uint32_t j;     // share of the lane's column
    uint32_t key0;  // first key of its share: key of value i is key0 + (i & 3) + 8 (i >> 2)
    __device__ __forceinline__ Cols() {
        const uint32_t lane = threadIdx.x & 63;
        j = (lane & 31) / RP;
        key0 = ((j * NV) & 3) + 8 * ((j * NV) >> 2) + 4 * (lane >> 5);
    }
    __device__ __forceinline__ void take(const f32x16_p &s, float (&x)[NV]) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            x[i] = s[i];
#pragma unroll
            for (int k = 1; k < NJ; ++k) x[i] = j == (uint32_t)k ? s[k * NV + i] : x[i];
        }
    }
    // P^T operands of the two halves of a block from the lane's own weights
    __device__ __forceinline__ void give(const uint32_t (&pk)[NV / 2], u32x4 (&f)[2]) const {
#pragma unroll
        for (int w = 0; w < 8; ++w) f[w / 4][w % 4] = (NJ == 1 || j == (uint32_t)(w / (NV / 2))) ? pk[w % (NV / 2)] : 0u;
    }
    // bf16 pairs (step, low) of the lane's keys
    __device__ __forceinline__ void pairs(const uint32_t *p, uint32_t (&x)[NV]) const {
#pragma unroll
        for (int i = 0; i < NV; i += 4) {
            if (NV == 2) {
                const u32x2 w = *reinterpret_cast<const u32x2 *>(p + key0);
                x[0] = w[0], x[1] = w[1];
            } else {
                const u32x4 w = *reinterpret_cast<const u32x4 *>(p + key0 + 8 * (i >> 2));
#pragma unroll
                for (int k = 0; k < 4; ++k) x[(i + k) % NV] = w[k];
            }
        }
    }
};

// The running state of a lane's column: maximum (in powers of two, of the scaled scores), sum, output.
template <int D>
struct Running {
    f32x16_p o[D / 32];
    float m, l, off;  // off: 4 bits: the part of the output that all channels share (sum of weight times the values' middles)
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] = splat16(0.0f);
        m = kNone;
        l = off = 0.0f;
    }
    // Raises the maximum where a block exceeds it by more than 2^8 (weights stay below 2^8 otherwise, which costs bf16 and
    // 32-bit sums no accuracy); what has been summed is scaled down only then.
    __device__ __forceinline__ void raise(float block_max) {
        if (__builtin_amdgcn_ballot_w64(block_max > m + 8.0f)) {
            const float to = fmaxf(m, block_max), f = m == kNone ? 0.0f : exp2_fast(m - to);
            m = to;
            l *= f;
            off *= f;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int k = 0; k < 16; ++k) o[i][k] *= f;
        }
    }
    __device__ __forceinline__ float base() const { return m == kNone ? 0.0f : m; }
    // whether something that was summed is an infinity or a NaN
    __device__ __forceinline__ bool no_number() const {
        float x = l * 0.0f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int k = 0; k < 16; ++k) x = fmaf(o[i][k], 0.0f, x);
        return x != x;
    }
};

// A value operand (s, h) without the keys that no row sees (what lies there need not be a number); `seen` has the lane's
// key 0 of the operand's half, 4 h, as bit 0.
__device__ __forceinline__ u32x4 keep_seen(u32x4 v, uint32_t seen, uint32_t s) {
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
        const uint32_t two = seen >> value_token(s, 0, 2 * w);
        v[w] &= ((two & 1) ? 0x0000FFFFu : 0u) | ((two & 2) ? 0xFFFF0000u : 0u);
    }
    return v;
}

template <int KIND, int D>
struct BlockData {  // keys and values of one block, as they lie in the cache
    static constexpr int N = KIND == CI_KV_BF16 ? D / 16 : D / 64;
    u32x4 k[N], v[N];
};

// Scores of a lane's keys of one block, from q . k (4 bits: q . (128 + code)); keys the row does not see get kNone.  `sees`:
// the lane's keys that its row sees, the share's first key as bit 0, looked at where `edge`.
template <int KIND, int D, int RP>
__device__ __forceinline__ void weigh_block(const AttendArgs &a, const Cols<RP> &cols, float q_sum, Running<D> &run, const f32x16_p &acc,
                                            bool edge, uint32_t sees, const uint32_t (&kp)[Cols<RP>::NV],
                                            const uint32_t (&vp)[Cols<RP>::NV], uint32_t (&pk)[Cols<RP>::NV / 2]) {
    constexpr int NV = Cols<RP>::NV;
    float t[NV];
    cols.take(acc, t);
    float best = kNone;
#pragma unroll
    for (int e = 0; e < NV; ++e) {
        // (q . (low + step code) from q . (128 + code))
        if (KIND != CI_KV_BF16) t[e] = (t[e] - 128.0f * q_sum) * bf16_lo(kp[e]) + q_sum * bf16_hi(kp[e]);
        t[e] *= a.scale_log2;
        if (edge) t[e] = sees >> ((e & 3) + 8 * (e >> 2)) & 1 ? t[e] : kNone;
        best = most(best, t[e]);
    }
    run.raise(max_halves(best));
    const float base = run.base();
#pragma unroll
    for (int e = 0; e < NV; e += 2) {
        const float p0 = exp2_fast(t[e] - base), p1 = exp2_fast(t[e + 1] - base);
        run.l += p0 + p1;
        if (KIND == CI_KV_BF16) {
            pk[e / 2] = bf16_pair(p0, p1);
        } else {
            // o = sum p (low + step code): the step goes into the weight r = p step, which is rounded, and what is added back
            // in 32 bits is sum p (low + 7.5 step) - sum r 135.5, so that the rounding of r meets code - 7.5 (as large as
            // the value is away from its row's middle) and not the code, or 128 with it.  A key that is not seen weighs
            // nothing, whatever its step and low are
            const float s0 = p0 * bf16_lo(vp[e]), s1 = p1 * bf16_lo(vp[e + 1]);
            float l0 = fmaf(s0, 7.5f, p0 * bf16_hi(vp[e])), l1 = fmaf(s1, 7.5f, p1 * bf16_hi(vp[e + 1]));
            pk[e / 2] = bf16_pair(s0, s1);
            if (edge) {
                const bool z0 = t[e] == kNone, z1 = t[e + 1] == kNone;
                l0 = z0 ? 0.0f : l0;
                l1 = z1 ? 0.0f : l1;
                pk[e / 2] &= (z0 ? 0u : 0xFFFFu) | (z1 ? 0u : 0xFFFF0000u);
            }
            run.off += l0 + l1 - 135.5f * (bf16_lo(pk[e / 2]) + bf16_hi(pk[e / 2]));
        }
    }
}

// ---- blocks done again ----------------------------------------------------------------------------------------------
// A matrix instruction multiplies the values of keys that SOME column of a tile takes by weights that are zero for the others;
// where such a value is an infinity or a NaN, and where a page was none of the cache's, sums come out as no numbers that
// should not.  A wavefront that finds one does its blocks again, with attend_again.
//
// Such values are taken out of the operands there, and what they are to the rows that do see them is found by a second
// product, of ones for the keys a column takes and of 1 for +infinity, 64 for -infinity, 4096 for NaN: up to 32 keys of each
// kind, counted exactly.  A key that is seen and weighs nothing has 4096 in place of the one: its infinities are NaN too.
//
// Measured with a NaN in a channel of the first value, which every row sees: a prompt of 8192 tokens, 32 heads over 8 of 128,
// 3.3 ms instead of 0.6; one token each over 20000, 45 us instead of 28.
constexpr uint32_t kBf16One = 0x3F80u, kBf16Minus = 0x4280u, kBf16NaN = 0x4580u;  // 1, 64, 4096

// A value operand without them; `most` is raised to the largest exponent (in place).
__device__ __forceinline__ u32x4 without_wild(u32x4 v, uint32_t &most) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const uint32_t lo = v[w] & 0x7F80u, hi = v[w] >> 16 & 0x7F80u;
        most = max(most, max(lo, hi));
        if (lo == 0x7F80u) v[w] &= 0xFFFF0000u;
        if (hi == 0x7F80u) v[w] &= 0xFFFFu;
    }
    return v;
}
// What they are, as numbers to count by.
__device__ __forceinline__ u32x4 kinds_of_wild(u32x4 v) {
    const auto kind = [](uint32_t x) { return x == 0x7F80u ? kBf16One : x == 0xFF80u ? kBf16Minus : (x & 0x7F80u) == 0x7F80u ? kBf16NaN : 0u; };
#pragma unroll
    for (int w = 0; w < 4; ++w) v[w] = kind(v[w] & 0xFFFFu) | kind(v[w] >> 16) << 16;
    return v;
}

// Sums of one wavefront's blocks block(i0), block(i0 + step) .. before `end` anew, for rows r0 .. r1 - 1.  Pages that do not
// exist are left out.  Nothing is asked for ahead and nothing is held from block to block but the sums (with heads of 64 a
// wavefront has 128 registers).
template <int KIND, int D, int RP, typename B>
__device__ __forceinline__ void attend_again(const AttendArgs &a, uint32_t seq, const SeqInfo &s, uint32_t head, uint32_t r0, uint32_t r1,
                                             uint32_t i0, uint32_t end, uint32_t step, B block, Running<D> &run) {
    constexpr int N = BlockData<KIND, D>::N, NV = Cols<RP>::NV;
    const uint32_t lane = threadIdx.x & 63, h = lane >> 5;
    const Cols<RP> cols;
    const CodeMask codes;
    run.clear();
#pragma unroll 1
    for (uint32_t i = i0; i < end; i += step) {
        const uint32_t blk = block(i);
        const int32_t kb = (int32_t)(blk * kKvBlock);
        if (kb >= s.len) continue;
        const uint32_t page = uniform(page_of(a.batch, a.cache, seq, blk));
        if (page == kNoPage) continue;
        const uint8_t *b = block_at<KIND, D>(a.cache, page, head, blk);
        asm volatile("" : "+s"(r0) : : "memory");  // (what is derived from it, or was asked for before, is so again)
        const uint32_t row = r0 + (lane & 31) % RP;
        const int32_t pos = position_of(a, s, row), p_lo = position_of(a, s, r0), p_hi = position_of(a, s, r1 - 1);
        const uint32_t sees = seen_keys(a, pos, pos, kb) >> cols.key0;
        f32x16_p acc = splat16(0.0f);
        uint32_t kp[NV], vp[NV], pk[NV / 2];
        float sum;
        {
            const Queries<D> q = load_queries<D>(a, s, head, row, r1);
            u32x4 x[N];
#pragma unroll
            for (int k = 0; k < N; ++k) x[k] = reinterpret_cast<const u32x4 *>(b)[k * 64 + lane];
            if (KIND != CI_KV_BF16) {
                const uint32_t *pairs = reinterpret_cast<const uint32_t *>(b + KvBlock<KIND, D>::kPairs);
                cols.pairs(pairs, kp);
                cols.pairs(pairs + kKvBlock, vp);
            }
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
                acc = mfma(KIND == CI_KV_BF16 ? x[k % N] : codes.to_bf16(x[k / 4 % N][k % 4]), q.f[k], acc);
            sum = q.sum;
        }
        weigh_block<KIND, D, RP>(a, cols, sum, run, acc, true, sees, kp, vp, pk);
        const uint32_t seen = seen_keys(a, p_lo, p_hi, kb) >> (4 * h);
        const auto value = [&](int s2, int db) {
            const int o = s2 * (D / 32) + db;
            const uint8_t *v = b + KvBlock<KIND, D>::kHalf;
            if (KIND != CI_KV_BF16) return codes.to_bf16(reinterpret_cast<const uint32_t *>(v)[(o / 4 * 64 + lane) * 4 + o % 4]);
            return keep_seen(reinterpret_cast<const u32x4 *>(v)[o * 64 + lane], seen, (uint32_t)s2);
        };
        uint32_t wild = 0;
        {
            u32x4 f[2];
            cols.give(pk, f);
#pragma unroll
            for (int db = 0; db < D / 32; ++db) {
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2)
                    run.o[db] = mfma(KIND == CI_KV_BF16 ? without_wild(value(s2, db), wild) : value(s2, db), f[s2], run.o[db]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (KIND != CI_KV_BF16 || !__builtin_amdgcn_ballot_w64(wild == 0x7F80u)) continue;
#pragma unroll
        for (int e = 0; e < NV; e += 2) {
            const uint32_t two = sees >> ((e & 3) + 8 * (e >> 2));
            const uint32_t lo = (pk[e / 2] & 0xFFFFu) ? kBf16One : kBf16NaN, hi = (pk[e / 2] >> 16) ? kBf16One : kBf16NaN;
            pk[e / 2] = ((two & 1) ? lo : 0u) | ((two & 2) ? hi << 16 : 0u);
        }
        u32x4 ones[2];
        cols.give(pk, ones);
#pragma unroll
        for (int db = 0; db < D / 32; ++db) {
            asm volatile("" ::: "memory");
            f32x16_p kinds = mfma(kinds_of_wild(value(0, db)), ones[0], splat16(0.0f));
            kinds = mfma(kinds_of_wild(value(1, db)), ones[1], kinds);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const uint32_t n = (uint32_t)kinds[k];
                if (n & 63) run.o[db][k] += __builtin_inff();
                if (n >> 6 & 63) run.o[db][k] -= __builtin_inff();
                if (n >> 12) run.o[db][k] = __builtin_nanf("");
            }
            __builtin_amdgcn_sched_barrier(0);  // (32 channels after the other: registers)
        }
    }
}

struct Item {
    uint32_t seq, tile, head;
};

// What the units of one (sequence, tile) are; every head of it has the same.
template <int RP>
__device__ __forceinline__ uint32_t units_of(const AttendArgs &a, const SeqInfo &s, uint32_t tile) {
    const uint32_t r0 = tile * RP, r1 = min(r0 + RP, rows_of(a, s));
    return max((span_of(a, s, r0, r1).nb + kUnit - 1) / kUnit, 1u);
}
template <int RP>
__device__ __forceinline__ uint32_t tiles_of(const AttendArgs &a, const SeqInfo &s) { return (rows_of(a, s) + RP - 1) / RP; }

// Units of a sequence over all its tiles and heads.
template <int RP>
__device__ __forceinline__ uint32_t weight_of(const AttendArgs &a, uint32_t i) {
    const SeqInfo s = load_seq_in_sum(a.batch, a.cache, i);
    uint32_t n = 0;
    for (uint32_t t = 0; t < tiles_of<RP>(a, s); ++t) n += units_of<RP>(a, s, t);
    return n * a.cache.kv_heads;
}
template <int RP>
__device__ __forceinline__ uint32_t items_of(const AttendArgs &a, uint32_t i) {
    return tiles_of<RP>(a, load_seq_in_sum(a.batch, a.cache, i)) * a.cache.kv_heads;
}

// Item number `index` of the batch.
template <int RP>
__device__ __forceinline__ bool find_item(const AttendArgs &a, uint32_t index, uint32_t *word, Item &it) {
    uint32_t begin;
    if (!a.batch.start && a.group <= RP) {  // one tile per sequence
        it.seq = index / a.cache.kv_heads;
        begin = it.seq * a.cache.kv_heads;
        if (it.seq >= a.batch.seqs) return false;
    } else {
        Found f;
        if (!locate(a.batch.seqs, [&](uint32_t i) { return items_of<RP>(a, i); }, [&](uint32_t) { return index; }, word, f))
            return false;
        it.seq = f.seq;
        begin = f.begin;
    }
    it.tile = (index - begin) / a.cache.kv_heads;
    it.head = (index - begin) % a.cache.kv_heads;
    return true;
}

// One workgroup's part of one item: units [u0, u1).  Joins its wavefronts and columns in the LDS, and writes the result:
// the item's rows, or (part of an item) the partial sums of RP rows to `slot`.
template <int KIND, int D, int RP>
__device__ __forceinline__ void attend_piece(const AttendArgs &a, const Item &it, const SeqInfo &s, uint32_t u0, uint32_t u1,
                                             bool whole, float *slot, uint8_t *lds) {
    constexpr int NV = Cols<RP>::NV, NJ = Cols<RP>::NJ;
    constexpr uint32_t kStride = D + 4;  // floats of a column in the LDS (the four spread the columns over the banks)
    typedef BlockData<KIND, D> Data;
    const uint32_t lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
    const uint32_t r0 = it.tile * RP, rows = min((uint32_t)RP, rows_of(a, s) - r0);
    const Span span = span_of(a, s, r0, r0 + rows);
    const Cols<RP> cols;
    const uint32_t row = col % RP;
    const Queries<D> q = load_queries<D>(a, s, it.head, r0 + row, r0 + rows);
    const int32_t pos = s.len - s.n + (int32_t)token_of(a, r0 + row);
    Running<D> run;
    run.clear();
    const uint32_t last = min(u1 * kUnit, span.nb);
    bool lost = false;

    auto fetch_k = [&](const uint8_t *b, Data &x) {
#pragma unroll
        for (int i = 0; i < Data::N; ++i) x.k[i] = reinterpret_cast<const u32x4 *>(b)[i * 64 + lane];
    };
    auto fetch_v = [&](const uint8_t *b, Data &x) {
#pragma unroll
        for (int i = 0; i < Data::N; ++i) x.v[i] = reinterpret_cast<const u32x4 *>(b + KvBlock<KIND, D>::kHalf)[i * 64 + lane];
    };
    PageRun table(a.batch, it.seq);
    // the block of a step (of a page that is none of the cache's: page 0; the blocks are done again)
    auto place = [&](uint32_t i) -> const uint8_t * {
        const uint32_t blk = span.block(i);
        table.hold(a.batch, a.cache, blk);
        const uint32_t page = table.page_of(a.cache, blk);
        lost = lost || page == kNoPage;
        return block_at<KIND, D>(a.cache, page == kNoPage ? 0 : page, it.head, blk);
    };

    // bf16: a block's keys are asked for a step ahead and its values at the head of its own step (8 KB or more are then always on
    // their way).  4 bits: a block is a quarter of that, so the next one is asked for whole, with its (step, low) pairs,
    // before this one is begun (48 chats of up to 32 k tokens: 214 us as for bf16, 195 so, 184 since codes become
    // operands in two instructions a pair; two blocks at a time 205).
    constexpr bool kPairsAhead = NV <= 8;  // (registers do not go further)
    const CodeMask codes;
    Data x, y;
    uint32_t kp[NV], vp[NV], kn[NV], vn[NV];
    auto fetch_pairs = [&](const uint8_t *b, uint32_t (&kw)[NV], uint32_t (&vw)[NV]) {
        const uint32_t *pairs = reinterpret_cast<const uint32_t *>(b + KvBlock<KIND, D>::kPairs);
        cols.pairs(pairs, kw);
        cols.pairs(pairs + kKvBlock, vw);
    };
    auto fetch_all = [&](const uint8_t *b, Data &d, uint32_t (&kw)[NV], uint32_t (&vw)[NV]) {
        fetch_k(b, d);
        fetch_v(b, d);
        if (kPairsAhead) fetch_pairs(b, kw, vw);
    };
    uint32_t i = u0 * kUnit + wave;
    const uint8_t *b = nullptr;
    if (i < last) {
        b = place(i);
        if (KIND == CI_KV_BF16) fetch_k(b, x);
        else fetch_all(b, x, kp, vp);
    }
    for (; i < last; i += kUnit) {
        const int32_t kb = (int32_t)(span.block(i) * kKvBlock);
        const bool edge = !all_visible(a, span, kb);
        uint32_t sees = 0xFFFFFFFFu;  // the lane's keys that its row sees, key0 as bit 0
        if (edge) sees = seen_keys(a, pos, pos, kb) >> cols.key0;
        if (KIND == CI_KV_BF16) {
            fetch_v(b, x);
        } else {
            if (!kPairsAhead) fetch_pairs(b, kp, vp);
            b = place(min(i + kUnit, last - 1));
            fetch_all(b, y, kn, vn);
        }
        f32x16_p acc = splat16(0.0f);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
            acc = mfma(KIND == CI_KV_BF16 ? x.k[k % Data::N] : codes.to_bf16(x.k[k / 4 % Data::N][k % 4]), q.f[k], acc);
        if (KIND == CI_KV_BF16) {
            b = place(min(i + kUnit, last - 1));
            fetch_k(b, x);
        }
        uint32_t pk[NV / 2];
        weigh_block<KIND, D, RP>(a, cols, q.sum, run, acc, edge, sees, kp, vp, pk);
        u32x4 f[2];
        cols.give(pk, f);
        if (KIND == CI_KV_BF16 && edge) {
            const uint32_t seen = seen_keys(a, span.p_lo, span.p_hi, kb) >> (4 * h);
#pragma unroll
            for (int k = 0; k < Data::N; ++k) x.v[k] = keep_seen(x.v[k], seen, (uint32_t)k / (D / 32));
        }
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
            for (int db = 0; db < D / 32; ++db) {
                const int k = s2 * (D / 32) + db;
                run.o[db] = mfma(KIND == CI_KV_BF16 ? x.v[k % Data::N] : codes.to_bf16(x.v[k / 4 % Data::N][k % 4]), f[s2], run.o[db]);
            }
        if (KIND != CI_KV_BF16) {
            x = y;
            if (kPairsAhead) {
#pragma unroll
                for (int e = 0; e < NV; ++e) kp[e] = kn[e], vp[e] = vn[e];
            }
        }
    }
    if (lost && lane == 0) report_bad_index(a.batch);
    if (__builtin_amdgcn_ballot_w64(row < rows && (lost || run.no_number())))
        attend_again<KIND, D, RP>(a, it.seq, s, it.head, r0, r0 + rows, u0 * kUnit + wave, last, kUnit,
                                  [&](uint32_t k) { return span.block(k); }, run);

    // ---- join: the columns of a wavefront that hold the same row (c, c + RP, ..), then the four wavefronts
    float *o_lds = reinterpret_cast<float *>(lds);                      // [4][32][kStride]
    float *m_lds = o_lds + 4 * 32 * kStride, *l_lds = m_lds + 4 * RP;  // [4][RP] each
    run.l += other_half(run.l);
    run.off += other_half(run.off);
    float m = run.m;
#pragma unroll
    for (int d = RP; d < 32; d *= 2) m = fmaxf(m, lane_xor(m, d));
    const float f = run.m == kNone ? 0.0f : exp2_fast(run.m - m);
    float l = run.l * f;  // (a NaN stays one: 0 x NaN)
#pragma unroll
    for (int d = RP; d < 32; d *= 2) l += lane_xor(l, d);
    __syncthreads();  // (the LDS is free of the piece before)
    if (lane < RP) {
        m_lds[wave * RP + lane] = m;
        l_lds[wave * RP + lane] = l;
    }
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            f32x4_p w;
#pragma unroll
            for (int c = 0; c < 4; ++c) w[c] = f * (run.o[db][4 * k + c] + (KIND == CI_KV_BF16 ? 0.0f : run.off));
            *reinterpret_cast<f32x4_p *>(o_lds + (wave * 32 + col) * kStride + 32 * db + 8 * k + 4 * h) = w;
        }
    __syncthreads();
    for (uint32_t o = threadIdx.x; o < rows * (D / 4); o += 256) {
        const uint32_t rr = o / (D / 4), d = o % (D / 4) * 4;
        const float top = fmaxf(fmaxf(m_lds[rr], m_lds[RP + rr]), fmaxf(m_lds[2 * RP + rr], m_lds[3 * RP + rr]));
        f32x4_p acc = {0.0f, 0.0f, 0.0f, 0.0f};
        float l = 0.0f;
#pragma unroll 1
        for (uint32_t w = 0; w < 4; ++w) {
            const float mw = m_lds[w * RP + rr], fw = mw == kNone ? 0.0f : exp2_fast(mw - top);
            l += fw * l_lds[w * RP + rr];
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const f32x4_p y = *reinterpret_cast<const f32x4_p *>(o_lds + (w * 32 + j * RP + rr) * kStride + d);
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[c] += fw * y[c];
            }
        }
        if (whole) {
            const float inv = inverse_sum(a, it.seq, s, r0 + rr, l);
            const uint32_t tok = token_of(a, r0 + rr), g = r0 + rr - tok * a.group;
            u32x2 w = {bf16_pair(acc[0] * inv, acc[1] * inv), bf16_pair(acc[2] * inv, acc[3] * inv)};
            *reinterpret_cast<u32x2 *>(a.out + (int64_t)(s.row + (int32_t)tok) * a.o_row +
                                       (int64_t)(it.head * a.group + g) * a.o_head + d) = w;
            if (a.lse && d == 0)
                a.lse[(int64_t)(s.row + (int32_t)tok) * a.l_row + it.head * a.group + g] =
                    top == kNone ? kNone : (top + log2f(l)) * 0.6931471805599453f;
        } else {
            *reinterpret_cast<f32x4_p *>(slot + rr * D + d) = acc;
            if (d == 0) {
                slot[RP * D + rr] = top;
                slot[RP * D + RP + rr] = l;
            }
        }
    }
}

template <int D, int RP>
constexpr uint32_t slot_floats() { return RP * (D + 2); }
constexpr uint32_t split_lds(int D) { return (4 * 32 * (D + 4) + 2 * 4 * 32) * 4; }

// Units of all items in the order (sequence, tile, head), cut evenly.
__device__ __forceinline__ uint32_t share_of(uint32_t total, uint32_t workers) { return max((total + workers - 1) / workers, 1u); }

template <int KIND, int D, int RP>
__global__ __launch_bounds__(256, 2) void attend_split_kernel(AttendArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    uint32_t *word = reinterpret_cast<uint32_t *>(lds);
    Item it;
    bool bad;
    // the share of this workgroup, and the item it begins in: one item, or units [at, end) of the batch's
    uint32_t at = 0, end = 0, u0 = 0, units = 0;
    SeqInfo s;
    if (a.whole) {
        if (!find_item<RP>(a, blockIdx.x, word, it)) return;
        s = load_seq(a.batch, a.cache, it.seq, bad);
        end = units = units_of<RP>(a, s, it.tile);
    } else {
        Found f;
        if (!locate(a.batch.seqs, [&](uint32_t i) { return weight_of<RP>(a, i); },
                    [&](uint32_t total) { return blockIdx.x * share_of(total, gridDim.x); }, word, f))
            return;
        it.seq = f.seq;
        at = f.target;
        end = min(at + share_of(f.total, gridDim.x), f.total);
        s = load_seq(a.batch, a.cache, it.seq, bad);
        uint32_t inside = at - f.begin;  // unit inside the sequence
        for (it.tile = 0;; ++it.tile) {
            units = units_of<RP>(a, s, it.tile);
            if (inside < units * a.cache.kv_heads) break;
            inside -= units * a.cache.kv_heads;
        }
        it.head = inside / units;
        u0 = inside % units;
    }
    for (;;) {
        if (bad && threadIdx.x == 0) report_bad_index(a.batch);
        const uint32_t u1 = min(units, u0 + end - at);
        // an item that goes on from the workgroup before leaves its sums in slot 0, one that goes on in the next in slot 1
        float *slot = a.work + (uint64_t)(blockIdx.x * 2 + (u0 == 0 ? 1 : 0)) * slot_floats<D, RP>();
        attend_piece<KIND, D, RP>(a, it, s, u0, u1, u0 == 0 && u1 == units, slot, lds);
        at += u1 - u0;
        if (at >= end) break;
        u0 = 0;
        if (++it.head < a.cache.kv_heads) continue;
        it.head = 0;
        if (++it.tile >= tiles_of<RP>(a, s)) {
            it.tile = 0;
            do {
                if (++it.seq >= a.batch.seqs) return;
                s = load_seq(a.batch, a.cache, it.seq, bad);
            } while (s.n == 0);
        }
        units = units_of<RP>(a, s, it.tile);
    }
}

// One row of one item that was cut: the sum of its parts, which 256 / (D / 4) groups of threads take in turn.
template <int KIND, int D, int RP>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs a, uint32_t workers) {
    constexpr uint32_t kLanes = D / 4, kGroups = 256 / kLanes;
    __shared__ uint32_t word[10];
    __shared__ float part[256 * 4];
    __shared__ float part_l[16];
    __shared__ float part_m[16];
    Item it;
    if (!find_item<RP>(a, blockIdx.x, word, it)) return;
    bool bad;
    const SeqInfo s = load_seq(a.batch, a.cache, it.seq, bad);
    const uint32_t r0 = it.tile * RP, rows = min((uint32_t)RP, rows_of(a, s) - r0), row = blockIdx.y;
    if (row >= rows) return;
    // where the item's units begin
    uint32_t total, before = 0;
    {
        const uint32_t per = (a.batch.seqs + 255) / 256, first = min(threadIdx.x * per, a.batch.seqs);
        const uint32_t end = min(first + per, a.batch.seqs);
        uint32_t mine = 0;
        for (uint32_t i = first; i < end; ++i) mine = add_work(mine, weight_of<RP>(a, i));
        before = scan_threads(mine, word, total);
        if (total == kTooMuch) return;  // (the same in every thread)
        if (it.seq >= first && it.seq < end) {
            for (uint32_t i = first; i < it.seq; ++i) before += weight_of<RP>(a, i);
            word[8] = before;
        }
        __syncthreads();
        before = uniform(word[8]);
        total = uniform(total);
    }
    for (uint32_t t = 0; t < it.tile; ++t) before += units_of<RP>(a, s, t) * a.cache.kv_heads;
    const uint32_t units = units_of<RP>(a, s, it.tile);
    before += it.head * units;
    const uint32_t share = share_of(total, workers), w0 = before / share, w1 = (before + units - 1) / share;
    if (w0 == w1) return;  // (written whole)
    // every group of threads takes each kGroups-th part, four of them asked for at a time, with a maximum of its own
    const uint32_t g = threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4;
    float m = kNone, l = 0.0f;
    f32x4_p acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t w = w0 + g; w <= w1; w += 4 * kGroups) {
        float mw[4], lw[4];
        f32x4_p y[4];
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {  // (past the last part: the last one again, with no weight)
            const uint32_t at = min(w + k * kGroups, w1);
            const float *slot = a.work + (uint64_t)(at * 2 + (at == w0 ? 1 : 0)) * slot_floats<D, RP>();
            mw[k] = slot[RP * D + row];
            lw[k] = slot[RP * D + RP + row];
            y[k] = *reinterpret_cast<const f32x4_p *>(slot + row * D + d);
        }
        float top = m;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) top = fmaxf(top, mw[k]);
        const float f0 = m == kNone ? 0.0f : exp2_fast(m - top);
        l *= f0;
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] *= f0;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            if (w + k * kGroups > w1) continue;
            const float f = mw[k] == kNone ? 0.0f : exp2_fast(mw[k] - top);
            l += f * lw[k];
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] += f * y[k][c];
        }
        m = top;
    }
    *reinterpret_cast<f32x4_p *>(part + threadIdx.x * 4) = acc;
    if (d == 0) part_l[g] = l, part_m[g] = m;
    __syncthreads();
    if (threadIdx.x < kLanes) {
        m = kNone;
#pragma unroll
        for (uint32_t k = 0; k < kGroups; ++k) m = fmaxf(m, part_m[k]);
        l = 0.0f;
        acc = f32x4_p{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t k = 0; k < kGroups; ++k) {
            const float f = part_m[k] == kNone ? 0.0f : exp2_fast(part_m[k] - m);
            l += f * part_l[k];
            const f32x4_p y = *reinterpret_cast<const f32x4_p *>(part + (k * kLanes + threadIdx.x) * 4);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] += f * y[c];
        }
        const float inv = inverse_sum(a, it.seq, s, r0 + row, l);
        const uint32_t tok = token_of(a, r0 + row), gh = it.head * a.group + r0 + row - tok * a.group;
        u32x2 w = {bf16_pair(acc[0] * inv, acc[1] * inv), bf16_pair(acc[2] * inv, acc[3] * inv)};
        *reinterpret_cast<u32x2 *>(a.out + (int64_t)(s.row + (int32_t)tok) * a.o_row + (int64_t)gh * a.o_head + d) = w;
        if (a.lse && d == 0)
            a.lse[(int64_t)(s.row + (int32_t)tok) * a.l_row + gh] = m == kNone ? kNone : (m + log2f(l)) * 0.6931471805599453f;
    }
}

// ---- many rows ------------------------------------------------------------------------------------------------------
constexpr uint32_t kStep = 64;  // keys
constexpr uint32_t kRowWaves = 8, kRowThreads = 64 * kRowWaves, kTileRows = 32 * kRowWaves;
constexpr uint32_t rows_lds(uint32_t kind, uint32_t D) {  // two buffers of two blocks, keys and values in bf16; steps and mids
    return 2 * 2 * 128 * D + (kind == CI_KV_BF16 ? 0 : 4 * 256 * 4);
}
// Workgroups resident on a CU: registers allow two wavefronts per SIMD, four for heads of 64 in bf16.
constexpr uint32_t row_groups(uint32_t kind, uint32_t dim) { return kind == CI_KV_BF16 && dim == 64 ? 2 : 1; }
constexpr uint32_t kWholeSteps = 32;                             // a tile of up to so many steps is never cut
constexpr uint32_t kLeastShare = 16;                             // steps (of 64 keys) worth a workgroup

struct Blocks {  // the two blocks of a step
    const uint8_t *b0, *b1;
};

// What a thread carries from memory to the LDS: its part of the keys of one step and of the values of the step before.
template <int KIND, int D>
struct Stage;

// The keys behind the end of a sequence need not be numbers; their scores are set, and their values (in 4 bits what these
// are scaled by) are put to zero here: clear(keys0, keys1, held0, held1) has a bit for every token that is there of the two
// blocks whose keys, and of the two whose values are staged.

// bf16: blocks are copied as they lie.
template <int D>
struct Stage<CI_KV_BF16, D> {
    static constexpr int N = 256 * D / (16 * kRowThreads);  // 16-byte pieces per thread of two blocks of 128 D bytes
    u32x4 x[N];
    static __device__ __forceinline__ uint32_t piece(int i) { return (i % (N / 2)) * kRowThreads + threadIdx.x; }  // of its block
    static __device__ __forceinline__ bool is_value(int i) { return uniform(piece(i)) >= 4 * D; }
    __device__ __forceinline__ void fetch(const Blocks &k, const Blocks &v) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint8_t *k01 = i < N / 2 ? k.b0 : k.b1, *v01 = i < N / 2 ? v.b0 : v.b1;
            x[i] = reinterpret_cast<const u32x4 *>(is_value(i) ? v01 : k01)[piece(i)];
        }
    }
    // values of tokens that are not there become zero
    __device__ __forceinline__ void clear(uint32_t, uint32_t, uint32_t held0, uint32_t held1) {
        const uint32_t h = (threadIdx.x >> 5) & 1;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (is_value(i)) x[i] = keep_seen(x[i], (i < N / 2 ? held0 : held1) >> (16 * ((piece(i) - 4 * D) / (2 * D)) + 4 * h), 0);
    }
    // keys to buffer `kb`, values to buffer `vb`
    __device__ __forceinline__ void store(uint8_t *kb, uint8_t *vb, float *, float) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            reinterpret_cast<u32x4 *>((is_value(i) ? vb : kb) + (i < N / 2 ? 0 : 128 * D))[piece(i)] = x[i];
    }
};

// 4 bits: codes become code - 7.5, exact in bf16, once for the wavefronts that use them; a key or value stands for
// mid + step (code - 7.5), mid = low + 7.5 step.  Step and mid are applied in 32 bits: to the scores (keys; with the scale), and to
// the weights before they are rounded (values), so what a 4-bit row stands for is never rounded itself, and a weight once,
// as over a bf16 cache.  A wavefront takes a whole 1 KB piece of codes, keys or values of one block (for heads of 64 there are
// four pieces, and the second group has none); the one with a block's first keys also takes the 64 (step, low) pairs.
template <int D>
struct Stage<CI_KV_INT4, D> {
    static constexpr int N = D / 64;  // pieces of the keys of a block
    u32x4 x;
    uint32_t pair;  // (step, low): of key `lane`, from lane 32 on of value lane - 32 of the step's keys' block
    static __device__ __forceinline__ uint32_t unit() { return uniform(threadIdx.x >> 6); }
    static __device__ __forceinline__ bool idle() { return unit() >= 4 * N; }
    static __device__ __forceinline__ uint32_t block() { return unit() / (2 * N) & 1; }
    static __device__ __forceinline__ uint32_t values() { return unit() / N & 1; }
    static __device__ __forceinline__ uint32_t index() { return unit() % N; }
    __device__ __forceinline__ void fetch(const Blocks &kb, const Blocks &vb) {
        const uint32_t lane = threadIdx.x & 63;
        // (chosen by arithmetic: a choice between the four would put them into memory)
        const int64_t blk = -(int64_t)block(), val = -(int64_t)values();
        const uint8_t *k = kb.b0 + ((kb.b1 - kb.b0) & blk), *v = vb.b0 + ((vb.b1 - vb.b0) & blk), *b = k + ((v - k) & val);
        x = reinterpret_cast<const u32x4 *>(b + values() * KvBlock<CI_KV_INT4, D>::kHalf)[index() * 64 + lane];
        pair = reinterpret_cast<const uint32_t *>(k + KvBlock<CI_KV_INT4, D>::kPairs)[lane];
    }
    // (a value of a token that is not there: step 0, mid 0)
    __device__ __forceinline__ void clear(uint32_t keys0, uint32_t keys1, uint32_t, uint32_t) {
        const uint32_t lane = threadIdx.x & 63, held = block() ? keys1 : keys0;
        if (lane >= 32 && !(held >> (lane & 31) & 1)) pair = 0;
    }
    static __device__ __forceinline__ u32x4 centred(uint32_t word) {
        const uint32_t even = word & 0x0F0F0F0Fu, odd = word >> 4 & 0x0F0F0F0Fu;  // codes 0, 4, 1, 5 and 2, 6, 3, 7, a byte each
        u32x4 r;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint32_t from = w % 2 ? odd : even;
            r[w] = bf16_pair((float)(from >> (w < 2 ? 0 : 8) & 0xFFu) - 7.5f, (float)(from >> (w < 2 ? 16 : 24) & 0xFFu) - 7.5f);
        }
        return r;
    }
    __device__ __forceinline__ void store(uint8_t *kb, uint8_t *vb, float *grid, float scale) const {
        if (N == 1 && idle()) return;
        const uint32_t lane = threadIdx.x & 63;
        u32x4 *dst = reinterpret_cast<u32x4 *>((values() ? vb : kb) + block() * 128 * D + values() * 64 * D) + index() * 256 + lane;
#pragma unroll
        for (int c = 0; c < 4; ++c) dst[c * 64] = centred(x[c]);
        if (!values() && index() == 0) {
            const float f = lane < 32 ? scale : 1.0f, step = bf16_lo(pair) * f;
            float *mine = grid + (lane >> 5) * 128 + block() * 32 + (lane & 31);
            mine[0] = step;
            mine[64] = fmaf(step, 7.5f, bf16_hi(pair) * f);
        }
    }
};

// The work of a sequence in steps, and how its items follow each other.  Under a causal mask tile t takes about as many
// steps more than the first as tile T - 1 - t takes fewer than the last: the two together are given a fixed number of
// places, `pair`, at least what any such two need, so a place in the list is found without summing over tiles.  Order:
// (head, pair of tiles, the shorter, the longer), the tile in the middle of an odd number alone at the end; a few places
// at the end of each pair are empty.
struct TileList {
    uint32_t tiles, pair, middle, head;  // head: places of one head
};

// The steps (64 keys from a multiple of 64) that rows at p_lo .. p_hi see a key of: [0, s1) and [w0, w0 + n - s1).
struct Steps {
    uint32_t s1, w0, n;
    __device__ __forceinline__ int32_t first_key(uint32_t i) const { return (int32_t)((i < s1 ? i : i - s1 + w0) * kStep); }
};
__device__ __forceinline__ Steps steps_between(const AttendArgs &a, int32_t p_lo, int32_t p_hi) {
    Steps x{};
    const uint32_t end = p_hi < 0 ? 0 : (uint32_t)p_hi / kStep + 1;
    if (a.window) {
        x.w0 = p_lo - a.window + 1 > 0 ? (uint32_t)(p_lo - a.window + 1) / kStep : 0;
        x.s1 = min(((uint32_t)a.sinks + kStep - 1) / kStep, end);
        if (x.s1 >= x.w0) x.s1 = x.w0 = 0;
    }
    x.n = x.s1 + end - x.w0;
    return x;
}
__device__ __forceinline__ uint32_t steps_of(const AttendArgs &a, const SeqInfo &s, uint32_t tile) {
    const uint32_t r0 = tile * kTileRows, r1 = min(r0 + kTileRows, rows_of(a, s));
    return max(steps_between(a, position_of(a, s, r0), position_of(a, s, r1 - 1)).n, 1u);
}

__device__ __forceinline__ TileList tiles_in(const AttendArgs &a, const SeqInfo &s) {
    TileList l;
    l.tiles = (rows_of(a, s) + kTileRows - 1) / kTileRows;
    if (l.tiles == 0) return TileList{0, 0, 0, 0};
    // without a window a tile whose last row stands at p takes p / 64 + 1 steps; positions grow evenly from tile to tile (the
    // last tile counted as a full one), rounded down, so two opposite tiles' sum at most 1 above the outer two's
    const int32_t first = s.len - s.n;
    const int32_t x = max(first + (int32_t)token_of(a, kTileRows - 1), 0);
    const int32_t y = max(first + (int32_t)token_of(a, l.tiles * kTileRows - 1), 0);
    l.pair = ((uint32_t)x + (uint32_t)y + 1) / 64 + 2;  // (positions up to 2^30 and a tile behind: no room for a sign)
    if (a.window) {  // a tile's steps: the sinks', and those from its first row's window to its last row
        const uint32_t tokens = token_of(a, kTileRows + a.group - 2) + 1;
        l.pair = min(l.pair, 2 * (((uint32_t)a.sinks + kStep - 1) / kStep + ((uint32_t)a.window + tokens) / kStep + 2));
    }
    l.middle = l.tiles % 2 ? steps_of(a, s, l.tiles / 2) : 0;
    l.head = l.tiles / 2 * l.pair + l.middle;
    return l;
}

// A tile's places: [begin, begin + places) of its head's.
struct TilePlace {
    uint32_t tile, begin, places;
};
__device__ __forceinline__ TilePlace tile_at(const AttendArgs &a, const SeqInfo &s, const TileList &l, uint32_t place) {
    const uint32_t half = l.tiles / 2, k = l.pair ? min(place / l.pair, half) : 0;
    if (k == half) return TilePlace{half, half * l.pair, l.middle};
    const uint32_t shorter = steps_of(a, s, k), at = k * l.pair;
    if (place - at < shorter) return TilePlace{k, at, shorter};
    return TilePlace{l.tiles - 1 - k, at + shorter, l.pair - shorter};
}
// The list is cut every `share` places, but a cut near a tile's begin or end is moved there.  A cut tile's partial sums go
// through memory, which costs about as much as eight steps (2 x 256 rows x D x 4 bytes written and read again, against
// 256 x 64 x D x 4 flops a step), so a share may be that much uneven, or a sixteenth.
struct RowShare {
    uint32_t share, slack;
    __device__ __forceinline__ RowShare(uint32_t total, uint32_t workers) {
        share = max((total + workers - 1) / workers, kLeastShare);
        slack = max(share / 16, 7u);
    }
    // where a cut `off` places behind a tile's begin (0 < off < places, or 0) goes; a tile of few steps is never cut
    __device__ __forceinline__ uint32_t cut(uint32_t off, uint32_t places) const {
        if (places <= kWholeSteps) return 2 * off < places ? 0 : places;
        return off <= slack ? 0 : places - off <= slack ? places : off;
    }
};

// The end of a phase: what was put into the LDS is there, loads from memory go on.
__device__ __forceinline__ void phase_end() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
}

// Steps [u0, u1) of one tile of one head.
//
// Two groups of four wavefronts, one of each on every SIMD, half a step apart: while one group's matrix instructions run (the
// output of the step before, the scores of this one), the other works out its weights on the vector unit.  A phase ends at
// a barrier.  With phases counted from 0, the first group's matrix phase of step u0 + t is phase 2 t, its vector phase
// 2 t + 1; the second group's are one later.  Step t's keys are read in phases 2 t and 2 t + 1, its values in 2 t + 2 and
// 2 t + 3, both from one of two buffers.  Both groups store their parts of keys t + 1 and values t in matrix phase t (phases
// 2 t and 2 t + 1): after the last read of what lay there (keys t - 1 and values t - 2: phase 2 t - 1) and before phase 2 t + 2
// reads them.  Storing, and asking for the next, is a matter of the matrix phase because there the other units are idle.
template <int KIND, int D>
__device__ __forceinline__ void attend_rows_piece(const AttendArgs &a, uint32_t seq, const SeqInfo &s, uint32_t head, uint32_t tile,
                                                  uint32_t u0, uint32_t u1, bool whole, float *slot, uint8_t *lds) {
    const uint32_t lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
    const uint32_t t0 = tile * kTileRows, t1 = min(t0 + kTileRows, rows_of(a, s));
    const Steps steps = steps_between(a, position_of(a, s, t0), position_of(a, s, t1 - 1));
    const uint32_t r0 = t0 + wave * 32, r1 = min(r0 + 32, t1);
    const bool any = r0 < r1;
    const Queries<D> q = load_queries<D>(a, s, head, r0 + col, t1);
    const int32_t pos = position_of(a, s, r0 + col);
    // the wavefront's rows stand at p_lo .. p_hi
    const int32_t p_lo = position_of(a, s, any ? r0 : t0), p_hi = any ? position_of(a, s, r1 - 1) : -1;
    Running<D> run;
    run.clear();

    const uint32_t last = min(u1, steps.n);
    const bool second = wave >= kRowWaves / 2;
    Stage<KIND, D> stage;
    PageRun table(a.batch, seq);
    bool lost = false;  // whether a block was on no page of the cache (page 0 then stands for it, and the rows are done again)
    const uint32_t last_block = s.len > 0 ? (uint32_t)(s.len - 1) / kKvBlock : 0;
    const auto buffer = [&](uint32_t st) { return lds + (st & 1) * (256 * D); };
    // 4 bits: steps and mids of a step's keys and values, [2][step 64, mid 64], stored with its keys and read in its vector phase
    // (the second group's is phase 2 t + 2, in which the first stores those of step t + 2): four of them in turn
    const auto grid = [&](uint32_t st) { return reinterpret_cast<float *>(lds + 512 * D) + (st & 3) * 256; };
    const auto first_block = [&](uint32_t st) { return (uint32_t)steps.first_key(min(st, last - 1)) / kKvBlock; };
    const auto at_block = [&](uint32_t blk) {
        const uint32_t x = table.page_of(a.cache, blk);
        lost = lost || x == kNoPage;
        return block_at<KIND, D>(a.cache, x == kNoPage ? 0 : x, head, blk);
    };
    Blocks kp{}, vp{};
    const auto ask = [&](uint32_t st) {  // keys of step st (the last one's again behind it), values of the step asked for before
        vp = kp;
        const uint32_t blk = first_block(st);
        kp.b0 = at_block(blk);
        kp.b1 = at_block(min(blk + 1, last_block));  // (none behind the sequence's end)
        stage.fetch(kp, vp);
    };
    // what is staged: keys of step ks, values of the step before
    const auto put = [&](uint32_t ks) { stage.store(buffer(ks), buffer(ks - 1), grid(ks), a.scale_log2); };
    const auto clear = [&](uint32_t ks) {
        const int32_t kb = (int32_t)(first_block(ks) * kKvBlock), vb = (int32_t)(first_block(ks - 1) * kKvBlock);
        if (max(kb, vb) + (int32_t)kStep > s.len)
            stage.clear(bits(0, s.len - kb), bits(0, s.len - kb - 32), bits(0, s.len - vb), bits(0, s.len - vb - 32));
    };
    const auto hold = [&](uint32_t st) {
        if (!table.hold(a.batch, a.cache, first_block(st)) || !a.window) return;
        // a page of a step that lies before the window's first key and behind the sinks is seen by no row of the tile and may be
        // gone: page 0 stands for it (looked at here, not where blocks are asked for: there it would stop the matrix unit,
        // 777 instead of 552 us for a prompt of 8192 tokens)
        const uint32_t at = table.held * 64 + lane, shift = a.cache.page_shift + 5;
        if ((int32_t)((at + 1) << shift) <= position_of(a, s, t0) - a.window + 1 && at << shift >= (uint32_t)a.sinks) table.pages = 0;
    };
    // steps [clean0, clean1) need no mask for the wavefront's rows
    const uint32_t clean0 = a.window ? steps.s1 + (p_hi - a.window < 0 ? 0u : max((uint32_t)(p_hi - a.window) / kStep + 1, steps.w0) - steps.w0) : 0;
    const uint32_t clean1 = p_lo + 1 < (int32_t)kStep ? 0 : steps.s1 + max((uint32_t)(p_lo + 1) / kStep, steps.w0) - steps.w0;

    constexpr int kBlk = 8 * D;  // 16-byte pieces of a block: keys, then values
    f32x16_p acc0, acc1;
    u32x4 p[4];
    const auto output = [&](uint32_t st) {
        const u32x4 *kv = reinterpret_cast<const u32x4 *>(buffer(st)) + 4 * D + lane;
#pragma unroll
        for (int s2 = 0; s2 < 4; ++s2)
#pragma unroll
            for (int db = 0; db < D / 32; ++db)
                run.o[db] = mfma(kv[(s2 / 2) * kBlk + ((s2 % 2) * (D / 32) + db) * 64], p[s2], run.o[db]);
    };
    const auto scores = [&](uint32_t st) {
        const u32x4 *kv = reinterpret_cast<const u32x4 *>(buffer(st)) + lane;
        acc0 = acc1 = splat16(0.0f);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            acc0 = mfma(kv[k * 64], q.f[k], acc0);
            acc1 = mfma(kv[kBlk + k * 64], q.f[k], acc1);
        }
    };
    __syncthreads();  // (the LDS is free of the piece before)
    if (u0 < last) {
        hold(u0);
        kp.b0 = at_block(first_block(u0));  // (the first step's values go with its keys, unread)
        kp.b1 = kp.b0;
        ask(u0);
        clear(u0);
        put(u0);
        hold(u0 + 1);
        ask(u0 + 1);
        hold(u0 + 2);
        clear(u0 + 1);
        __syncthreads();
        if (second) phase_end();
        put(u0 + 1);
        ask(u0 + 2);
        scores(u0);
        phase_end();
    }
    for (uint32_t st = u0; st < last; ++st) {
        // ---- vector phase
        hold(st + 3);
        clear(st + 2);
        const f32x4_p *of = reinterpret_cast<const f32x4_p *>(grid(st)) + h;
        if (KIND != CI_KV_BF16) {  // scale q . (mid + step (code - 7.5)), from q . (code - 7.5) and the sum of q
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4_p s0 = of[2 * g], s1 = of[8 + 2 * g], m0 = of[16 + 2 * g], m1 = of[24 + 2 * g];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    acc0[4 * g + c] = fmaf(acc0[4 * g + c], s0[c], q.sum * m0[c]);
                    acc1[4 * g + c] = fmaf(acc1[4 * g + c], s1[c], q.sum * m1[c]);
                }
            }
        }
        if (st < clean0 || st >= clean1) {
            const int32_t kb = steps.first_key(st);
            const uint32_t s0 = seen_keys(a, pos, pos, kb) >> (4 * h), s1 = seen_keys(a, pos, pos, kb + 32) >> (4 * h);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                acc0[e] = s0 >> ((e & 3) + 8 * (e >> 2)) & 1 ? acc0[e] : kNone;
                acc1[e] = s1 >> ((e & 3) + 8 * (e >> 2)) & 1 ? acc1[e] : kNone;
            }
        }
        float best = kNone;
#pragma unroll
        for (int e = 0; e < 16; ++e) best = most(best, most(acc0[e], acc1[e]));
        const float scale = KIND == CI_KV_BF16 ? a.scale_log2 : 1.0f;
        run.raise(max_halves(best) * scale);
        const float base = run.base();
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            float x0 = exp2_fast(acc0[e] * scale - base), x1 = exp2_fast(acc0[e + 1] * scale - base);
            float y0 = exp2_fast(acc1[e] * scale - base), y1 = exp2_fast(acc1[e + 1] * scale - base);
            run.l += (x0 + x1) + (y0 + y1);
            if (KIND != CI_KV_BF16) {  // sum w (mid + step (code - 7.5))
                const int g = e / 4, c = e % 4;
                const f32x4_p s0 = of[32 + 2 * g], s1 = of[40 + 2 * g], m0 = of[48 + 2 * g], m1 = of[56 + 2 * g];
                run.off = fmaf(x0, m0[c], fmaf(x1, m0[c + 1], fmaf(y0, m1[c], fmaf(y1, m1[c + 1], run.off))));
                x0 *= s0[c], x1 *= s0[c + 1], y0 *= s1[c], y1 *= s1[c + 1];
            }
            p[e / 8][e / 2 % 4] = bf16_pair(x0, x1);
            p[2 + e / 8][e / 2 % 4] = bf16_pair(y0, y1);
        }
        phase_end();
        // ---- matrix phase (behind the last step: the scores of what lies there, for nothing)
        __builtin_amdgcn_s_setprio(1);
        // (in the order that keeps the matrix unit fed: turning codes into numbers takes the vector unit a while, and runs
        // beside the first half's matrix instructions; copies are best out of the way first.  The other way round: the 4-bit
        // prompt part 1100 instead of 925 us, the bf16 prompt of 8192 tokens 645 instead of 553)
        if (KIND != CI_KV_BF16) output(st);
        put(st + 2);
        ask(st + 3);
        if (KIND == CI_KV_BF16) output(st);
        scores(st + 1);
        __builtin_amdgcn_s_setprio(0);
        phase_end();
    }
    if (u0 < last && !second) phase_end();  // (the second group's last phase)
    if (lost && threadIdx.x == 0) report_bad_index(a.batch);
    const bool mine = r0 + col < t1;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(mine && (lost || run.no_number())) != 0, 0)) {
        // (with steps and sums of its own: taking those above the loop is scheduled worse, 4-bit prompt part 943 instead of 924 us)
        const Steps again = steps_between(a, position_of(a, s, t0), position_of(a, s, t1 - 1));
        Running<D> anew;
        attend_again<KIND, D, 32>(a, seq, s, head, r0, r1, 2 * u0, 2 * min(u1, again.n), 1,
                                  [&](uint32_t k) { return (uint32_t)again.first_key(k / 2) / kKvBlock + k % 2; }, anew);
        run = anew;
    }
    const float l = run.l + other_half(run.l);
    if (KIND != CI_KV_BF16) {
        const float off = run.off + other_half(run.off);
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int k = 0; k < 16; ++k) run.o[db][k] += off;
    }
    if (!whole) {
        if (!mine) return;
        float *o = slot + (r0 - t0 + col) * D;
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const f32x4_p w = {run.o[db][4 * k], run.o[db][4 * k + 1], run.o[db][4 * k + 2], run.o[db][4 * k + 3]};
                *reinterpret_cast<f32x4_p *>(o + 32 * db + 8 * k + 4 * h) = w;
            }
        if (h == 0) {
            slot[kTileRows * D + r0 - t0 + col] = run.m;
            slot[kTileRows * (D + 1) + r0 - t0 + col] = l;
        }
        return;
    }
    if (mine) {
        const float inv = inverse_sum(a, seq, s, r0 + col, l);
        const uint32_t tok = token_of(a, r0 + col), gh = head * a.group + r0 + col - tok * a.group;
        uint16_t *dst = a.out + (int64_t)(s.row + (int32_t)tok) * a.o_row + (int64_t)gh * a.o_head;
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float y[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) y[c] = run.o[db][4 * k + c] * inv;
                u32x2 w = {bf16_pair(y[0], y[1]), bf16_pair(y[2], y[3])};
                *reinterpret_cast<u32x2 *>(dst + 32 * db + 8 * k + 4 * h) = w;
            }
        if (a.lse && h == 0)
            a.lse[(int64_t)(s.row + (int32_t)tok) * a.l_row + gh] = run.m == kNone ? kNone : (run.m + log2f(l)) * 0.6931471805599453f;
    }
}

template <int KIND, int D>
__global__ __launch_bounds__(kRowThreads, 2 * row_groups(KIND, D)) void attend_rows_kernel(AttendArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    uint32_t *word = reinterpret_cast<uint32_t *>(lds);
    // Workgroups go to the eight XCDs in turn, and each has an L2 of its own: an XCD takes a contiguous run of the list, so
    // that the tiles of a head read its keys and values through one L2.
    Found f;
    bool bad;
    if (a.whole) {  // one tile each, those with the most keys of a head first
        const auto items = [&](uint32_t i) { return tiles_in(a, load_seq_in_sum(a.batch, a.cache, i)).tiles * a.cache.kv_heads; };
        const auto mine = [&](uint32_t total) {
            const uint32_t run = (total + 7) / 8, k = blockIdx.x >> 3;
            return k < run ? (blockIdx.x & 7) * run + k : 0xFFFFFFFFu;
        };
        if (!locate(a.batch.seqs, items, mine, word, f)) return;
        const SeqInfo s = load_seq(a.batch, a.cache, f.seq, bad);
        if (bad && threadIdx.x == 0) report_bad_index(a.batch);
        const uint32_t tiles = tiles_in(a, s).tiles, head = (f.target - f.begin) / tiles;
        attend_rows_piece<KIND, D>(a, f.seq, s, head, tiles - 1 - (f.target - f.begin) % tiles, 0, 0xFFFFFFFFu, true, nullptr, lds);
        return;
    }
    const uint32_t worker = (blockIdx.x & 7) * (gridDim.x / 8) + (blockIdx.x >> 3);
    const auto weight = [&](uint32_t i) { return tiles_in(a, load_seq_in_sum(a.batch, a.cache, i)).head * a.cache.kv_heads; };
    if (!locate(a.batch.seqs, weight, [&](uint32_t total) { return worker * RowShare(total, gridDim.x).share; }, word, f)) return;
    const RowShare cuts(f.total, gridDim.x);
    uint32_t seq = f.seq, base = f.begin;  // of the list, where the sequence begins
    const uint32_t end = min(f.target + cuts.share, f.total);
    SeqInfo s = load_seq(a.batch, a.cache, seq, bad);
    TileList list = tiles_in(a, s);
    uint32_t place = f.target - base;
    bool begins = true;  // the first tile: the cut before this workgroup
    for (;;) {
        if (bad && threadIdx.x == 0) report_bad_index(a.batch);
        const uint32_t head = place / list.head;
        const TilePlace t = tile_at(a, s, list, place - head * list.head);
        const uint32_t at = base + head * list.head + t.begin;  // where the tile begins in the list
        if (at >= end) return;
        const uint32_t u0 = begins ? cuts.cut(f.target - at, t.places) : 0;
        const uint32_t u1 = end - at >= t.places ? t.places : cuts.cut(end - at, t.places);
        begins = false;
        if (u0 < u1) {
            // a tile that goes on from the workgroup before leaves its sums in slot 0, one that goes on in the next in slot 1
            float *slot = a.work + (uint64_t)(worker * 2 + (u0 == 0 ? 1 : 0)) * (kTileRows * (D + 2));
            attend_rows_piece<KIND, D>(a, seq, s, head, t.tile, u0, u1, u0 == 0 && u1 == t.places, slot, lds);
        }
        place = head * list.head + t.begin + t.places;
        if (place < list.head * a.cache.kv_heads) continue;
        base += place;
        place = 0;
        do {
            if (++seq >= a.batch.seqs) return;
            s = load_seq(a.batch, a.cache, seq, bad);
            list = tiles_in(a, s);
        } while (list.head == 0);
    }
}

// 32 rows of the tile that the cut before workgroup blockIdx.x + 1 goes through: the sum of its parts.
template <int KIND, int D>
__global__ __launch_bounds__(256) void attend_rows_join_kernel(AttendArgs a, uint32_t workers) {
    __shared__ uint32_t word[10];
    const uint32_t k = blockIdx.x + 1;
    Found f;
    const auto weight = [&](uint32_t i) { return tiles_in(a, load_seq_in_sum(a.batch, a.cache, i)).head * a.cache.kv_heads; };
    if (!locate(a.batch.seqs, weight, [&](uint32_t total) { return k * RowShare(total, workers).share; }, word, f)) return;
    const RowShare cuts(f.total, workers);
    bool bad;
    const SeqInfo s = load_seq(a.batch, a.cache, f.seq, bad);
    const TileList list = tiles_in(a, s);
    const uint32_t place = f.target - f.begin, head = place / list.head;
    const TilePlace t = tile_at(a, s, list, place - head * list.head);
    const uint32_t at = f.begin + head * list.head + t.begin, off = f.target - at;
    const uint32_t moved = cuts.cut(off, t.places);
    if (moved == 0 || moved == t.places) return;                                      // not cut here
    if (off > cuts.share && cuts.cut(off - cuts.share, t.places) != 0) return;  // cut before: joined there
    const uint32_t t0 = t.tile * kTileRows, r0 = t0 + blockIdx.y * 32, r1 = min(r0 + 32, rows_of(a, s));
    if (r0 >= r1) return;
    const uint32_t w0 = k - 1;
    uint32_t w1 = (at + t.places - 1) / cuts.share;
    if (w1 > k && cuts.cut(w1 * cuts.share - at, t.places) == t.places) --w1;
    constexpr uint32_t kLanes = D / 4;
    const uint32_t d = threadIdx.x % kLanes * 4;
    for (uint32_t r = r0 + threadIdx.x / kLanes; r < r1; r += 256 / kLanes) {
        float m = kNone, l = 0.0f;
        f32x4_p acc = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t w = w0; w <= w1; ++w) {
            const float *slot = a.work + (uint64_t)(w * 2 + (w == w0 ? 1 : 0)) * (kTileRows * (D + 2));
            const float mw = slot[kTileRows * D + r - t0], lw = slot[kTileRows * (D + 1) + r - t0];
            const f32x4_p y = *reinterpret_cast<const f32x4_p *>(slot + (r - t0) * D + d);
            const float top = fmaxf(m, mw), f0 = m == kNone ? 0.0f : exp2_fast(m - top), f1 = mw == kNone ? 0.0f : exp2_fast(mw - top);
            l = l * f0 + lw * f1;
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = acc[c] * f0 + y[c] * f1;
            m = top;
        }
        const float inv = inverse_sum(a, f.seq, s, r, l);
        const uint32_t tok = token_of(a, r), gh = head * a.group + r - tok * a.group;
        u32x2 w = {bf16_pair(acc[0] * inv, acc[1] * inv), bf16_pair(acc[2] * inv, acc[3] * inv)};
        *reinterpret_cast<u32x2 *>(a.out + (int64_t)(s.row + (int32_t)tok) * a.o_row + (int64_t)gh * a.o_head + d) = w;
        if (a.lse && d == 0)
            a.lse[(int64_t)(s.row + (int32_t)tok) * a.l_row + gh] = m == kNone ? kNone : (m + log2f(l)) * 0.6931471805599453f;
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
struct AttendPlan {
    bool many;         // attend_rows_kernel
    bool whole;        // split kernel, one workgroup per item
    uint32_t rp, grid, items, workers;
    size_t work_bytes;
};

// `longest`, `new_longest`: the caller's bounds on the lengths.  They choose kernels; the results do not rest on them.
static int plan_attend(const KvView &v, const KvBatch &b, uint32_t kind, uint32_t head_dim, uint32_t group, int32_t window, int32_t sinks,
                       uint32_t new_longest, uint32_t longest, AttendPlan *p) {
    uint32_t cus = 1;
    if (int rc = cu_count(&cus)) return rc;
    const uint64_t rows = (uint64_t)b.tokens * group;
    const uint64_t per_seq = (uint64_t)(b.start ? new_longest : 1) * group;
    // Measured with few | many rows' kernel, 32 heads over 8 of 128 in bf16: 512 tokens from the first on 29 | 28 us, 1024 557 |
    // 41; 64 tokens behind 8192 41 | 67; 16 times 16 tokens behind 8192 147 | 151.  In 4 bits: 512 tokens 21 | 39, 1024 563 | 63.
    // The rule does not look at the keys: 256 tokens behind 32768 go to the kernel for few (392 | 168).
    p->many = per_seq >= 64 && rows * v.kv_heads / kTileRows >= cus / 4;
    p->whole = false;
    p->work_bytes = 0;
    p->rp = per_seq <= 4 ? 4 : per_seq <= 8 ? 8 : per_seq <= 16 ? 16 : 32;
    const uint64_t tiles = b.start ? rows / (p->many ? kTileRows : p->rp) + b.seqs : (uint64_t)b.seqs * ceil_div(group, p->rp);
    const uint64_t items = tiles * v.kv_heads;
    if (items > 0x7FFFFF00ull) return fail(CI_ERR_ARG, "ci_paged_attention: too many rows for one call");
    p->items = (uint32_t)items;
    // places in the list of work, at most (an item of few rows goes in units, a tile of many in steps): 32 bits count them
    const uint64_t room = (uint64_t)b.table_width << (v.page_shift + 5);
    if (room / (p->many ? kStep : kUnit * kKvBlock) + 2 > 0xFF000000ull / (items ? items : 1))
        return fail(CI_ERR_ARG, "ci_paged_attention: too many rows over too long a block table for one call; give the rows in several");
    if (p->many) {
        p->workers = p->grid = (cus * row_groups(kind, head_dim) + 7) / 8 * 8;
        // tiles of few steps: one workgroup each, handed out by the hardware, and nothing to join (ragged prompts of up to 6001
        // tokens under a window of 1000: 152 us in shares, 124 whole; 2 prompts of 2048, 12 heads of 64, 80 and 47, of 4096 110
        // and 131)
        uint64_t keys = longest;
        const uint64_t reach = (uint64_t)window + sinks + kTileRows / group + 3 * kStep;
        if (window && reach < keys) keys = reach;
        p->whole = keys <= kWholeSteps * kStep;
        if (p->whole) p->grid = (p->items + 7) / 8 * 8;
        else p->work_bytes = (size_t)p->workers * 2 * kTileRows * (head_dim + 2) * sizeof(float);
        return CI_OK;
    }
    uint64_t keys = longest;
    if (window && (uint64_t)window + sinks + 64 < keys) keys = (uint64_t)window + sinks + 64;
    // (64 tokens over 512 each: 35 us in shares, 28 whole; over 2048 each 113 and 107, but there a batch of unlike lengths would
    // wait for its longest)
    p->whole = keys <= 4 * kUnit * kKvBlock;
    // as many as are resident (48 ragged chats of up to 32768 tokens in bf16, one to four workgroups per CU: 620, 615, 654, 618
    // us; with heads of 64 329, 283, 278, 306); for 4 bits, where a workgroup waits longer for its first block than it then
    // reads, twice as many if each still has much to do (the same chats 261, 215, 223, 213, with heads of 64 184, 134, 119, 115;
    // 16 over 16384 each, at the border, 68, 56, 77, 64; one document of 65531 would lose, 28 -> 36)
    const uint64_t units = (uint64_t)b.seqs * v.kv_heads * (keys / (kUnit * kKvBlock));
    p->workers = (kind != CI_KV_BF16 && units >= 64ull * cus ? 4 : 2) * cus;
    p->grid = p->whole ? p->items : p->workers;
    if (!p->whole) p->work_bytes = (size_t)p->workers * 2 * p->rp * (head_dim + 2) * sizeof(float);
    return CI_OK;
}

template <int KIND, int D, int RP>
static int launch_split(const AttendArgs &a, const AttendPlan &p, hipStream_t s) {
    CI_ALLOW_FULL_LDS((attend_split_kernel<KIND, D, RP>));
    CI_KV_LAUNCH((attend_split_kernel<KIND, D, RP>), dim3(p.grid), dim3(256), split_lds(D), s, a);
    CI_LAUNCH_CHECK("attend_split_kernel");
    if (!p.whole) {
        CI_KV_LAUNCH((attend_join_kernel<KIND, D, RP>), dim3(p.items, RP), dim3(256), 0, s, a, p.workers);
        CI_LAUNCH_CHECK("attend_join_kernel");
    }
    return CI_OK;
}

template <int KIND, int D>
static int launch_attend(const AttendArgs &a, const AttendPlan &p, hipStream_t s) {
    if (p.many) {
        CI_ALLOW_FULL_LDS((attend_rows_kernel<KIND, D>));
        CI_KV_LAUNCH((attend_rows_kernel<KIND, D>), dim3(p.grid), dim3(kRowThreads), rows_lds(KIND, D), s, a);
        CI_LAUNCH_CHECK("attend_rows_kernel");
        if (!p.whole && p.workers > 1) {
            CI_KV_LAUNCH((attend_rows_join_kernel<KIND, D>), dim3(p.workers - 1, kTileRows / 32), dim3(256), 0, s, a, p.workers);
            CI_LAUNCH_CHECK("attend_rows_join_kernel");
        }
        return CI_OK;
    }
    switch (p.rp) {
        case 4: return launch_split<KIND, D, 4>(a, p, s);
        case 8: return launch_split<KIND, D, 8>(a, p, s);
        case 16: return launch_split<KIND, D, 16>(a, p, s);
        default: return launch_split<KIND, D, 32>(a, p, s);
    }
}

static int check_attend(const char *who, const ci_kv_cache *cache, const ci_kv_batch *batch, uint32_t q_heads, int32_t window,
                        int32_t sinks, KvView *v, KvBatch *b) {
    if (int rc = check_kv_cache(who, cache, v)) return rc;
    if (int rc = check_kv_batch(who, batch, *v, b)) return rc;
    if (q_heads == 0 || q_heads % v->kv_heads || q_heads > 65536)
        return fail(CI_ERR_ARG, "%s: q_heads must be a multiple of kv_heads", who);
    if (window < 0 || sinks < 0) return fail(CI_ERR_ARG, "%s: window and sinks must not be negative", who);
    if ((uint64_t)b->tokens * (q_heads / v->kv_heads) > 0x7FFFFF00ull)
        return fail(CI_ERR_ARG, "%s: too many rows for one call", who);
    return CI_OK;
}

}  // namespace ci

using namespace ci;

extern "C" size_t ci_paged_attention_workspace_bytes(const ci_kv_cache *cache, const ci_kv_batch *batch, uint32_t q_heads,
                                                     int32_t window, int32_t sinks, uint32_t max_query_len,
                                                     uint32_t max_seq_len) {
    KvView v;
    KvBatch b;
    AttendPlan p;
    if (check_attend("ci_paged_attention_workspace_bytes", cache, batch, q_heads, window, sinks, &v, &b)) return 0;
    if (b.seqs == 0 || b.tokens == 0) return 0;
    if (plan_attend(v, b, cache->kind, cache->head_dim, q_heads / v.kv_heads, window, sinks, max_query_len ? max_query_len : b.tokens,
                    max_seq_len ? max_seq_len : b.table_width << (v.page_shift + 5), &p))
        return 0;
    return p.work_bytes;
}

extern "C" int ci_paged_attention(const ci_kv_cache *cache, const ci_kv_batch *batch, const ci_rows *q, const ci_rows *out,
                                  float *d_lse, int64_t lse_stride, uint32_t q_heads, float scale, int32_t window,
                                  int32_t sinks, uint32_t max_query_len, uint32_t max_seq_len, void *d_workspace,
                                  size_t workspace_bytes, ci_stream_t stream) {
    static const char *who = "ci_paged_attention";
    AttendArgs a{};
    if (int rc = check_attend(who, cache, batch, q_heads, window, sinks, &a.cache, &a.batch)) return rc;
    if (!q || !out) return fail(CI_ERR_ARG, "%s: null q or out", who);
    if (!(scale > 0.0f) || !(scale < 1e30f)) return fail(CI_ERR_ARG, "%s: scale must be positive and finite", who);
    if (a.batch.seqs == 0 || a.batch.tokens == 0) return CI_OK;
    for (const ci_rows *r : {q, out}) {
        if (!r->d_data || !aligned(r->d_data, 16) || r->row_stride % 8 || r->head_stride % 8 || r->row_stride < 0 || r->head_stride < 0)
            return fail(CI_ERR_ARG, "%s: %s must be a 16-byte aligned device pointer with strides that are non-negative multiples of 8",
                        who, r == q ? "q" : "out");
    }
    if (rows_may_overlap(*q, q_heads, *out, q_heads, a.batch.tokens, cache->head_dim))  // (a row may be done a second time)
        return fail(CI_ERR_ARG, "%s: out must share no memory with q", who);
    a.q = static_cast<const uint16_t *>(q->d_data);
    a.out = static_cast<uint16_t *>(out->d_data);
    a.lse = d_lse;
    a.l_row = lse_stride;
    a.q_row = q->row_stride, a.q_head = q->head_stride, a.o_row = out->row_stride, a.o_head = out->head_stride;
    a.group = q_heads / a.cache.kv_heads;
    a.per_group = 1.0 / (double)a.group;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.window = window < (1 << 30) ? window : 1 << 30;  // (no sequence is longer: sums of positions stay in 32 bits)
    a.sinks = sinks < (1 << 30) ? sinks : 1 << 30;
    AttendPlan p;
    if (int rc = plan_attend(a.cache, a.batch, cache->kind, cache->head_dim, a.group, window, sinks, max_query_len ? max_query_len : a.batch.tokens,
                             max_seq_len ? max_seq_len : a.batch.table_width << (a.cache.page_shift + 5), &p))
        return rc;
    if (p.work_bytes && (!d_workspace || !aligned(d_workspace, 16) || workspace_bytes < p.work_bytes))
        return fail(CI_ERR_CAPACITY, "%s: the workspace must be 16-byte aligned and hold %zu bytes", who, p.work_bytes);
    if (int rc = device_status_word(&a.batch.status)) return rc;
    a.work = static_cast<float *>(d_workspace);
    a.whole = p.whole ? 1 : 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool wide = cache->head_dim == 128;
    if (cache->kind == CI_KV_BF16) return wide ? launch_attend<CI_KV_BF16, 128>(a, p, s) : launch_attend<CI_KV_BF16, 64>(a, p, s);
    return wide ? launch_attend<CI_KV_INT4, 128>(a, p, s) : launch_attend<CI_KV_INT4, 64>(a, p, s);
}
