// The paged key/value cache: appending the new tokens of a batch (rotated on the way, optionally held in 4 bits) and
// reading tokens back.  Layout: paged.h.
//
// One workgroup takes the new tokens that fall into one block of 32 of one sequence, and a group of heads: rotated
// queries, or keys and values.  So every word of the cache has one writer per call, also where the 4-bit values of eight
// tokens share a word: such a word is read, the new tokens' codes are put in, and it is written whole -- no atomics, and
// tokens already in the block stay as they are.
//
// All of it is bound by memory: q is read and written once (a thread holds eight channels and their partners half a
// rotation further, sixteen bytes each), keys and values are read once and written in the order attention reads them.
// The rotation is computed in 64 bits, where its products are exact (8 by 24 bits), and rounded to 32 bits and then to bf16:
// whatever the angle, a rotated value is off by half a step of bf16 and 2^-24 of itself.  Measured, 4 prompts of 1001 to 4097
// tokens into 4 bits, 16 heads over 2 of 64: 15.2 us, of which the rotation takes 2.6 (12.6 without a table; a copy moves
// the 51 MB in 10.4); vector units busy 36 % of the time, 28 % without.  7 prompts of 333 to 2100 in bf16, 32 heads over 8 of
// 128: 38 us for 213 MB.
#include "paged.h"

#include <numeric>

namespace ci {

// ---- what a row in 4 bits is ---------------------------------------------------------------------------------------
// low = min, step = (max - min) / 15 rounded UP to bf16 (so that code 15 reaches the maximum), both from the row's exact
// values; code = (x - low) / step rounded to the nearest, ties to even.  Rows that hold an infinity or a NaN get
// low = step = NaN and read back as NaN throughout.
__device__ __forceinline__ uint32_t step_and_low(float low, float high) {
    const double width = (double)high - (double)low;
    // the least bf16 number whose fifteenfold (exact here) is not below the width: the quotient's neighbour, put right
    uint32_t step = (__float_as_uint((float)(width * (1.0 / 15.0))) + 0xFFFFu) >> 16;
    if (step && 15.0 * (double)bf16_lo(step - 1) >= width) --step;
    if (15.0 * (double)bf16_lo(step) < width) ++step;
    return step | (__float_as_uint(low) & 0xFFFF0000u);  // (low is one of the row's bf16 values)
}

// step and low of a row, and how its codes are found.
struct Grid {
    float step, low, inverse;
    bool extreme;  // 1 / step or max - low is outside what 32 bits hold
};

__device__ __forceinline__ Grid grid_of(uint32_t pair) {
    Grid g;
    g.step = bf16_lo(pair);
    g.low = bf16_hi(pair);
    g.extreme = g.step > 0.0f && (g.step < 1e-37f || g.step > 1e37f);
    g.inverse = g.step > 0.0f ? 1.0f / g.step : 0.0f;  // (a constant row, and a row of NaN: code 0)
    return g;
}

__device__ __forceinline__ uint32_t code_of(float x, const Grid &g) {
    float t = (x - g.low) * g.inverse;
    if (g.extreme) t = (float)(((double)x - (double)g.low) / (double)g.step);
    float c = rintf(t);
    // the float quotient, up to 15, is off by at most three roundings (3 x 15 x 2^-24 < 3e-6): only that near to a border can
    // it round wrongly
    if (fabsf(fabsf(t - c) - 0.5f) < 4e-6f || g.extreme) {
        const double r = ((double)x - (double)g.low) - (double)c * (double)g.step, half = 0.5 * (double)g.step;
        const bool odd = ((int)c & 1) != 0;
        if (r > half || (r == half && odd)) c += 1.0f;
        if (r < -half || (r == -half && odd)) c -= 1.0f;
    }
    return (uint32_t)fminf(fmaxf(c, 0.0f), 15.0f);  // (a NaN becomes 0; its row reads back as NaN through low)
}

struct AppendArgs {
    KvView cache;
    KvBatch batch;
    const uint16_t *q, *k, *v;
    uint16_t *q_out;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;  // strides in elements
    uint32_t q_heads, q_group, kv_group;                                  // heads per workgroup
    uint32_t kv_parts;                                                    // workgroups in y that take keys and values
    const float *rotary;
    uint32_t rotary_rows, rotary_dim;
};

// The new tokens of one sequence that fall into one block.
struct Tile {
    uint32_t seq, blk, page;
    int32_t row;   // row of q / k / v of the tile's first token
    uint32_t t0;   // its place in the block
    uint32_t n;    // tokens of the tile; 0: nothing to do
    int32_t pos;   // its position
    bool bad;
};

__device__ __forceinline__ uint32_t tiles_of(const SeqInfo &s) {
    const int32_t first = max(s.len - s.n, 0);
    return s.len > first ? (uint32_t)((s.len - 1) / (int32_t)kKvBlock - first / (int32_t)kKvBlock + 1) : 0;
}

__device__ __forceinline__ Tile find_tile(const KvBatch &b, const KvView &v, uint32_t index, uint32_t *word) {
    Tile t{};
    uint32_t seq = index, begin = index;
    bool bad = false;
    if (b.start) {
        Found f;
        if (!locate(b.seqs, [&](uint32_t i) { return tiles_of(load_seq_in_sum(b, v, i)); }, [&](uint32_t) { return index; }, word, f)) return t;
        seq = f.seq;
        begin = f.begin;
    }
    const SeqInfo s = load_seq(b, v, seq, bad);
    const int32_t first = max(s.len - s.n, 0);
    t.bad = bad;
    t.seq = seq;
    if (s.len <= first) return t;
    t.blk = (uint32_t)first / kKvBlock + (index - begin);
    const int32_t lo = max(first, (int32_t)(t.blk * kKvBlock)), hi = min(s.len, (int32_t)((t.blk + 1) * kKvBlock));
    t.page = page_of(b, v, seq, t.blk);
    if (t.page == kNoPage) t.bad = true;
    t.row = s.row + s.n - (s.len - lo);
    t.t0 = (uint32_t)lo % kKvBlock;
    t.pos = lo;
    t.n = hi > lo ? (uint32_t)(hi - lo) : 0;
    return t;
}

struct Pair8 {
    u32x4 a, b;
};

// Channels [a, a + 8) and [b, b + 8) of one row, b = a + rotary_dim / 2, turned by the angles of position `pos`.
__device__ __forceinline__ Pair8 rotate8(Pair8 x, const float *__restrict__ row, uint32_t a, uint32_t half) {
    const f32x4_p *c4 = reinterpret_cast<const f32x4_p *>(row + a), *s4 = reinterpret_cast<const f32x4_p *>(row + half + a);
    Pair8 y;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        float o[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const double c = c4[w / 2][2 * (w & 1) + i], s = s4[w / 2][2 * (w & 1) + i];
            const double x1 = i ? bf16_hi(x.a[w]) : bf16_lo(x.a[w]), x2 = i ? bf16_hi(x.b[w]) : bf16_lo(x.b[w]);
            o[i] = (float)(x1 * c - x2 * s);
            o[2 + i] = (float)(x2 * c + x1 * s);
        }
        y.a[w] = bf16_pair(o[0], o[1]);
        y.b[w] = bf16_pair(o[2], o[3]);
    }
    return y;
}

__device__ __forceinline__ float min8(u32x4 x) {
    float m = bf16_lo(x[0]);
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fminf(m, fminf(bf16_lo(x[w]), bf16_hi(x[w])));
    return m;
}
__device__ __forceinline__ float max8(u32x4 x) {
    float m = bf16_lo(x[0]);
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, fmaxf(bf16_lo(x[w]), bf16_hi(x[w])));
    return m;
}
// Whether one of the eight is an infinity or a NaN (min and max skip a NaN).
__device__ __forceinline__ bool wild8(u32x4 x) {
    bool any = false;
#pragma unroll
    for (int w = 0; w < 4; ++w)
        any = any || (x[w] & 0x7F80u) == 0x7F80u || (x[w] & 0x7F800000u) == 0x7F800000u;
    return any;
}
__device__ __forceinline__ uint32_t codes8(u32x4 x, const Grid &g) {
    uint32_t word = 0;
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) {
        const float f = (e & 1) ? bf16_hi(x[e / 2]) : bf16_lo(x[e / 2]);
        word |= code_of(f, g) << nibble_shift(e);
    }
    return word;
}

// The value of a neighbour in a row's threads: the other of a pair, of two pairs in four, of two fours in eight (in
// which, by then, all of a four hold the same).
template <int CTRL>
__device__ __forceinline__ float neighbour(float x) {
    const int v = __float_as_int(x);
    return __int_as_float(__builtin_amdgcn_update_dpp(v, v, CTRL, 15, 15, false));
}

// min and max over the D / 16 neighbouring threads that share a row; (step, low) of the row.  Both carry a NaN (an infinity is
// made one).
template <int D>
__device__ __forceinline__ uint32_t row_pair(u32x4 a, u32x4 b) {
    const float wild = wild8(a) || wild8(b) ? __builtin_nanf("") : 0.0f;
    float lo = fminf(min8(a), min8(b)) + wild, hi = fmaxf(max8(a), max8(b)) + wild;
    lo = __builtin_elementwise_minimum(lo, neighbour<0xB1>(lo));
    hi = __builtin_elementwise_maximum(hi, neighbour<0xB1>(hi));
    lo = __builtin_elementwise_minimum(lo, neighbour<0x4E>(lo));
    hi = __builtin_elementwise_maximum(hi, neighbour<0x4E>(hi));
    if (D == 128) {
        lo = __builtin_elementwise_minimum(lo, neighbour<0x141>(lo));
        hi = __builtin_elementwise_maximum(hi, neighbour<0x141>(hi));
    }
    return lo != lo ? 0x7FC07FC0u : step_and_low(lo, hi);
}

template <int KIND, int D>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs p) {
    __shared__ uint32_t word[10];
    __shared__ uint32_t codes[256 / (D / 16) * D / 8];  // 4 bits: the values' codes of the rows in hand
    constexpr uint32_t kSlots = D / 16, kRows = 256 / kSlots;
    const Tile t = find_tile(p.batch, p.cache, blockIdx.x, word);
    const bool keys = blockIdx.y < p.kv_parts;
    if (t.bad && threadIdx.x == 0 && blockIdx.y == 0) report_bad_index(p.batch);
    if (t.n == 0 || t.page == kNoPage) return;
    const uint32_t slot = threadIdx.x % kSlots, my_row = threadIdx.x / kSlots;
    const uint32_t half = p.rotary_dim / 2;
    const bool turns = p.rotary && slot < p.rotary_dim / 16;
    const uint32_t a = !p.rotary ? 16 * slot : turns ? 8 * slot : p.rotary_dim + 16 * (slot - p.rotary_dim / 16);
    const uint32_t b = turns ? a + half : a + 8;

    if (!keys) {  // queries
        const uint32_t h0 = (blockIdx.y - p.kv_parts) * p.q_group, nh = min(p.q_group, p.q_heads - h0);
        for (uint32_t r = my_row; r < nh * t.n; r += kRows) {
            const uint32_t tok = r / nh, head = h0 + r % nh;
            const uint32_t pos = (uint32_t)t.pos + tok;
            if (p.rotary && pos >= p.rotary_rows) {
                if (slot == 0) report_bad_index(p.batch);
                continue;
            }
            const uint16_t *src = p.q + (int64_t)(t.row + (int32_t)tok) * p.q_row + (int64_t)head * p.q_head;
            uint16_t *dst = p.q_out + (int64_t)(t.row + (int32_t)tok) * p.o_row + (int64_t)head * p.o_head;
            Pair8 x = {*reinterpret_cast<const u32x4 *>(src + a), *reinterpret_cast<const u32x4 *>(src + b)};
            if (turns) x = rotate8(x, p.rotary + (uint64_t)pos * p.rotary_dim, a, half);
            *reinterpret_cast<u32x4 *>(dst + a) = x.a;
            *reinterpret_cast<u32x4 *>(dst + b) = x.b;
        }
        return;
    }

    // (head, token) rows: at most kRows of them (a workgroup takes the tokens of one head, or many heads of one token)
    const uint32_t h0 = blockIdx.y * p.kv_group, nh = min(p.kv_group, p.cache.kv_heads - h0);
    const bool mine = my_row < nh * t.n;
    const uint32_t head = h0 + (mine ? my_row / t.n : 0), tok = mine ? my_row % t.n : 0;
    const uint32_t pos = (uint32_t)t.pos + tok, at = t.t0 + tok;
    uint8_t *block = block_at<KIND, D>(p.cache, t.page, head, t.blk);
    const bool store = mine && !(p.rotary && pos >= p.rotary_rows);
    if (mine && !store && slot == 0) report_bad_index(p.batch);
    // (threads without a row of their own go along with the first one)
    const uint16_t *ksrc = p.k + (int64_t)(t.row + (int32_t)tok) * p.k_row + (int64_t)head * p.k_head;
    Pair8 x = {*reinterpret_cast<const u32x4 *>(ksrc + a), *reinterpret_cast<const u32x4 *>(ksrc + b)};
    if (turns) x = rotate8(x, p.rotary + (uint64_t)min(pos, p.rotary_rows - 1) * p.rotary_dim, a, half);
    if (KIND == CI_KV_BF16) {
        if (store) {
            u32x4 *dst = reinterpret_cast<u32x4 *>(block);
            dst[key_operand(a / 8, at)] = x.a;
            dst[key_operand(b / 8, at)] = x.b;
        }
    } else {
        const uint16_t *src = p.v + (int64_t)(t.row + (int32_t)tok) * p.v_row + (int64_t)head * p.v_head + 16 * slot;
        const Pair8 y = {*reinterpret_cast<const u32x4 *>(src), *reinterpret_cast<const u32x4 *>(src + 8)};
        const uint32_t kpair = row_pair<D>(x.a, x.b), vpair = row_pair<D>(y.a, y.b);
        if (store) {
            uint32_t *dst = reinterpret_cast<uint32_t *>(block), *pairs = reinterpret_cast<uint32_t *>(block + KvBlock<KIND, D>::kPairs);
            const Grid kg = grid_of(kpair), vg = grid_of(vpair);
            dst[key_word(a / 8, at)] = codes8(x.a, kg);
            dst[key_word(b / 8, at)] = codes8(x.b, kg);
            if (slot == 0) pairs[at] = kpair, pairs[kKvBlock + at] = vpair;
            // the values' codes go through the LDS, eight to a word per row, to be gathered by channel
            codes[my_row * (D / 8) + 2 * slot] = codes8(y.a, vg);
            codes[my_row * (D / 8) + 2 * slot + 1] = codes8(y.b, vg);
        }
        __syncthreads();
    }
    // Values, operand by operand: (head, channel, the eight tokens of (s, h)); one new token touches one (s, h) only.
    const bool single = t.n == 1;
    const uint32_t only = (t.t0 >> 4) * 2 + ((t.t0 >> 2) & 1);
    for (uint32_t i = threadIdx.x; i < nh * (single ? 1 : 4) * D; i += 256) {
        const uint32_t hd = single ? i / D : i / (4 * D), d = i % D, sh = single ? only : i / D % 4, s = sh >> 1, h = sh & 1;
        uint8_t *vals = block_at<KIND, D>(p.cache, t.page, h0 + hd, t.blk) + KvBlock<KIND, D>::kHalf;
        const uint32_t o = value_operand<D>(d, 16 * s + 4 * h);
        const uint16_t *src = p.v + (int64_t)t.row * p.v_row + (int64_t)(h0 + hd) * p.v_head + d;
        uint32_t fresh = 0;  // the operand's elements that are new tokens
        uint32_t got[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            const uint32_t tok_e = value_token(s, h, e) - t.t0;
            got[e] = 0;
            if (tok_e < t.n && !(p.rotary && (uint32_t)t.pos + tok_e >= p.rotary_rows)) {
                fresh |= 1u << e;
                if (KIND == CI_KV_BF16)
                    got[e] = src[(int64_t)tok_e * p.v_row];
                else
                    got[e] = codes[(hd * t.n + tok_e) * (D / 8) + d / 8] >> nibble_shift(d & 7) & 15u;
            }
        }
        if (!fresh) continue;
        if (KIND == CI_KV_BF16) {
            uint16_t *dst = reinterpret_cast<uint16_t *>(vals) + o * 8;
            if (fresh == 255) {
                u32x4 w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = got[2 * j] | got[2 * j + 1] << 16;
                *reinterpret_cast<u32x4 *>(dst) = w;
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e)
                    if (fresh >> e & 1) dst[e] = (uint16_t)got[e];
            }
        } else {
            uint32_t *dst = reinterpret_cast<uint32_t *>(vals) + value_word(o);
            uint32_t w = fresh == 255 ? 0 : *dst;
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e)
                if (fresh >> e & 1) w = (w & ~(15u << nibble_shift(e))) | got[e] << nibble_shift(e);
            *dst = w;
        }
    }
}

// ---- reading back ---------------------------------------------------------------------------------------------------
struct ReadArgs {
    KvView cache;
    KvBatch batch;
    uint16_t *k, *v;
    int64_t k_row, k_head, v_row, v_head;
    uint32_t kv_group;
};

// Keys and values of the last n tokens of every sequence as rows again; a stored 4-bit value stands for low + code * step
// (rounded once to 32 bits, then to bf16).  A value's channels are gathered by loads of two bytes (a word in 4 bits), sixteen
// bytes apart, which is what bounds it: 70 MB of bf16 in 25 us, where a copy takes 14; 6.7 MB of 4 bits in 6.
template <int KIND, int D>
__global__ __launch_bounds__(256) void kv_read_kernel(ReadArgs p) {
    __shared__ uint32_t word[10];
    constexpr uint32_t kSlots = D / 8;
    const Tile t = find_tile(p.batch, p.cache, blockIdx.x, word);
    if (t.bad && threadIdx.x == 0 && blockIdx.y == 0) report_bad_index(p.batch);
    if (t.n == 0 || t.page == kNoPage) return;
    const uint32_t h0 = blockIdx.y * p.kv_group, nh = min(p.kv_group, p.cache.kv_heads - h0);
    for (uint32_t i = threadIdx.x; i < nh * t.n * kSlots; i += 256) {
        const uint32_t c = i % kSlots, head = h0 + i / kSlots % nh, tok = i / kSlots / nh, at = t.t0 + tok;
        const uint8_t *block = block_at<KIND, D>(p.cache, t.page, head, t.blk);
        u32x4 k, v;
        if (KIND == CI_KV_BF16) {
            k = reinterpret_cast<const u32x4 *>(block)[key_operand(c, at)];
            const uint16_t *vals = reinterpret_cast<const uint16_t *>(block + KvBlock<KIND, D>::kHalf);
            const uint32_t o = value_operand<D>(8 * c, at), e = value_element(at);
#pragma unroll
            for (int w = 0; w < 4; ++w)
                v[w] = (uint32_t)vals[(o + 2 * w) * 8 + e] | (uint32_t)vals[(o + 2 * w + 1) * 8 + e] << 16;
        } else {
            const uint32_t *pairs = reinterpret_cast<const uint32_t *>(block + KvBlock<KIND, D>::kPairs);
            const uint32_t kw = reinterpret_cast<const uint32_t *>(block)[key_word(c, at)];
            const uint32_t *vals = reinterpret_cast<const uint32_t *>(block + KvBlock<KIND, D>::kHalf);
            const uint32_t kp = pairs[at], vp = pairs[kKvBlock + at];
            const uint32_t o = value_operand<D>(8 * c, at), sh = nibble_shift(value_element(at));
#pragma unroll
            for (uint32_t w = 0; w < 4; ++w) {
                float f[4];
#pragma unroll
                for (uint32_t i2 = 0; i2 < 2; ++i2) {
                    const float ck = (float)(kw >> nibble_shift(2 * w + i2) & 15u);
                    const float cv = (float)(vals[value_word(o + 2 * w + i2)] >> sh & 15u);
                    f[i2] = fmaf(ck, bf16_lo(kp), bf16_hi(kp));
                    f[2 + i2] = fmaf(cv, bf16_lo(vp), bf16_hi(vp));
                }
                k[w] = bf16_pair(f[0], f[1]);
                v[w] = bf16_pair(f[2], f[3]);
            }
        }
        const int64_t row = t.row + (int32_t)tok;
        *reinterpret_cast<u32x4 *>(p.k + row * p.k_row + (int64_t)head * p.k_head + 8 * c) = k;
        *reinterpret_cast<u32x4 *>(p.v + row * p.v_row + (int64_t)head * p.v_head + 8 * c) = v;
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
static uint32_t block_bytes(uint32_t kind, uint32_t dim) { return kind == CI_KV_BF16 ? 128 * dim : 32 * dim + 256; }

static const char *cache_problem(uint32_t num_pages, uint32_t page_size, uint32_t kv_heads, uint32_t head_dim, uint32_t kind) {
    if (kind != CI_KV_BF16 && kind != CI_KV_INT4) return "kind must be CI_KV_BF16 or CI_KV_INT4";
    if (head_dim != 64 && head_dim != 128) return "head_dim must be 64 or 128";
    if (page_size < kKvBlock || page_size > 4096 || (page_size & (page_size - 1)))
        return "page_size must be a power of two from 32 to 4096";
    if (num_pages == 0 || num_pages > 0x7FFFFFFFu) return "num_pages must be 1 to 2^31 - 1";
    if (kv_heads == 0 || kv_heads > 1024) return "kv_heads must be 1 to 1024";
    return nullptr;
}

int check_kv_cache(const char *who, const ci_kv_cache *c, KvView *v) {
    if (!c) return fail(CI_ERR_ARG, "%s: null cache", who);
    if (const char *what = cache_problem(c->num_pages, c->page_size, c->kv_heads, c->head_dim, c->kind))
        return fail(CI_ERR_ARG, "%s: %s", who, what);
    if (!c->d_data || !aligned(c->d_data, 16)) return fail(CI_ERR_ARG, "%s: cache data must be a 16-byte aligned device pointer", who);
    const uint64_t need = ci_kv_cache_bytes(c->num_pages, c->page_size, c->kv_heads, c->head_dim, c->kind);
    if (c->data_bytes < need)
        return fail(CI_ERR_ARG, "%s: cache data holds %llu bytes, its shape needs %llu", who, (unsigned long long)c->data_bytes,
                    (unsigned long long)need);
    uint32_t shift = 0;
    while ((kKvBlock << shift) < c->page_size) ++shift;
    *v = KvView{static_cast<uint8_t *>(c->d_data), c->num_pages, shift, c->kv_heads,
                c->page_size / kKvBlock * block_bytes(c->kind, c->head_dim)};
    return CI_OK;
}

int check_kv_batch(const char *who, const ci_kv_batch *b, const KvView &v, KvBatch *out) {
    if (!b) return fail(CI_ERR_ARG, "%s: null batch", who);
    if (b->num_seqs >= 1u << 30 || b->num_tokens >= 1u << 30)
        return fail(CI_ERR_ARG, "%s: num_seqs and num_tokens must be below 2^30", who);
    if (b->num_seqs && (!b->d_block_table || !b->d_seq_lens)) return fail(CI_ERR_ARG, "%s: null block table or lengths", who);
    if (b->num_seqs && b->table_width == 0) return fail(CI_ERR_ARG, "%s: the block table has no columns", who);
    if (b->num_seqs > 1 && b->table_stride < b->table_width)
        return fail(CI_ERR_ARG, "%s: rows of the block table overlap", who);
    if (((uint64_t)b->table_width << (v.page_shift + 5)) > 1ull << 30)
        return fail(CI_ERR_ARG, "%s: a row of the block table spans more than 2^30 tokens", who);
    if (!b->d_query_start && b->num_tokens != b->num_seqs)
        return fail(CI_ERR_ARG, "%s: without query_start there is one new token per sequence (%u tokens, %u sequences)", who,
                    b->num_tokens, b->num_seqs);
    *out = KvBatch{b->d_block_table, b->table_stride, b->table_width, b->d_seq_lens, b->d_query_start,
                   b->num_seqs,      b->num_tokens,   nullptr};
    return CI_OK;
}

// Whether two row tensors may share an element.  They share none if their extents are apart, if one's rows lie in the gaps
// between the other's (slices of [tokens, heads, dim] along heads), or if the heads do (slices of [tokens, heads, 3, dim]).
bool rows_may_overlap(const ci_rows &a, uint32_t a_heads, const ci_rows &b, uint32_t b_heads, uint32_t tokens, uint32_t dim) {
    const auto width = [&](const ci_rows &r, uint32_t heads) { return (int64_t)(heads - 1) * r.head_stride + dim; };
    const int64_t wa = width(a, a_heads), wb = width(b, b_heads), D = dim;
    const int64_t off = ((intptr_t)b.d_data - (intptr_t)a.d_data) / 2;  // (both 16-byte aligned)
    const int64_t rows = tokens - 1;
    if (off >= rows * a.row_stride + wa || -off >= rows * b.row_stride + wb) return false;
    const auto apart = [&](int64_t every, int64_t first, int64_t second) {  // [0, first) and off + [0, second), every so many
        const int64_t at = every ? (off % every + every) % every : 0;
        return every && at >= first && at + second <= every;
    };
    if (rows && a.row_stride == b.row_stride && apart(a.row_stride, wa, wb)) return false;
    int64_t every = 0;
    if (rows) every = std::gcd(a.row_stride, b.row_stride);
    if (a_heads > 1) every = std::gcd(every, a.head_stride);
    if (b_heads > 1) every = std::gcd(every, b.head_stride);
    return !apart(every, D, D);
}

// Workgroups in x: the blocks of 32 that the new tokens of a batch can touch at most (a sequence with n of them touches at
// most n, and at most n / 32 + 2).
static uint32_t tile_bound(const KvBatch &b) {
    if (!b.start) return b.seqs;
    const uint64_t most = (uint64_t)b.tokens / kKvBlock + 2ull * b.seqs;
    return (uint32_t)(most < b.tokens ? most : b.tokens);
}

static int check_rows(const char *who, const char *what, const void *p, int64_t row, int64_t head, uint32_t heads) {
    if (!p || !aligned(p, 16) || row % 8 || head % 8 || row < 0 || (heads > 1 && head < 0))
        return fail(CI_ERR_ARG, "%s: %s must be a 16-byte aligned device pointer with strides that are non-negative multiples of 8", who, what);
    return CI_OK;
}

}  // namespace ci

using namespace ci;

extern "C" uint64_t ci_kv_cache_bytes(uint32_t num_pages, uint32_t page_size, uint32_t kv_heads, uint32_t head_dim, uint32_t kind) {
    if (cache_problem(num_pages, page_size, kv_heads, head_dim, kind)) return 0;
    return (uint64_t)num_pages * kv_heads * (page_size / kKvBlock) * block_bytes(kind, head_dim);
}

extern "C" int ci_paged_kv_append(const ci_kv_cache *cache, const ci_kv_batch *batch, const ci_rows *k, const ci_rows *v,
                                  const ci_rows *q, const ci_rows *q_out, uint32_t q_heads, const float *d_rotary,
                                  uint32_t rotary_rows, uint32_t rotary_dim, ci_stream_t stream) {
    static const char *who = "ci_paged_kv_append";
    AppendArgs a{};
    if (int rc = check_kv_cache(who, cache, &a.cache)) return rc;
    if (int rc = check_kv_batch(who, batch, a.cache, &a.batch)) return rc;
    if (!k || !v) return fail(CI_ERR_ARG, "%s: null keys or values", who);
    if ((q == nullptr) != (q_out == nullptr)) return fail(CI_ERR_ARG, "%s: q and q_out go together", who);
    if (q && (q_heads == 0 || q_heads > 65536)) return fail(CI_ERR_ARG, "%s: q_heads must be 1 to 65536", who);
    if (d_rotary) {
        if (rotary_dim == 0 || rotary_dim % 16 || rotary_dim > cache->head_dim)
            return fail(CI_ERR_ARG, "%s: rotary_dim must be a multiple of 16 up to head_dim", who);
        if (rotary_rows == 0) return fail(CI_ERR_ARG, "%s: the rotary table has no rows", who);
        if (!aligned(d_rotary, 16)) return fail(CI_ERR_ARG, "%s: the rotary table must be 16-byte aligned", who);
    }
    if (a.batch.seqs == 0 || a.batch.tokens == 0) return CI_OK;
    if (int rc = check_rows(who, "k", k->d_data, k->row_stride, k->head_stride, a.cache.kv_heads)) return rc;
    if (int rc = check_rows(who, "v", v->d_data, v->row_stride, v->head_stride, a.cache.kv_heads)) return rc;
    a.k = static_cast<const uint16_t *>(k->d_data);
    a.v = static_cast<const uint16_t *>(v->d_data);
    a.k_row = k->row_stride, a.k_head = k->head_stride, a.v_row = v->row_stride, a.v_head = v->head_stride;
    if (q) {
        if (int rc = check_rows(who, "q", q->d_data, q->row_stride, q->head_stride, q_heads)) return rc;
        if (int rc = check_rows(who, "q_out", q_out->d_data, q_out->row_stride, q_out->head_stride, q_heads)) return rc;
        const bool same = q->d_data == q_out->d_data && q->row_stride == q_out->row_stride && q->head_stride == q_out->head_stride;
        const uint32_t n = a.batch.tokens, dim = cache->head_dim, kv = a.cache.kv_heads;
        if ((!same && rows_may_overlap(*q, q_heads, *q_out, q_heads, n, dim)) || rows_may_overlap(*k, kv, *q_out, q_heads, n, dim) ||
            rows_may_overlap(*v, kv, *q_out, q_heads, n, dim))
            return fail(CI_ERR_ARG, "%s: q_out must be q itself or share no memory with q, k and v", who);
        a.q = static_cast<const uint16_t *>(q->d_data);
        a.q_out = static_cast<uint16_t *>(q_out->d_data);
        a.q_row = q->row_stride, a.q_head = q->head_stride, a.o_row = q_out->row_stride, a.o_head = q_out->head_stride;
        a.q_heads = q_heads;
    }
    if (int rc = device_status_word(&a.batch.status)) return rc;
    a.rotary = d_rotary;
    a.rotary_rows = rotary_rows;
    a.rotary_dim = d_rotary ? rotary_dim : 0;
    // a workgroup handles 32 (64 for heads of 64) rows of one (token, head) each at a time: whole heads of a full tile, or
    // many heads of a single token
    const uint32_t rows = 4096 / cache->head_dim;
    a.kv_group = a.batch.start ? 1 : rows < a.cache.kv_heads ? rows : a.cache.kv_heads;
    a.q_group = a.batch.start ? 4 : rows;
    a.kv_parts = ceil_div(a.cache.kv_heads, a.kv_group);
    const dim3 grid(tile_bound(a.batch), a.kv_parts + (q ? ceil_div(q_heads, a.q_group) : 0));
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool wide = cache->head_dim == 128;
    if (cache->kind == CI_KV_BF16) {
        if (wide) CI_KV_LAUNCH((kv_append_kernel<CI_KV_BF16, 128>), grid, dim3(256), 0, s, a);
        else CI_KV_LAUNCH((kv_append_kernel<CI_KV_BF16, 64>), grid, dim3(256), 0, s, a);
    } else {
        if (wide) CI_KV_LAUNCH((kv_append_kernel<CI_KV_INT4, 128>), grid, dim3(256), 0, s, a);
        else CI_KV_LAUNCH((kv_append_kernel<CI_KV_INT4, 64>), grid, dim3(256), 0, s, a);
    }
    CI_LAUNCH_CHECK("kv_append_kernel");
    return CI_OK;
}

extern "C" int ci_paged_kv_read(const ci_kv_cache *cache, const ci_kv_batch *batch, const ci_rows *k, const ci_rows *v,
                                ci_stream_t stream) {
    static const char *who = "ci_paged_kv_read";
    ReadArgs a{};
    if (int rc = check_kv_cache(who, cache, &a.cache)) return rc;
    if (int rc = check_kv_batch(who, batch, a.cache, &a.batch)) return rc;
    if (!k || !v) return fail(CI_ERR_ARG, "%s: null keys or values", who);
    if (a.batch.seqs == 0 || a.batch.tokens == 0) return CI_OK;
    if (int rc = check_rows(who, "k", k->d_data, k->row_stride, k->head_stride, a.cache.kv_heads)) return rc;
    if (int rc = check_rows(who, "v", v->d_data, v->row_stride, v->head_stride, a.cache.kv_heads)) return rc;
    if (rows_may_overlap(*k, a.cache.kv_heads, *v, a.cache.kv_heads, a.batch.tokens, cache->head_dim))
        return fail(CI_ERR_ARG, "%s: k and v must not share memory", who);
    a.k = static_cast<uint16_t *>(k->d_data);
    a.v = static_cast<uint16_t *>(v->d_data);
    a.k_row = k->row_stride, a.k_head = k->head_stride, a.v_row = v->row_stride, a.v_head = v->head_stride;
    if (int rc = device_status_word(&a.batch.status)) return rc;
    a.kv_group = a.batch.start ? 1 : 16;
    const dim3 grid(tile_bound(a.batch), ceil_div(a.cache.kv_heads, a.kv_group));
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool wide = cache->head_dim == 128;
    if (cache->kind == CI_KV_BF16) {
        if (wide) CI_KV_LAUNCH((kv_read_kernel<CI_KV_BF16, 128>), grid, dim3(256), 0, s, a);
        else CI_KV_LAUNCH((kv_read_kernel<CI_KV_BF16, 64>), grid, dim3(256), 0, s, a);
    } else {
        if (wide) CI_KV_LAUNCH((kv_read_kernel<CI_KV_INT4, 128>), grid, dim3(256), 0, s, a);
        else CI_KV_LAUNCH((kv_read_kernel<CI_KV_INT4, 64>), grid, dim3(256), 0, s, a);
    }
    CI_LAUNCH_CHECK("kv_read_kernel");
    return CI_OK;
}
