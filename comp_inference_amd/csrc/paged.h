// The paged key/value cache: where a token's key and value lie, and how a batch of sequences is read.
//
// A page holds page_size tokens of every kv head; inside it the tokens of one head lie in blocks of 32, and a block
// holds its keys and values in the order in which the matrix instruction takes them, so that attention loads its
// operands with whole-wavefront 16-byte loads and neither shuffles nor stages anything on the way:
//
//   v_mfma_f32_32x32x16_bf16 computes C[32 x 32] += A[32 x 16] B[16 x 32]; lane l holds row l % 32 of A (column l % 32
//   of B), elements k = 8 (l / 32) .. + 7, and of C column l % 32, rows (r & 3) + 8 (r >> 2) + 4 (l / 32), r = 0..15.
//
//   scores   S^T[key, query] = K Q^T: operand i (16 channels each) of lane l is key l % 32, channels 16 i + 8 (l / 32) ..
//            -> keys lie as [D/16][2][32 keys][8 channels]
//   output   O^T[channel, query] = V^T P^T: the lane that holds column q of S^T holds, in r order, exactly the keys
//            16 s + 8 a + 4 h + b (h = l / 32; s, a = 0, 1; b = 0..3).  The sum over keys may run in any order as long as
//            both operands agree, so these are the keys operand s of the lane takes: P never leaves its lane, and
//            -> values lie as [2 (s)][D/32][2 (h)][32 channels][8 (a, b)]
//
// bf16:   keys 64 D bytes, then values 64 D bytes.
// 4 bits: the same operands in codes, eight to a 32-bit word (element e of an operand in bits 4 (e / 2) + 16 (e % 2), so
//         that one shift and one and-or give two bf16 numbers), the words a lane needs one after the other side by side:
//         keys [D/64][64 lanes][4 words], values [D/64][64 lanes][4 words], then per key and per value the bf16 pair
//         (step, low): 32 words each.
#pragma once
#include "ci_common.h"
#include "rans_device.h"

namespace ci {

constexpr uint32_t kKvBlock = 32;  // tokens of a block
constexpr uint32_t kNoPage = 0xFFFFFFFFu;

typedef __bf16 bf16x8_p __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_p __attribute__((ext_vector_type(2)));
typedef float f32x2_p __attribute__((ext_vector_type(2)));
typedef float f32x4_p __attribute__((ext_vector_type(4)));
typedef float f32x16_p __attribute__((ext_vector_type(16)));

template <int KIND, int D>
struct KvBlock {
    static constexpr uint32_t kHalf = KIND == CI_KV_BF16 ? 64 * D : 16 * D;  // bytes of the keys (or values) of a block
    static constexpr uint32_t kPairs = 2 * kHalf;                            // offset of the (step, low) pairs, 4 bits only
    static constexpr uint32_t kBytes = 2 * kHalf + (KIND == CI_KV_BF16 ? 0 : 256);
};

// Offset in 8-element operands of the key operand that holds channels 8 c .. 8 c + 7 of token t of a block.
__device__ __forceinline__ uint32_t key_operand(uint32_t c, uint32_t t) { return c * 32 + t; }
// Word of the 4-bit keys that holds them.
__device__ __forceinline__ uint32_t key_word(uint32_t c, uint32_t t) {
    return (c >> 3) * 256 + ((c & 1) * 32 + t) * 4 + ((c >> 1) & 3);
}
// Operand that holds channel d of token t in the values, and the token's element in it.
template <int D>
__device__ __forceinline__ uint32_t value_operand(uint32_t d, uint32_t t) {
    return ((t >> 4) * (D / 32) + (d >> 5)) * 64 + ((t >> 2) & 1) * 32 + (d & 31);
}
__device__ __forceinline__ uint32_t value_element(uint32_t t) { return ((t >> 3) & 1) * 4 + (t & 3); }
// Word of the 4-bit values that holds operand `o` (as value_operand gives it).
__device__ __forceinline__ uint32_t value_word(uint32_t o) { return ((o >> 8) * 64 + (o & 63)) * 4 + ((o >> 6) & 3); }
// Token of element e of the operands (s, h) of the values.
__device__ __forceinline__ uint32_t value_token(uint32_t s, uint32_t h, uint32_t e) {
    return 16 * s + 8 * (e >> 2) + 4 * h + (e & 3);
}
__device__ __forceinline__ uint32_t nibble_shift(uint32_t e) { return 4 * (e >> 1) + 16 * (e & 1); }

struct KvView {
    uint8_t *data;
    uint32_t num_pages, page_shift, kv_heads;  // page_shift: log2 of the blocks of a page
    uint32_t head_bytes;                       // bytes of a page that belong to one head
};

struct KvBatch {
    const int32_t *table;
    uint32_t table_stride, table_width;
    const int32_t *lens, *start;  // start == nullptr: one new token per sequence
    uint32_t seqs, tokens;
    uint32_t *status;  // device status word
};

struct SeqInfo {
    int32_t row, n, len;  // first row of q / k / v, new tokens, tokens in all
};

// The lengths a kernel works with: never outside the tensors they index, whatever the arrays hold.
__device__ __forceinline__ SeqInfo load_seq(const KvBatch &b, const KvView &v, uint32_t i, bool &bad) {
    SeqInfo s;
    const int32_t rows = (int32_t)b.tokens;
    if (b.start) {
        const int32_t a = b.start[i], e = b.start[i + 1];
        s.row = min(max(a, 0), rows);
        const int32_t end = min(max(e, s.row), rows);
        s.n = end - s.row;
        bad = a != s.row || e != end;
    } else {
        s.row = (int32_t)i;
        s.n = 1;
        bad = false;
    }
    const int32_t len = b.lens[i];
    const int64_t room = (int64_t)b.table_width << (v.page_shift + 5);
    s.len = len < 0 ? 0 : (int64_t)len > room ? (int32_t)room : len;
    // (a place of a padded batch: one token by the form of the call, and no tokens at all)
    bad = bad || len != s.len || (s.n > s.len && !(s.len == 0 && !b.start));
    return s;
}

__device__ __forceinline__ void report_bad_index(const KvBatch &b) {
    if (b.status) atomicOr(b.status, (uint32_t)CI_STATUS_BAD_INDEX);
}

// The same inside a sum over all sequences, which also meets those that have no work of their own to say it (offsets that
// fall, lengths outside the table without a new token): the first workgroup's sum reports them.
__device__ __forceinline__ SeqInfo load_seq_in_sum(const KvBatch &b, const KvView &v, uint32_t i) {
    bool bad;
    const SeqInfo s = load_seq(b, v, i, bad);
    if (bad && blockIdx.x == 0 && blockIdx.y == 0) report_bad_index(b);
    return s;
}

// Page that holds block `blk` of a sequence, or kNoPage if the table names none of the cache's.
__device__ __forceinline__ uint32_t page_of(const KvBatch &b, const KvView &v, uint32_t seq, uint32_t blk) {
    const uint32_t page = (uint32_t)b.table[(uint64_t)seq * b.table_stride + (blk >> v.page_shift)];
    return page < v.num_pages ? page : kNoPage;
}

// The same for a wavefront that walks through a sequence: 64 entries of the table at a time, one in each lane, so that a
// step finds its page without waiting for memory.
struct PageRun {
    const int32_t *row;
    uint32_t held, pages;  // which 64 entries; this lane's
    __device__ __forceinline__ PageRun(const KvBatch &b, uint32_t seq) : row(b.table + (uint64_t)seq * b.table_stride), held(kNoPage), pages(0) {}
    // makes sure that the entry of block `blk` is among those held; whether they were loaded anew
    __device__ __forceinline__ bool hold(const KvBatch &b, const KvView &v, uint32_t blk) {
        const uint32_t which = blk >> v.page_shift >> 6;
        if (which == held) return false;
        held = which;
        const uint32_t at = held * 64 + (threadIdx.x & 63);
        pages = at < b.table_width ? (uint32_t)row[at] : kNoPage;
        return true;
    }
    // the page of a block whose entry is held
    __device__ __forceinline__ uint32_t page_of(const KvView &v, uint32_t blk) const {
        const uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)pages, (int)((blk >> v.page_shift) & 63));
        return page < v.num_pages ? page : kNoPage;
    }
};

template <int KIND, int D>
__device__ __forceinline__ uint8_t *block_at(const KvView &v, uint32_t page, uint32_t head, uint32_t blk) {
    return v.data + (uint64_t)page * (v.head_bytes * v.kv_heads) + (uint64_t)(head * v.head_bytes) +
           (blk & ((1u << v.page_shift) - 1)) * KvBlock<KIND, D>::kBytes;  // (a page is below 4 GiB)
}

// Sums of work stop at the largest word.  The host has checked that the work of a batch stays below it, but for a batch
// whose row offsets fall: rows then belong to several sequences, and the sum may be anything.  Wrapped around, it would
// name places that do not exist; a sum that has reached kTooMuch is no sum, and nothing is done for that batch.
constexpr uint32_t kTooMuch = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t add_work(uint32_t x, uint32_t y) { return __builtin_elementwise_add_sat(x, y); }

// Exclusive prefix sum over the threads of a workgroup (up to eight wavefronts); `total` gets the sum (kTooMuch: the prefixes
// mean nothing).  `part` holds eight words of LDS.
__device__ __forceinline__ uint32_t scan_threads(uint32_t x, uint32_t *part, uint32_t &total) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t inc = x;
#pragma unroll
    for (uint32_t d = 1; d < 64; d *= 2) {
        const uint32_t y = (uint32_t)__shfl_up((int)inc, d, 64);
        if (lane >= d) inc = add_work(inc, y);
    }
    __syncthreads();
    if (lane == 63) part[wave] = inc;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
    for (uint32_t w = 0; w < blockDim.x / 64; ++w) {
        const uint32_t p = part[w];
        if (w < wave) before = add_work(before, p);
        total = add_work(total, p);
    }
    return before + inc - x;
}

// A running sum over the sequences, weight(i) each (evaluated by one thread: a contiguous run of sequences per thread).
// `target` maps the total to the place looked for: the sequence in whose share it falls, and where that share begins.
// Returns false when there is no such place.  `word` holds ten words of LDS.
struct Found {
    uint32_t seq, begin, total, target;
};

template <typename W, typename T>
__device__ __forceinline__ bool locate(uint32_t seqs, W weight, T target, uint32_t *word, Found &f) {
    const uint32_t per = (seqs + blockDim.x - 1) / blockDim.x, first = min(threadIdx.x * per, seqs), last = min(first + per, seqs);
    uint32_t mine = 0;
    for (uint32_t i = first; i < last; ++i) mine = add_work(mine, weight(i));
    uint32_t at = scan_threads(mine, word, f.total);
    f.total = (uint32_t)__builtin_amdgcn_readfirstlane((int)f.total);
    if (f.total == kTooMuch) return false;
    f.target = target(f.total);
    if (f.target >= f.total) return false;
    if (f.target >= at && f.target - at < mine) {
        uint32_t i = first;
        for (; i + 1 < last; ++i) {
            const uint32_t w = weight(i);
            if (f.target - at < w) break;
            at += w;
        }
        word[8] = i;
        word[9] = at;
    }
    __syncthreads();
    f.seq = (uint32_t)__builtin_amdgcn_readfirstlane((int)word[8]);
    f.begin = (uint32_t)__builtin_amdgcn_readfirstlane((int)word[9]);
    __syncthreads();
    return true;
}

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    f32x2_p v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_p));
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// host side
int check_kv_cache(const char *who, const ci_kv_cache *c, KvView *v);
int check_kv_batch(const char *who, const ci_kv_batch *b, const KvView &v, KvBatch *out);
bool rows_may_overlap(const ci_rows &a, uint32_t a_heads, const ci_rows &b, uint32_t b_heads, uint32_t tokens, uint32_t dim);

#define CI_KV_LAUNCH(kernel, grid, block, shmem, stream, ...) hipLaunchKernelGGL(kernel, grid, block, shmem, stream, __VA_ARGS__)

}  // namespace ci
