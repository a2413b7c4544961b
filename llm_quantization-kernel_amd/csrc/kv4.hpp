// kv4.hpp -- the paged 4-bit key/value cache: its layout, shared by the kernels that write, read
// and attend over it (kv4_store.hip, kv4_attn.hip).
//
// A vector x of one token and kv head is held as 4-bit codes c, a scale s and an integer zero point
// z in 0..15, x = s (c - z).  s and z share one 32-bit word: the word read as a float is s, its low
// four mantissa bits are z (s is known to 2^-20 of itself when the codes are chosen, so they are
// chosen for the s that will be read back).  A token with a value that is not finite has s = NaN.
//
// A page holds `page` tokens (a power of two, at least 32) of every kv head; pages is int32
// [pages, kv heads, words], a (page, head) being page / 32 blocks of 32 tokens.  With
// NS = ceil(D / 32) a block holds, in 32-bit words:
//   K codes  [token 0..31][4 NS]: word w of a token has values d = 8 w .. 8 w + 7
//   V codes  [piece][g 0..3][m 0..15][e 0..PW-1]: the word of d = 16 (piece PW + e) + m has the
//            tokens 4 g + j (j < 4) and 16 + 4 g + j - 4 (j >= 4) of the block
//   K words [32], V words [32] of scale and zero point
// Value j of a word takes four bits from bit 2 + 4 (j / 2) + 16 (j % 2) on (bit 32 is bit 0 again), so that
// `word & 0x003C003C` is the pair (0, 1), `word & 0x03C003C0` the pair (2, 3) times 16, and the same of the word
// rotated right by 8 the pairs (4, 5) and (6, 7).  Read as fp16 such a pair is two denormals, c 2^-22 or c 2^-18, exact
// operands of the matrix cores: decoding eight codes takes five instructions.  (The place within the mantissa
// matters: the products of a step are aligned by their operands' exponents, which a denormal does not carry in full.
// Two terms far apart lost up to 2^-18 of the larger with codes in the lowest mantissa bits, 2^-24 at the top ones.)
// The order of K's words within a row and of V's tokens within a word is that of the 16x16x32 operands: a
// lane's loads are 16-byte pieces (8- and 12-byte for odd NS) of a contiguous KB, and V needs no transposition.
#pragma once

#include "cbk_device.hpp"

namespace cbk {

constexpr int KV4_BLOCK = 32;                        // tokens of a block
constexpr int KV4_MAX_D = 256;
constexpr int KV4_WHOLE = 8;                           // attention does not cut units of this many blocks
// the smallest scale a token may have: values below it count as zeros
constexpr float KV4_MIN_SCALE = 0x1p-100f;

__host__ __device__ constexpr int kv4_ns(int d) { return (d + 31) / 32; }
__host__ __device__ constexpr int kv4_block_words(int ns) { return 256 * ns + 2 * KV4_BLOCK; }
__host__ __device__ constexpr int kv4_piece(int ns) { return ns % 2 == 0 ? 4 : 2; }    // PW
// first bit of value j in a word of eight codes
__host__ __device__ constexpr int kv4_bit(int j) { return 2 + 4 * (j >> 1) + 16 * (j & 1); }
__host__ __device__ constexpr uint32_t kv4_put(uint32_t code, int j) {
    const int b = kv4_bit(j);
    return b > 28 ? code << b | code >> (32 - b) : code << b;
}
__device__ __forceinline__ uint32_t kv4_get(uint32_t word, int bit) {
    return __builtin_amdgcn_alignbit(word, word, bit) & 15u;
}
// slot of token t (0..31) of a block in its V word: group g and value j
__host__ __device__ constexpr int kv4_group(int t) { return (t & 15) >> 2; }
__host__ __device__ constexpr int kv4_value(int t) { return (t & 3) + 4 * (t >> 4); }

// A cache and the sequences a call works on.
struct Kv4View {
    uint32_t* pages;
    const int32_t* table;      // [seqs, width] page of each `page` tokens
    const int32_t* lens;       // [seqs] tokens, a call's new ones included
    int num_pages, heads, d, ns;
    int page_shift;            // log2(page / 32): blocks of a page
    int width, seqs;
};

// An entry of an index tensor that no kernel of the call writes, read at a wave-uniform place: through the constant
// address space, so that it is a scalar load, which waits for no vector load under way.
__device__ __forceinline__ int index_at(const int32_t* p, long i) {
    return reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p))[i];
}

// The first word of block `blk` of sequence `b`, head `h`; nullptr where the table has no page of the
// pool for it (behind the table, or an entry outside the pool): such tokens do not exist.
__device__ __forceinline__ uint32_t* kv4_block(const Kv4View& C, int b, int blk, int h) {
    const int p = blk >> C.page_shift;
    if (blk < 0 || p >= C.width) return nullptr;
    const int page = index_at(C.table, (long)b * C.width + p);
    if ((unsigned)page >= (unsigned)C.num_pages) return nullptr;
    const long row = ((long)page * C.heads + h) << C.page_shift;
    return C.pages + (row + (blk & ((1 << C.page_shift) - 1))) * kv4_block_words(C.ns);
}

// Calls that store or read tokens: row r of the new ones, cu[b] <= r < cu[b + 1], is token
// lens[b] - (cu[b + 1] - cu[b]) + r - cu[b] of sequence b; without cu, row b is the newest token of b.
struct Kv4Rows {
    const int32_t* cu;         // [seqs + 1] or nullptr
    int rows;
};

// kv4_store.hip
struct Kv4StoreArgs {
    Kv4View c;
    Kv4Rows r;
    const void* k;             // [rows, heads, d]; strides in elements, d contiguous
    const void* v;
    long k_row, k_head, v_row, v_head;
    void* k_out;               // read: contiguous [rows, heads, d]
    void* v_out;
};
hipError_t launch_kv4_append(const Kv4StoreArgs& A, int dt, hipStream_t stream);
hipError_t launch_kv4_read(const Kv4StoreArgs& A, int dt, hipStream_t stream);

// kv4_attn.hip
// Workgroups of the attention kernel that a CU holds, by its registers.
__host__ __device__ constexpr int kv4_waves(int ns, int dt) {
    return dt == DT_F32 ? (ns <= 2 ? 3 : ns <= 4 ? 2 : 1) : ns <= 4 ? 3 : 2;
}
struct Kv4AttnArgs {
    Kv4View c;
    const void* q;             // [seqs, t, hq, d] contiguous, 16-byte aligned
    void* out;                 // the same
    float* partial;            // [2 groups][cols, d], then [2 groups][cols, 2]; nullptr: no unit can be cut
    uint32_t* split_cnt;       // an arrival counter per workgroup; nullptr: a combine launch
    int t, hq, group;          // new tokens a sequence, query heads, query heads per kv head
    int rows, tiles, cols;     // t * group query rows per kv head, tiles of 16 of them, rows of a partial
    int groups, min_blocks;    // workgroups; blocks each takes at least where units are cut
    int unit_cost;             // blocks that a unit costs beside its own
    float scale;
    FastDiv div_group;
};
hipError_t launch_kv4_attn(const Kv4AttnArgs& A, int dt, hipStream_t stream);

// From here on a running reference is too far from zero for s c - M as one FMA: the product's rest, up to half a last place
// of M, would go into the exponent.
constexpr float FAR = 0x1p20f;
// s c, rounded, minus M
__device__ __forceinline__ float less_rounded(float s, float c, float M) {
#pragma clang fp contract(off)
    const float p = s * c;
    return p - M;
}

// prompt_attn.hip, prompt_attn_f32.hip
struct PromptArgs {
    const void *q, *k, *v;
    void* out;                 // contiguous [rows, hq, d]
    const int32_t* cu;         // [seqs + 1]
    long q_row, q_head, k_row, k_head, v_row, v_head;     // strides in elements
    int rows, seqs, hq, hkv, group, d;
    int longest;               // no sequence has more rows
    int zero_tail;             // rows of no sequence are set to zero
    float scale;
};
hipError_t launch_prompt_attn(const PromptArgs& A, int dt, hipStream_t stream);
hipError_t launch_prompt_attn_f32(const PromptArgs& A, hipStream_t stream);

}  // namespace cbk
