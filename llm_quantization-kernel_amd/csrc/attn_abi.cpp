// attn_abi.cpp -- the extern "C" entry points of include/crispybits_attention.h.  As in abi.cpp every check
// runs before the first HIP call.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "cbk_host.hpp"
#include "cbk_kernels.hpp"
#include "crispybits_attention.h"
#include "kv4.hpp"

using namespace cbk;

namespace {

constexpr int64_t MOST = INT32_MAX / 2;        // rows, pages, tokens of a table: positions stay in 32 bits
constexpr int64_t MOST_GRID = 65535;           // the second and third grid dimension

constexpr int64_t MOST_GROUPS = (1 << 24) - 1; // workgroups of 256 threads: a launch has fewer than 2^32 threads
constexpr int64_t MOST_STORED = 1 << 28;       // rows of an append or a read (32 a workgroup)
constexpr int64_t MAX_ROW_STRIDE = 1 << 23;

bool valid_dtype(int dt) { return dt == CBK_F16 || dt == CBK_BF16 || dt == CBK_F32; }
bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
int esize(int dt) { return dt == CBK_F32 ? 4 : 2; }

int check_heads(const char* what, int dtype, int64_t heads, int64_t kv_heads, int head_dim) {
    if (!valid_dtype(dtype)) return fail(CBK_EINVAL, "%s: tensors must be fp16/bf16/fp32", what);
    if (head_dim <= 0 || head_dim > KV4_MAX_D || head_dim % 8 != 0)
        return fail(CBK_EINVAL, "%s: head_dim must be a multiple of 8 up to %d", what, KV4_MAX_D);
    if (kv_heads <= 0 || heads <= 0 || heads % kv_heads != 0 || heads > MOST_GRID)
        return fail(CBK_EINVAL, "%s: heads must be a positive multiple of kv_heads (at most %d)", what, (int)MOST_GRID);
    return CBK_OK;
}

// 16-byte rows of a head: strides that the kernels step by with vector accesses (and 32-bit offsets within 64 rows).
int check_strides(const char* what, int dtype, int64_t row, int64_t head) {
    const int64_t unit = 16 / esize(dtype);
    if (row < 0 || head < 0 || row % unit != 0 || head % unit != 0)
        return fail(CBK_EINVAL, "%s: rows of a head must be 16-byte aligned", what);
    if (row > MAX_ROW_STRIDE) return fail(CBK_EINVAL, "%s: row strides are at most 2^23 elements", what);
    return CBK_OK;
}

// scale log2 e is an fp32 factor of the kernels
int check_scale(const char* what, float scale) {
    if (!(scale > 0.f && scale <= 0x1p127f)) return fail(CBK_EINVAL, "%s: scale must be positive and at most 2^127", what);
    return CBK_OK;
}

int log2_of(int64_t v) {
    int s = 0;
    while ((1ll << s) < v) ++s;
    return s;
}

// The cache and sequences of a call; 0 sequences are the caller's to skip.
int view(const char* what, const int32_t* pages, int64_t num_pages, int64_t kv_heads, int head_dim, int64_t page_size,
         const int32_t* table, int64_t width, const int32_t* lens, int64_t seqs, Kv4View& C) {
    if (cbk_kv4_page_words(head_dim, page_size) < 0)
        return fail(CBK_EINVAL, "%s: page_size must be a power of two from 32 to 65536", what);
    if (num_pages < 0 || num_pages > MOST) return fail(CBK_EINVAL, "%s: bad number of pages", what);
    if (seqs < 0 || seqs > MOST_GRID) return fail(CBK_EINVAL, "%s: at most %d sequences", what, (int)MOST_GRID);
    if (width < 0 || width * page_size > MOST) return fail(CBK_EINVAL, "%s: block table too wide", what);
    if (seqs > 0 && (!lens || (width > 0 && !table) || (num_pages > 0 && !pages)))
        return fail(CBK_EINVAL, "%s: pages, block_table and seq_lens must be non-null", what);
    if (!aligned(pages)) return fail(CBK_EINVAL, "%s: pages must be 16-byte aligned", what);
    C.pages = reinterpret_cast<uint32_t*>(const_cast<int32_t*>(pages));
    C.table = table;
    C.lens = lens;
    C.num_pages = (int)num_pages;
    C.heads = (int)kv_heads;
    C.d = head_dim;
    C.ns = kv4_ns(head_dim);
    C.page_shift = log2_of(page_size / KV4_BLOCK);
    C.width = (int)width;
    C.seqs = (int)seqs;
    return CBK_OK;
}

int check_rows(const char* what, int64_t rows, const int32_t* cu, int64_t seqs) {
    if (rows < 0 || rows > MOST_STORED) return fail(CBK_EINVAL, "%s: bad number of rows", what);
    if (!cu && rows != seqs) return fail(CBK_EINVAL, "%s: without cu_seqlens there is one row a sequence", what);
    return CBK_OK;
}

// Workgroups of a cache attention call: as many as are on the chip's 256 CUs at once, and where the work is
// less, one for each unit or MIN_BLOCKS blocks.  Units cannot be cut where none has more than KV4_WHOLE blocks.
constexpr int64_t CUS = 256;
static_assert(3 * CUS <= SPLIT_COUNTERS, "a counter per workgroup");
constexpr int MIN_BLOCKS = 12;
constexpr int UNIT_COST = 12;

struct AttnPlan {
    int64_t rows, tiles, groups, floats, blocks;
    int cols;
};

AttnPlan plan_attn(int dtype, int64_t seqs, int64_t t, int64_t heads, int64_t kv_heads, int d, int64_t page,
                   int64_t width) {
    AttnPlan p;
    p.rows = t * (heads / kv_heads);
    p.tiles = (p.rows + 15) / 16;
    p.cols = (int)std::min<int64_t>(p.rows, 16);
    const int64_t units = std::max<int64_t>(1, seqs * kv_heads * p.tiles);
    const int64_t most = std::max<int64_t>(1, width * (page / KV4_BLOCK));
    p.blocks = units * (most + UNIT_COST);
    p.groups = std::min(kv4_waves(kv4_ns(d), dtype) * CUS, std::max(units, p.blocks / MIN_BLOCKS));
    p.floats = most > KV4_WHOLE && p.groups > 1 ? 2 * p.groups * p.cols * (d + 2) : 0;
    return p;
}

}  // namespace

extern "C" {

int64_t cbk_kv4_page_words(int head_dim, int64_t page_size) {
    if (head_dim <= 0 || head_dim > KV4_MAX_D || head_dim % 8 != 0) return -1;
    if (page_size < KV4_BLOCK || page_size > 65536 || (page_size & (page_size - 1)) != 0) return -1;
    return page_size / KV4_BLOCK * kv4_block_words(kv4_ns(head_dim));
}

int cbk_kv4_append(int32_t* pages, int64_t num_pages, int64_t kv_heads, int head_dim, int64_t page_size,
                   const void* k, const void* v, int dtype, int64_t rows,
                   int64_t k_row, int64_t k_head, int64_t v_row, int64_t v_head,
                   const int32_t* block_table, int64_t table_width, const int32_t* seq_lens,
                   const int32_t* cu_seqlens, int64_t num_seqs, int device, void* stream) {
    const char* what = "kv4_append";
    Kv4StoreArgs A = {};
    if (int e = check_heads(what, dtype, kv_heads, kv_heads, head_dim)) return e;
    if (int e = check_strides(what, dtype, k_row, k_head)) return e;
    if (int e = check_strides(what, dtype, v_row, v_head)) return e;
    if (int e = view(what, pages, num_pages, kv_heads, head_dim, page_size, block_table, table_width, seq_lens, num_seqs,
                     A.c))
        return e;
    if (int e = check_rows(what, rows, cu_seqlens, num_seqs)) return e;
    if (rows == 0 || num_seqs == 0) return CBK_OK;
    if (!k || !v) return fail(CBK_EINVAL, "%s: k and v must be non-null", what);
    if (!aligned(k) || !aligned(v)) return fail(CBK_EINVAL, "%s: k and v must be 16-byte aligned", what);
    A.r = {cu_seqlens, (int)rows};
    A.k = k, A.v = v;
    A.k_row = k_row, A.k_head = k_head, A.v_row = v_row, A.v_head = v_head;
    DeviceGuard guard(device);
    if (guard.err != hipSuccess) return hip_fail(guard.err, "set device");
    const hipError_t e = launch_kv4_append(A, dtype, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? CBK_OK : hip_fail(e, what);
}

int cbk_kv4_read(const int32_t* pages, int64_t num_pages, int64_t kv_heads, int head_dim, int64_t page_size,
                 void* k, void* v, int dtype, int64_t rows,
                 const int32_t* block_table, int64_t table_width, const int32_t* seq_lens,
                 const int32_t* cu_seqlens, int64_t num_seqs, int device, void* stream) {
    const char* what = "kv4_read";
    Kv4StoreArgs A = {};
    if (int e = check_heads(what, dtype, kv_heads, kv_heads, head_dim)) return e;
    if (int e = view(what, pages, num_pages, kv_heads, head_dim, page_size, block_table, table_width, seq_lens, num_seqs,
                     A.c))
        return e;
    if (int e = check_rows(what, rows, cu_seqlens, num_seqs)) return e;
    if (rows == 0) return CBK_OK;
    if (num_seqs == 0) return fail(CBK_EINVAL, "%s: rows without a sequence", what);
    if (!k || !v) return fail(CBK_EINVAL, "%s: k and v must be non-null", what);
    if (!aligned(k) || !aligned(v)) return fail(CBK_EINVAL, "%s: k and v must be 16-byte aligned", what);
    A.r = {cu_seqlens, (int)rows};
    A.k_out = k, A.v_out = v;
    DeviceGuard guard(device);
    if (guard.err != hipSuccess) return hip_fail(guard.err, "set device");
    const hipError_t e = launch_kv4_read(A, dtype, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? CBK_OK : hip_fail(e, what);
}

int64_t cbk_kv4_attention_partial_floats(int64_t num_seqs, int64_t t, int64_t heads, int64_t kv_heads, int head_dim,
                                         int64_t page_size, int64_t table_width) {
    if (num_seqs <= 0 || t <= 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads != 0 ||
        cbk_kv4_page_words(head_dim, page_size) < 0 || table_width < 0)
        return 0;
    return plan_attn(CBK_F16, num_seqs, t, heads, kv_heads, head_dim, page_size, table_width).floats;      // the most of any type
}

int cbk_kv4_attention(const void* q, int dtype, int64_t num_seqs, int64_t t, int64_t heads,
                      const int32_t* pages, int64_t num_pages, int64_t kv_heads, int head_dim, int64_t page_size,
                      const int32_t* block_table, int64_t table_width, const int32_t* seq_lens, float scale,
                      float* partial, int64_t partial_floats, void* out, int device, void* stream) {
    const char* what = "kv4_attention";
    Kv4AttnArgs A = {};
    if (int e = check_heads(what, dtype, heads, kv_heads, head_dim)) return e;
    if (int e = view(what, pages, num_pages, kv_heads, head_dim, page_size, block_table, table_width, seq_lens, num_seqs,
                     A.c))
        return e;
    if (int e = check_scale(what, scale)) return e;
    if (t < 0 || t > MOST || t * heads > MOST) return fail(CBK_EINVAL, "%s: bad number of new tokens", what);
    if (num_seqs == 0 || t == 0) return CBK_OK;
    if (!q || !out) return fail(CBK_EINVAL, "%s: q and out must be non-null", what);
    if (!aligned(q) || !aligned(out)) return fail(CBK_EINVAL, "%s: q and out must be 16-byte aligned", what);
    const AttnPlan p = plan_attn(dtype, num_seqs, t, heads, kv_heads, head_dim, page_size, table_width);
    if (kv_heads * p.tiles > MOST_GRID) return fail(CBK_EINVAL, "%s: too many new tokens", what);
    if (p.blocks > INT32_MAX / 2) return fail(CBK_EINVAL, "%s: block table too wide for the call's sequences and heads", what);
    if (p.floats > 0 && (!partial || partial_floats < p.floats))
        return fail(CBK_EINVAL, "%s: partial must hold %lld floats", what, (long long)p.floats);
    A.q = q, A.out = out;
    A.partial = p.floats > 0 ? partial : nullptr;
    A.t = (int)t, A.hq = (int)heads, A.group = (int)(heads / kv_heads);
    A.rows = (int)p.rows, A.tiles = (int)p.tiles, A.cols = p.cols;
    A.groups = (int)p.groups, A.min_blocks = MIN_BLOCKS, A.unit_cost = UNIT_COST;
    A.scale = scale;
    A.div_group = make_fastdiv((uint32_t)A.group);
    DeviceGuard guard(device);
    if (guard.err != hipSuccess) return hip_fail(guard.err, "set device");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    A.split_cnt = p.floats > 0 ? attn_window(device, s) : nullptr;
    const hipError_t e = launch_kv4_attn(A, dtype, s);
    return e == hipSuccess ? CBK_OK : hip_fail(e, what);
}

int cbk_prompt_attention(const void* q, const void* k, const void* v, int dtype, int64_t rows, int64_t heads,
                         int64_t kv_heads, int head_dim, int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head,
                         int64_t v_row, int64_t v_head, const int32_t* cu_seqlens, int64_t num_seqs,
                         int64_t max_seqlen, float scale, int zero_tail, void* out, int device, void* stream) {
    const char* what = "prompt_attention";
    if (int e = check_heads(what, dtype, heads, kv_heads, head_dim)) return e;
    if (int e = check_strides(what, dtype, q_row, q_head)) return e;
    if (int e = check_strides(what, dtype, k_row, k_head)) return e;
    if (int e = check_strides(what, dtype, v_row, v_head)) return e;
    if (rows < 0 || rows > MOST) return fail(CBK_EINVAL, "%s: bad number of rows", what);
    if (num_seqs < 0 || num_seqs > MOST_GRID) return fail(CBK_EINVAL, "%s: at most %d sequences", what, (int)MOST_GRID);
    if (int e = check_scale(what, scale)) return e;
    if (rows == 0) return CBK_OK;
    if (num_seqs == 0) return fail(CBK_EINVAL, "%s: rows without a sequence", what);
    if (max_seqlen <= 0 || max_seqlen > rows)
        return fail(CBK_EINVAL, "%s: max_seqlen must be from 1 to the number of rows", what);
    if (!q || !k || !v || !out || !cu_seqlens)
        return fail(CBK_EINVAL, "%s: q, k, v, out and cu_seqlens must be non-null", what);
    if (!aligned(q) || !aligned(k) || !aligned(v) || !aligned(out))
        return fail(CBK_EINVAL, "%s: q, k, v and out must be 16-byte aligned", what);
    if ((max_seqlen + 127) / 128 * (num_seqs + 1) * heads > MOST_GROUPS)
        return fail(CBK_EINVAL, "%s: max_seqlen x sequences x heads is too large", what);
    PromptArgs A = {};
    A.q = q, A.k = k, A.v = v, A.out = out, A.cu = cu_seqlens;
    A.q_row = q_row, A.q_head = q_head, A.k_row = k_row, A.k_head = k_head, A.v_row = v_row, A.v_head = v_head;
    A.rows = (int)rows, A.seqs = (int)num_seqs, A.hq = (int)heads, A.hkv = (int)kv_heads;
    A.group = (int)(heads / kv_heads), A.d = head_dim;
    A.longest = (int)max_seqlen, A.zero_tail = zero_tail ? 1 : 0;
    A.scale = scale;
    DeviceGuard guard(device);
    if (guard.err != hipSuccess) return hip_fail(guard.err, "set device");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t e = dtype == CBK_F32 ? launch_prompt_attn_f32(A, s) : launch_prompt_attn(A, dtype, s);
    return e == hipSuccess ? CBK_OK : hip_fail(e, what);
}

}  // extern "C"
