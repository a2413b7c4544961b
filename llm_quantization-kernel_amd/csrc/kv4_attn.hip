// kv4_attn.hip -- attention of each sequence's newest tokens over its paged 4-bit cache (kv4.hpp).
//
// For query row r (token i of t, head) and cached token j the score is
//   scale q.k_j = scale s_j (q.c_j - z_j sum q)
// and the output sum_j p_j s'_j (c'_j - z'_j) with p the softmax of the scores: scales and zero points
// stay outside the products, which run on the codes as they are stored (fp16 denormals, exact) on
// v_mfma_f32_16x16x32_f16.  A wave takes blocks of 32 tokens:
//   S^T[token, row] = K codes x q    (two 16-token tiles, NS steps of 32 values)
//   O^T[d, row]    += V codes x w    (2 NS tiles of 16 values, one step of 32 tokens), w = p s'
// The lane layout of S^T (column = row, four tokens a lane group and tile) is the operand layout of w
// when V's words hold a lane group's tokens (kv4.hpp), so w never leaves its lane.  sum_j w_j z'_j is one
// more product, with the zero points as codes.
//
// q is scaled by a power of two per row, to values below 2^11, so that its fp16 is exact for fp16 and
// bf16 q; where the stored pairs count 16 times, q is held / 16, and
// w takes the 1/16 in its exponent.  w must fit fp16 at any scale s': the running reference M of a row
// bounds score + log2 s' of each token seen, w = 2^(score - M + 12) s', so that w < 2^15, the largest is 2^10 or
// more, and only what lies 2^31 below it is lost; the sum of p is held with the same factor, of unrounded p.  For fp16
// outputs w goes as two fp16 terms, 22 bits: one term's rounding is as large as the output's own (errors of 2.9e-4 against 2.1e-4,
// at 37.2 against 39.5 us for the ragged batch of 32); for bf16 outputs it is an eighth of it.  M moves only when it
// would have to by 3 or more (the accumulators are rescaled then).
// fp32 q and w go as three fp16 terms, 33 bits: a whole number below 2^11 and two of the rest, with sums of their own, and
// codes with the zero point taken off.  Sums of whole numbers are exact in the matrix product, so the scores' own rounding
// is what is left: 1e-7 of an output at 500 tokens, fp32 products of torch 5e-7.  (Two terms in one sum: up to 1e-5, at 14.6 us
// instead of 16.1 for 5 sequences of 200..1501 tokens, 32 heads of 80; fp32 matrix instructions have a sixteenth of the rate.)
//
// Work: a unit is a sequence, kv head and tile of 16 query rows, of as many blocks as the sequence has (one at
// least, whose workgroup writes the zeros of an empty one).  The blocks of all units stand in one row, sequence by
// sequence, and each workgroup takes an equal piece of it, counted from the lengths on the device: ragged batches
// and single long sequences load the chip alike.  Its four waves take a unit's blocks in turn, the next block's
// loads under way, and meet in LDS.  A unit cut by a border is joined from fp32 partials, at most two a
// workgroup, by the last of its workgroups to arrive (or a second launch), in a fixed order.  Units of few blocks are not
// cut: the workgroup that has their first block takes them whole.
//
// Bound: the cache's bytes, 4352 a block at D = 128 (64 sequences of 1024..8192 tokens, 8 kv heads, bf16: 245 MB in 57.0 us,
// 4.3 TB/s of the 4.9 a large copy reaches); about 320 vector instructions a block fill a third of the issue slots.  Short
// calls are latencies: 32 heads of one sequence of 77 tokens 6.1 us.  An even cut against a fixed number of splits a
// sequence, 32 sequences of 64..4096 tokens in fp16, with one term of w: 36.4 us against 45.4 (39.6 with two).
#include "kv4.hpp"
#include "cbk_kernels.hpp"

namespace cbk {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int WAVES = 4;
constexpr float LOW = -0x1.fffffep127f;        // reference of a row that has seen nothing
constexpr float SLACK = 3.f;
// w < 2^(HEADROOM + SLACK): 2^15, in fp16's range; fp32's w below 2^11, whose whole part is one fp16 term
template <int DT>
constexpr float HEADROOM = DT == DT_F32 ? 8.f : 12.f;

union Op {
    h8 v;
    uint32_t u[4];
    _Float16 h[8];
};

// Eight codes of a word as an operand: pairs (0,1) and (4,5) as c 2^-22, (2,3) and (6,7) as c 2^-18.
__device__ __forceinline__ h8 decode(uint32_t w) {
    Op o;
    o.u[0] = w & 0x003C003Cu;
    o.u[1] = w & 0x03C003C0u;
    const uint32_t s = __builtin_amdgcn_alignbit(w, w, 8);
    o.u[2] = s & 0x003C003Cu;
    o.u[3] = s & 0x03C003C0u;
    return o.v;
}

// The same with each code's zero point taken off, as whole numbers in fp16 (for fp32 q: no term of the sums is larger
// than it has to be).  lo = -(256 + z), hi = -(16 + z) for each of the pair: the codes are put behind the leading one of 256
// (bits 2..5) and 16 (bits 6..9).
__device__ __forceinline__ h2 pair_of(uint32_t v) { return __builtin_bit_cast(h2, v); }
__device__ __forceinline__ h8 decode_exact(uint32_t w, h2 lo0, h2 hi0, h2 lo1, h2 hi1) {
    Op o;
    const uint32_t s = __builtin_amdgcn_alignbit(w, w, 8);
    o.u[0] = __builtin_bit_cast(uint32_t, pair_of((w & 0x003C003Cu) | 0x5C005C00u) + lo0);
    o.u[1] = __builtin_bit_cast(uint32_t, pair_of((w & 0x03C003C0u) | 0x4C004C00u) + hi0);
    o.u[2] = __builtin_bit_cast(uint32_t, pair_of((s & 0x003C003Cu) | 0x5C005C00u) + lo1);
    o.u[3] = __builtin_bit_cast(uint32_t, pair_of((s & 0x03C003C0u) | 0x4C004C00u) + hi1);
    return o.v;
}

// x of magnitude below 2^11 as a + b 2^-11 + c 2^-11, a and b whole numbers: products with codes sum up exactly in a
// matrix product (24 bits below its largest term are kept), those of c to 2^-33 of the largest x.
__device__ __forceinline__ void in_three(float x, _Float16& a, _Float16& b, _Float16& c) {
    const float i = __builtin_rintf(x), r = (x - i) * 2048.f, k = __builtin_rintf(r);
    a = (_Float16)i, b = (_Float16)k, c = (_Float16)(r - k);
}

__device__ __forceinline__ f4 mfma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// The largest, and the sum, over the four lane groups (lanes l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float group_max(float v) {
    const uint32_t u = __float_as_uint(v);
    auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const uint32_t t = __float_as_uint(v);
    r = __builtin_amdgcn_permlane16_swap(t, t, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float group_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// One block's words as a lane holds them, keys and values loaded apart.
template <int NS, bool EXACT>
struct Block {
    uint32_t k[2][NS];
    uint32_t v[2 * NS];
    u4 km[2], vm[2];
    uint32_t kz[2];                    // EXACT: the words of the tokens whose codes this lane decodes

    // byte offsets from the (uniform) block, 32-bit: one register an address
    __device__ __forceinline__ void load_k(const uint32_t* p, uint32_t lane) {
        const char* base = reinterpret_cast<const char*>(p);
        const uint32_t ko = ((lane & 15) * 4 * NS + (lane >> 4) * NS) * 4, mo = 1024 * NS + (lane >> 4) * 16;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            __builtin_memcpy(k[i], base + (ko + i * 256 * NS), 4 * NS);
            km[i] = *reinterpret_cast<const u4*>(base + (mo + 64 * i));
            if constexpr (EXACT) kz[i] = *reinterpret_cast<const uint32_t*>(base + (1024 * NS + 64 * i + (lane & 15) * 4));
        }
    }
    __device__ __forceinline__ void load_v(const uint32_t* p, uint32_t lane) {
        constexpr int PW = kv4_piece(NS);
        const char* base = reinterpret_cast<const char*>(p);
        const uint32_t vo = 512 * NS + lane * PW * 4, mo = 1024 * NS + 128 + (lane >> 4) * 16;
#pragma unroll
        for (int i = 0; i < 2; ++i) vm[i] = *reinterpret_cast<const u4*>(base + (mo + 64 * i));
#pragma unroll
        for (int i = 0; i < 2 * NS / PW; ++i) __builtin_memcpy(v + i * PW, base + (vo + i * 256 * PW), 4 * PW);
    }
};

template <int DT>
__device__ __forceinline__ void load8(const void* p, long i, float (&x)[8]) {
    using S = typename Dt<DT>::S;
    struct alignas(16) V { S v[8]; };
    const V v = *reinterpret_cast<const V*>(reinterpret_cast<const S*>(p) + i);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = Dt<DT>::to_f(v.v[j]);
}

// Blocks of a sequence in the row of all units' blocks.
__device__ __forceinline__ int blocks_of(const Kv4AttnArgs& A, int len) {
    const int room = A.c.width << A.c.page_shift;
    return max(min((max(len, 0) + 31) >> 5, room), 1);
}

// Sum over lanes 0 .. lane.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);      // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);      // row_bcast 15, 31
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

// The row of blocks and this workgroup's piece of it: positions count blocks, a sequence's units (kv heads x row
// tiles) follow each other.  A unit costs more than its blocks (its query, the waves' meeting): it stands
// for unit_cost blocks more, before its own.
struct Row {
    int len0;                          // this lane's length among the first 64 sequences
    int total, piece, whole;           // blocks; of a piece; units of at most so many are not cut

    __device__ __forceinline__ int count(const Kv4AttnArgs& A, int b0, int lane) const {
        const int b = b0 + lane;
        return b < A.c.seqs ? blocks_of(A, b0 == 0 ? len0 : A.c.lens[b]) + A.unit_cost : 0;
    }
    __device__ __forceinline__ void set(const Kv4AttnArgs& A, int lane) {
        len0 = lane < A.c.seqs ? A.c.lens[lane] : 0;
        int sum = 0;
        uint64_t large = 0;
        for (int b0 = 0; b0 < A.c.seqs; b0 += 64) {
            const int c = count(A, b0, lane);
            large |= __builtin_amdgcn_ballot_w64(c > KV4_WHOLE + A.unit_cost);
            sum += __builtin_amdgcn_readlane(wave_scan(c), 63);
        }
        total = sum * A.c.heads * A.tiles;
        piece = max((total + A.groups - 1) / A.groups, large ? A.min_blocks : 1);
        whole = max(KV4_WHOLE, piece >> 3);
    }
};

// A unit: its sequence, which of the sequence's units, its blocks and the first one's position.
struct Unit {
    int b, j, blocks, start;
};

__device__ __forceinline__ Unit unit_at(const Kv4AttnArgs& A, const Row& R, int x, int lane) {
    const int each = A.c.heads * A.tiles;
    Unit u;
    int before = 0;
    for (int b0 = 0;; b0 += 64) {
        const int c = R.count(A, b0, lane), upto = wave_scan(c);
        const uint64_t m = __builtin_amdgcn_ballot_w64(b0 + lane < A.c.seqs && (before + upto) * each <= x);
        const int k = __builtin_popcountll(m);
        if (k < 64 || b0 + 64 >= A.c.seqs) {
            const int i = min(k, 63);
            u.b = b0 + i;
            u.blocks = __builtin_amdgcn_readlane(c, i);
            const int first = (before + __builtin_amdgcn_readlane(upto, i) - u.blocks) * each;
            u.j = (x - first) / max(u.blocks, 1);
            u.start = first + u.j * u.blocks + A.unit_cost;
            u.blocks -= A.unit_cost;
            return u;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
}

// The partials of a slot (two a workgroup: its piece's first unit, and a later one): [cols][D] sums, and behind
// those of all slots [cols][2], each row's reference M and sum of p.  They pass between workgroups on any XCD: written
// and read past the L2s (sc1), as split_arrive's note says.
constexpr int SC1 = 16;
__device__ __forceinline__ float* part_sums(const Kv4AttnArgs& A, int slot) {
    return A.partial + (long)slot * A.cols * A.c.d;
}
__device__ __forceinline__ float* part_rows(const Kv4AttnArgs& A, int slot) {
    return A.partial + 2l * A.groups * A.cols * A.c.d + (long)slot * A.cols * 2;
}
// The parts of a unit that borders cut: workgroups first .. first + count - 1; its part in the first is that one's
// later slot unless the unit starts its piece.
struct Parts {
    int first, count, later;
    __device__ __forceinline__ int slot(int i) const { return 2 * (first + i) + (i == 0 ? later : 0); }
};
__device__ __forceinline__ Parts parts_of(const Row& R, const Unit& u) {
    Parts p;
    p.first = u.start / R.piece;
    p.count = (u.start + u.blocks - 1) / R.piece - p.first + 1;
    p.later = u.start != p.first * R.piece ? 1 : 0;
    return p;
}

template <int DT>
__device__ __forceinline__ long out_at(const Kv4AttnArgs& A, int b, int h, int row) {
    const int i = (int)fdiv((uint32_t)row, A.div_group);
    return (((long)b * A.t + i) * A.hq + h * A.group + (row - i * A.group)) * A.c.d;
}

// LDS of the combine: what each part's row counts for, and the sums of the thread groups.
constexpr int SHARES = 64;             // parts whose shares are held at once
struct CombineLds {
    float share[SHARES * 16];
    float m[16][16], l[16][16];
    float4 sum[64 * WAVES];
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const float* p, long floats) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(p), 0, (int)min(floats * 4, (long)0x7FFFFFF0), 0x00027000);
}

// Adds a cut unit's partials in order and writes its rows.  Threads share the parts.  Up to 64 parts (8 a thread of
// the sums) all loads are under way before the first is waited for: the joining workgroup is the call's last one, and
// its latencies add up.
template <int DT>
__device__ __forceinline__ void combine(const Kv4AttnArgs& A, CombineLds& L, const Parts& P, int b, int h, int tile) {
    constexpr int EARLY = 8;
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));                                // its places are found here, not held in registers all along
    const int D = A.c.d, cols = min(A.cols, A.rows - 16 * tile);
    const int col = tid & 15, s0 = tid >> 4;
    const __amdgpu_buffer_rsrc_t sums = buffer_of(part_sums(A, 2 * P.first), 2l * P.count * A.cols * D);
    const __amdgpu_buffer_rsrc_t rows = buffer_of(part_rows(A, 2 * P.first), 4l * P.count * A.cols);
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    // (M, sum of p) of this thread's row in part s; past the last part, or a row that is not there: nothing seen
    auto row_of = [&](int s) {
        const int at = s < P.count && col < cols ? ((P.slot(s) - 2 * P.first) * A.cols + col) * 8 : -1;
        const u2 v = __builtin_amdgcn_raw_buffer_load_b64(rows, at, 0, SC1);
        return at < 0 ? u2{__float_as_uint(LOW), 0u} : v;
    };
    const int items = cols * (D >> 2), stride = A.cols * D * 4;
    const int groups = max(1, 64 * WAVES / items);               // thread groups that share the parts
    const int grp = groups > 1 ? tid / items : 0;
    auto sum_of = [&](int s, int c, int d) {
        const int at = s < P.count ? (P.slot(s) - 2 * P.first) * stride + (c * D + d) * 4 : -1;
        return __builtin_amdgcn_raw_buffer_load_b128(sums, at, 0, SC1);      // past the buffer: zeros
    };
    u2 ml[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) ml[i] = row_of(s0 + 16 * i);
    u4 early[EARLY];
    {
        const int x = groups > 1 ? tid - grp * items : tid, c = min(x / (D >> 2), cols - 1), d = (x - x / (D >> 2) * (D >> 2)) * 4;
#pragma unroll
        for (int i = 0; i < EARLY; ++i) early[i] = sum_of(grp < groups ? grp + i * groups : P.count, c, d);
    }
    float m = LOW, l = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, __uint_as_float(ml[i][0]));
    for (int s = s0 + SHARES; s < P.count; s += 16) m = fmaxf(m, __uint_as_float(row_of(s)[0]));
    L.m[s0][col] = m;
    lds_barrier();
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, L.m[i][col]);
    for (int x0 = 0; x0 < items; x0 += 64 * WAVES) {
        const int x = groups > 1 ? tid - grp * items : x0 + tid;
        const int c = min(x / (D >> 2), cols - 1), d = (x - x / (D >> 2) * (D >> 2)) * 4;
        float4 o = {0.f, 0.f, 0.f, 0.f};
        for (int p0 = 0; p0 < P.count; p0 += SHARES) {
            const int p1 = min(p0 + SHARES, P.count);
            if (x0 == 0 || P.count > SHARES) {                   // the shares of parts p0 .. p1
                lds_barrier();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const u2 v = p0 == 0 ? ml[i] : row_of(p0 + s0 + 16 * i);
                    const float f = __builtin_amdgcn_exp2f(__uint_as_float(v[0]) - m);
                    if (col < cols) L.share[(s0 + 16 * i) * 16 + col] = f;
                    if (x0 == 0) l += f * __uint_as_float(v[1]);
                }
                lds_barrier();
            }
            if (x < items && grp < groups) {
                for (int s = p0 + grp; s < p1;) {
                    if (x0 != 0 || s != grp) {                   // the next batch
#pragma unroll
                        for (int i = 0; i < EARLY; ++i) early[i] = sum_of(s + i * groups, c, d);
                    }
#pragma unroll
                    for (int i = 0; i < EARLY; ++i, s += groups) {
                        const float f = s < p1 ? L.share[(s - p0) * 16 + c] : 0.f;
                        o.x += f * __uint_as_float(early[i][0]), o.y += f * __uint_as_float(early[i][1]);
                        o.z += f * __uint_as_float(early[i][2]), o.w += f * __uint_as_float(early[i][3]);
                    }
                }
            }
        }
        if (x0 == 0) L.l[s0][col] = l;
        if (groups > 1) L.sum[tid] = o;
        lds_barrier();
        if (grp > 0 || x >= items) continue;
        for (int g = 1; g < groups; ++g) {
            const float4 v = L.sum[g * items + x];
            o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
        }
        float all = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) all += L.l[i][c];
        const float inv = all == 0.f ? 0.f : 1.f / all;
        const long to = out_at<DT>(A, b, h, 16 * tile + c) + d;
        store_f<DT>(A.out, to, o.x * inv), store_f<DT>(A.out, to + 1, o.y * inv);
        store_f<DT>(A.out, to + 2, o.z * inv), store_f<DT>(A.out, to + 3, o.w * inv);
    }
}

template <int NS, int DT>
__global__ __launch_bounds__(64 * WAVES, kv4_waves(NS, DT) == 3 ? 3 : 1) void kv4_attn_kernel(Kv4AttnArgs A) {
    constexpr int TILES = 2 * NS, DP = 32 * NS;
    constexpr bool EXACT = DT == DT_F32;
    constexpr int TERMS = EXACT ? 3 : 1, SUMS = EXACT ? 2 : 1, W_TERMS = EXACT ? 3 : DT == DT_F16 ? 2 : 1;
    constexpr float HEAD = HEADROOM<DT>;
    constexpr int UP = EXACT ? 0 : 22;                 // codes in the products are c 2^-UP
    union Lds {
        float red[2][16][DP + 4];
        CombineLds combine;
        __device__ Lds() {}
    };
    __shared__ __align__(16) Lds lds;
    auto& red = lds.red;
    __shared__ float red_m[WAVES][16], red_l[WAVES][16];
    __shared__ int flag;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const Kv4View& C = A.c;
    const int D = C.d;
    const int group = blockIdx.x;
    Row R;
    R.set(A, lane);
    int x = group * R.piece;
    const int end = min(x + R.piece, R.total);
    for (; x < end; __syncthreads()) {
        const Unit U = unit_at(A, R, x, lane);
        const bool small = U.blocks <= R.whole;
        const int from = max(x - U.start, 0), upto = small ? U.blocks : min(U.blocks, end - U.start);
        // a small unit that starts before the piece is another workgroup's, and so is one whose blocks start behind it
        const bool mine = small ? x == U.start - A.unit_cost : upto > 0;
        x = U.start + max(upto, 0);
        if (!mine) continue;
        const int part_slot = 2 * group + (from == 0 && U.start != group * R.piece ? 1 : 0);
        const int b = U.b, h = U.j / A.tiles, tile = U.j - h * A.tiles;
        const int len = index_at(C.lens, b);
        const int first = from, last = len > 0 && C.num_pages > 0 ? upto : 0;

        // The wave's blocks in turn.  A block without a page counts as unseen; its loads (and those past the last block) go
        // to the pool's first block, so that the loads under way are always as many and a step waits for its own alone.
        Block<NS, EXACT> B;
        auto where = [&](int blk, bool& there) {
            const uint32_t* p = blk < last ? kv4_block(C, b, blk, h) : nullptr;
            there = p != nullptr;
            return there ? p : C.pages;
        };
        int blk = first + wave;
        bool there = false;
        if (blk < last) {
            const uint32_t* p = where(blk, there);
            B.load_k(p, lane);
            B.load_v(p, lane);
        }

        // this lane's query row; its newest visible token
        const int row = 16 * tile + n;
        const int tok = (int)fdiv((uint32_t)row, A.div_group);
        const bool real = row < A.rows;
        const int newest = real ? len - A.t + tok : -1;
        const int all_see = len - A.t + (int)fdiv((uint32_t)(16 * tile), A.div_group);    // every row sees tokens up to here

        // q scaled to below 2^11, and its sum
        Op q[TERMS][NS];
        float cc, cl = 0.f, qsum = 0.f;                // exponents are y cc (+ y cl) + at
        const double c2 = (double)A.scale * 1.44269504088896340736;
        const float cm = __builtin_amdgcn_frexp_mantf((float)c2);
        {
            float x[NS][8];
            float top = 0.f;
            // loads of a row and values that exist, whatever the lane's own, so that all go out at once
            const long at = out_at<DT>(A, b, h, min(row, A.rows - 1));
#pragma unroll
            for (int s = 0; s < NS; ++s) load8<DT>(A.q, at + min(8 * (g * NS + s), D - 8), x[s]);
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const bool has = real && 8 * (g * NS + s) < D;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    x[s][j] = has ? x[s][j] : 0.f;
                    top = fmaxf(top, __builtin_fabsf(x[s][j]));
                }
            }
            top = group_max(top);
            const int e = top > 0.f && top < __builtin_inff() ? __builtin_amdgcn_frexp_expf(top) : 0;   // top < 2^e
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float v = __builtin_ldexpf(x[s][j], 11 - e);
                    if constexpr (EXACT) {
                        in_three(v, q[0][s].h[j], q[1][s].h[j], q[2][s].h[j]);
                    } else {
                        const _Float16 h = (_Float16)((j & 2) ? v * 0.0625f : v);
                        q[0][s].h[j] = h;
                        qsum += (j & 2) ? (float)h * 16.f : (float)h;
                    }
                }
            if constexpr (!EXACT) qsum = group_sum(qsum) * 0x1p-22f;
            // scale log2 e; for fp32 in two terms: its rounding would bend every score by 2^-24 of itself
            const int ce = UP - 11 + e + __builtin_amdgcn_frexp_expf((float)c2);
            cc = fmaxf(__builtin_ldexpf(cm, ce), 0x1p-149f);           // not zero: hidden tokens are -inf times it
            red_l[wave][n] = (float)ce;                // cc is cm 2^ce, kept there until the waves meet
            if constexpr (EXACT) cl = __builtin_ldexpf((float)(c2 - (double)(float)c2), UP - 11 + e);
        }

        f4 acc[TILES * SUMS], accz = {0.f, 0.f, 0.f, 0.f};           // EXACT: whole parts, then the rest 2^11 times
#pragma unroll
        for (int i = 0; i < TILES * SUMS; ++i) acc[i] = f4{0.f, 0.f, 0.f, 0.f};
        float M = LOW, la = 0.f, lb = 0.f;
        // A row with a reference FAR from zero stands apart: its exponents are the rounded score minus M, the largest score
        // alone, and minus E, the largest exponent of a value scale among scores near it (sums of such scores and
        // exponents would not be floats).  far: some row of the wave does.
        float at = HEAD;                               // HEAD - M; of a row apart HEAD - E
        bool apart = !(cc < 0x1p126f), far = __builtin_amdgcn_ballot_w64(apart) != 0;

        while (blk < last) {
            bool next_there;
            const uint32_t* next = where(blk + WAVES, next_there);
            // scores of 8 tokens: y = s (dot - z sum q), and log2 of the probability's factor = cc y
            float y[8], sv[8];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                f4 s = {0.f, 0.f, 0.f, 0.f}, rest = s;
#pragma unroll
                for (int st = 0; st < NS; ++st) {
                    if constexpr (EXACT) {
                        const _Float16 z = (_Float16)(float)(B.kz[i] & 15u);
                        const h2 lo = h2{(_Float16)-256.f, (_Float16)-256.f} - h2{z, z};
                        const h2 hi = h2{(_Float16)-16.f, (_Float16)-16.f} - h2{z, z};
                        const h8 kc = decode_exact(B.k[i][st], lo, hi, lo, hi);
                        s = mfma(kc, q[0][st].v, s);
                        rest = mfma(kc, q[1][st].v, rest);
                        rest = mfma(kc, q[2][st].v, rest);
                    } else {
                        s = mfma(decode(B.k[i][st]), q[0][st].v, s);
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t w = B.km[i][j];
                    y[4 * i + j] = __uint_as_float(w) * (EXACT ? __builtin_fmaf(rest[j], 0x1p-11f, s[j])
                                                             : __builtin_fmaf(-(float)(w & 15u), qsum, s[j]));
                }
            }
            // the next block's keys, under way from here on (kept behind the last use of this one's, in its registers)
            __builtin_amdgcn_sched_barrier(0);
            B.load_k(next, lane);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < 8; ++j) sv[j] = __uint_as_float(B.vm[j >> 2][j & 3]);
            if (!there || 32 * blk + 31 > all_see) {
                const int base = there ? 32 * blk + 4 * g : INT32_MAX / 2;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const bool seen = base + (j & 3) + 16 * (j >> 2) <= newest;
                    y[j] = seen ? y[j] : -__builtin_inff();
                    sv[j] = seen ? sv[j] : 0.f;
                }
            }
            // what score + log2 s' stays below, token by token (the largest of each would pass every real weight by their spread)
            float bound = -__builtin_inff();
#pragma unroll
            for (int j = 0; j < 8; ++j)
                bound = fmaxf(bound, __builtin_fmaf(y[j], cc, (float)max(__builtin_amdgcn_frexp_expf(sv[j]), -90)));
            bound = group_max(bound);
            if (far || __builtin_amdgcn_ballot_w64(bound > M + SLACK) != 0) {
                const bool moves = !apart && bound > M + SLACK, joins = moves && !(__builtin_fabsf(bound) < FAR);
                const float E = apart ? HEAD - at : 0.f;
                float to = moves ? __builtin_ceilf(bound) : M, Eto = 0.f;            // whole: what they scale stays exact
                far = __builtin_amdgcn_ballot_w64(apart || joins) != 0;
                if (__builtin_expect(far, 0)) {
                    const int ce = (int)red_l[wave][n];
                    float top = M;
#pragma unroll
                    for (int j = 0; j < 8; ++j) top = fmaxf(top, __builtin_ldexpf(y[j] * cm, ce));
                    top = group_max(top);
                    int ex = -90;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        ex = max(ex, __builtin_ldexpf(y[j] * cm, ce) >= top - 256.f ? (int)(__float_as_uint(sv[j]) >> 23) - 126 : -90);
                    Eto = fmaxf(group_max((float)ex), apart && M >= top - 256.f ? E : -90.f);
                    apart |= joins;
                    to = apart ? top : to;
                    Eto = apart ? Eto : 0.f;
                    cc = apart ? 1.f : cc, cl = apart ? 0.f : cl;
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[j] = apart ? __builtin_ldexpf(y[j] * cm, ce) - top : y[j];
                }
                const float f = __builtin_amdgcn_exp2f(M - to + (E - Eto));
                M = to;
                at = HEAD - (apart ? Eto : to);
                la *= f, lb *= f;
#pragma unroll
                for (int i = 0; i < TILES * SUMS; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] *= f;
#pragma unroll
                for (int j = 0; j < 4; ++j) accz[j] *= f;
            }
            float w[8];
            if constexpr (EXACT) {
                // The whole part of the exponent apart: with it in one sum the fraction would keep 20 bits.
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float whole = __builtin_rintf(y[j] * cc);
                    const float part = __builtin_fmaf(y[j], cl, __builtin_fmaf(y[j], cc, -whole));
                    const float p = __builtin_ldexpf(__builtin_amdgcn_exp2f(part), (int)fmaxf(whole + at, -1000.f));
                    w[j] = y[j] == -__builtin_inff() ? 0.f : p;
                    la += w[j];
                    w[j] *= sv[j];
                }
            } else {
                const float ma = at, mb = ma - 4.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(y[j], cc, (j & 2) ? mb : ma));
                    if (j & 2) lb += p;
                    else la += p;
                    w[j] = p * sv[j];
                }
            }
            Op wo[W_TERMS], zo;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (EXACT) in_three(w[j], wo[0].h[j], wo[1].h[j], wo[2].h[j]);
                else wo[0].h[j] = (_Float16)w[j];
                if constexpr (W_TERMS == 2) wo[1].h[j] = (_Float16)(w[j] - (float)wo[0].h[j]);
            }
            if constexpr (EXACT) {
                h2 bias[4];                                // of tokens (0, 1), (2, 3), (4, 5), (6, 7)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const h2 z = {(_Float16)(float)(B.vm[i >> 1][2 * (i & 1)] & 15u),
                                  (_Float16)(float)(B.vm[i >> 1][2 * (i & 1) + 1] & 15u)};
                    const _Float16 lead = (_Float16)(i & 1 ? -16.f : -256.f);
                    bias[i] = h2{lead, lead} - z;
                }
#pragma unroll
                for (int i = 0; i < TILES; ++i) {
                    const h8 vc = decode_exact(B.v[i], bias[0], bias[1], bias[2], bias[3]);
                    acc[i] = mfma(vc, wo[0].v, acc[i]);
                    acc[TILES + i] = mfma(vc, wo[1].v, acc[TILES + i]);
                    acc[TILES + i] = mfma(vc, wo[2].v, acc[TILES + i]);
                }
            } else {
                // zero points as codes: pairs (0,1), (4,5) plain, (2,3), (6,7) 16-fold
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    zo.u[2 * i] = (__builtin_amdgcn_perm(B.vm[i][1], B.vm[i][0], 0x0C040C00u) & 0x000F000Fu) << 2;
                    zo.u[2 * i + 1] = (__builtin_amdgcn_perm(B.vm[i][3], B.vm[i][2], 0x0C040C00u) & 0x000F000Fu) << 6;
                }
                accz = mfma(zo.v, wo[0].v, accz);
                if constexpr (W_TERMS == 2) accz = mfma(zo.v, wo[1].v, accz);
#pragma unroll
                for (int i = 0; i < TILES; ++i) {
                    const h8 vc = decode(B.v[i]);
                    acc[i] = mfma(vc, wo[0].v, acc[i]);
                    if constexpr (W_TERMS == 2) acc[i] = mfma(vc, wo[1].v, acc[i]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            B.load_v(next, lane);
            blk += WAVES;
            there = next_there;
        }

        // the waves' rows meet
        float l = group_sum(__builtin_fmaf(16.f, lb, la));
        if constexpr (EXACT) {
#pragma unroll
            for (int i = 0; i < TILES; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_fmaf(acc[TILES + i][j], 0x1p-11f, acc[i][j]);
        }
        if (__builtin_expect(far, 0)) {                    // rows apart: sums at the reference M + HEAD alone
            const int e = apart ? -(int)at : 0;
            M += apart ? HEAD : 0.f;
            l = __builtin_ldexpf(l, e);
#pragma unroll
            for (int i = 0; i < TILES; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_ldexpf(acc[i][j], e);
#pragma unroll
            for (int j = 0; j < 4; ++j) accz[j] = __builtin_ldexpf(accz[j], e);
        }
        if (g == 0) red_m[wave][n] = M, red_l[wave][n] = l;
        __syncthreads();
        float top = red_m[0][n];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) top = fmaxf(top, red_m[w][n]);
        const float f = __builtin_amdgcn_exp2f(M - top) * (EXACT ? 1.f : 0x1p22f);
#pragma unroll
        for (int turn = 0; turn < 2; ++turn) {             // waves 0 and 1 write, 2 and 3 add
            if ((wave >> 1) == turn) {
#pragma unroll
                for (int i = 0; i < TILES; ++i) {
                    float4* at = reinterpret_cast<float4*>(&red[wave & 1][n][16 * i + 4 * g]);
                    float4 o = turn ? *at : float4{0.f, 0.f, 0.f, 0.f};
                    o.x += (acc[i][0] - accz[0]) * f, o.y += (acc[i][1] - accz[0]) * f;
                    o.z += (acc[i][2] - accz[0]) * f, o.w += (acc[i][3] - accz[0]) * f;
                    *at = o;
                }
            }
            __syncthreads();
        }
        const bool all = from == 0 && upto == U.blocks;
        const int cols = min(16, A.rows - 16 * tile);
        for (int y = threadIdx.x; y < cols * (D >> 2); y += 64 * WAVES) {
            const int c = y / (D >> 2), d = (y - c * (D >> 2)) * 4;
            float o[4], ls = 0.f, mt = red_m[0][c];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) mt = fmaxf(mt, red_m[w][c]);
#pragma unroll
            for (int w = 0; w < WAVES; ++w) ls += red_l[w][c] * __builtin_amdgcn_exp2f(red_m[w][c] - mt);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = red[0][c][d + i] + red[1][c][d + i];
            if (all) {
                const float inv = ls == 0.f ? 0.f : 1.f / ls;
                const long at = out_at<DT>(A, b, h, 16 * tile + c) + d;
#pragma unroll
                for (int i = 0; i < 4; ++i) store_f<DT>(A.out, at + i, o[i] * inv);
            } else {
                const __amdgpu_buffer_rsrc_t buf = buffer_of(part_sums(A, part_slot), (long)A.cols * D);
                const u4 v = {__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3])};
                __builtin_amdgcn_raw_buffer_store_b128(v, buf, (c * D + d) * 4, 0, SC1);
                if (d == 0) {
                    float* r = part_rows(A, part_slot) + 2 * c;
                    partial_put(r, mt), partial_put(r + 1, ls);
                }
            }
        }
        if (all || !A.split_cnt) continue;
        const Parts P = parts_of(R, U);
        if (split_arrive(A.split_cnt + P.first, P.count, &flag)) combine<DT>(A, lds.combine, P, b, h, tile);
    }
}

// The combine as a launch of its own, for calls without counters: a workgroup joins the unit that the end of its
// piece cuts, if its first part is there.
template <int DT>
__global__ __launch_bounds__(64 * WAVES) void kv4_combine_kernel(Kv4AttnArgs A) {
    __shared__ __align__(16) CombineLds lds;
    const int lane = threadIdx.x & 63, group = blockIdx.x;
    Row R;
    R.set(A, lane);
    const int end = (group + 1) * R.piece;
    if (end >= R.total) return;
    const Unit U = unit_at(A, R, end - 1, lane);
    if (U.blocks <= R.whole || U.start + U.blocks <= end || U.start >= end || U.start < group * R.piece) return;
    const int h = U.j / A.tiles;
    combine<DT>(A, lds, parts_of(R, U), U.b, h, U.j - h * A.tiles);
}

template <int NS>
const void* kernel_for(int dt) {
    return dt == DT_F16 ? (const void*)kv4_attn_kernel<NS, DT_F16>
         : dt == DT_BF16 ? (const void*)kv4_attn_kernel<NS, DT_BF16> : (const void*)kv4_attn_kernel<NS, DT_F32>;
}

}  // namespace

hipError_t launch_kv4_attn(const Kv4AttnArgs& A, int dt, hipStream_t stream) {
    static const void* (*const table[8])(int) = {kernel_for<1>, kernel_for<2>, kernel_for<3>, kernel_for<4>,
                                                 kernel_for<5>, kernel_for<6>, kernel_for<7>, kernel_for<8>};
    const void* f = table[A.c.ns - 1](dt);
    Kv4AttnArgs a = A;
    void* args[] = {&a};
    hipError_t e = launch(f, dim3(A.groups), dim3(64 * WAVES), args, 0, stream);
    if (e != hipSuccess || !A.partial || A.split_cnt) return e;
    f = dt == DT_F16 ? (const void*)kv4_combine_kernel<DT_F16>
      : dt == DT_BF16 ? (const void*)kv4_combine_kernel<DT_BF16> : (const void*)kv4_combine_kernel<DT_F32>;
    return launch(f, dim3(A.groups), dim3(64 * WAVES), args, 0, stream);
}

}  // namespace cbk
