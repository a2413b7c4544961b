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
// bf16 q (fp32 q and w go as two fp16 terms each); where the stored pairs count 16 times, q is held / 16, and
// w takes the 1/16 in its exponent.  w must fit fp16 at any scale s': the running reference M of a row
// bounds score + log2 s' over the tokens seen, w = 2^(score - M + 12) s', so that w < 2^16 and 26 bits
// below the largest still count; the sum of p is held with the same factor.  M moves only when it would
// have to by 3 or more (the accumulators are rescaled then).
//
// A sequence's blocks go to `splits` workgroups of four waves at most (min_blocks each at least; counted
// from the length on the device), whose waves take them in turn, the next block's loads under way; waves meet in LDS, workgroups through fp32 partials
// and an arrival counter (or a second launch), in a fixed order.
#include "kv4.hpp"
#include "cbk_kernels.hpp"

namespace cbk {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int WAVES = 4;
constexpr float LOW = -1e30f;          // reference of a row that has seen nothing
constexpr float HEADROOM = 12.f;       // w < 2^(HEADROOM + 3 + 1)
constexpr float SLACK = 3.f;

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

// One block's words as a lane holds them.
template <int NS, bool EXACT>
struct Block {
    uint32_t k[2][NS];
    uint32_t v[2 * NS];
    u4 km[2], vm[2];
    uint32_t kz[2];                    // EXACT: the words of the tokens whose codes this lane decodes

    __device__ __forceinline__ void load(const uint32_t* p, int lane) {
        constexpr int PW = kv4_piece(NS);
        const uint32_t* kp = p + (lane & 15) * 4 * NS + (lane >> 4) * NS;
#pragma unroll
        for (int i = 0; i < 2; ++i) __builtin_memcpy(k[i], kp + i * 64 * NS, 4 * NS);
        const uint32_t* vp = p + 128 * NS + lane * PW;
#pragma unroll
        for (int i = 0; i < 2 * NS / PW; ++i) __builtin_memcpy(v + i * PW, vp + i * 64 * PW, 4 * PW);
        const u4* mp = reinterpret_cast<const u4*>(p + 256 * NS) + (lane >> 4);
        km[0] = mp[0], km[1] = mp[4], vm[0] = mp[8], vm[1] = mp[12];
        if constexpr (EXACT) kz[0] = p[256 * NS + (lane & 15)], kz[1] = p[256 * NS + 16 + (lane & 15)];
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

// Workgroups that share sequence b's blocks, and the blocks each takes.
__device__ __forceinline__ void shares(const Kv4AttnArgs& A, int len, int& blocks, int& per, int& active) {
    const int room = min((long)A.c.width << A.c.page_shift, (long)1 << 26);
    blocks = min((max(len, 0) + 31) >> 5, room);
    per = max((blocks + A.splits - 1) / A.splits, A.min_blocks);
    active = max((blocks + per - 1) / per, 1);
}

// The partials of a (sequence, head, row tile) and split: [cols][D] sums, and behind those of all units
// [cols][2], each row's reference M and sum of p.  They pass between workgroups on any XCD: written and read
// past the L2s (sc1), as split_arrive's note says.
constexpr int SC1 = 16;
__device__ __forceinline__ long part_sums(const Kv4AttnArgs& A, int unit, int split) {
    return ((long)unit * A.splits + split) * A.cols * A.c.d;
}
__device__ __forceinline__ float* part_rows(const Kv4AttnArgs& A, int unit, int split) {
    const long units = (long)A.c.seqs * A.c.heads * A.tiles;
    return A.partial + units * A.splits * A.cols * A.c.d + ((long)unit * A.splits + split) * A.cols * 2;
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const float* p, long floats) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(p), 0, (int)min(floats * 4, (long)0x7FFFFFF0), 0x00027000);
}

template <int DT>
__device__ __forceinline__ long out_at(const Kv4AttnArgs& A, int b, int h, int row) {
    const int i = (int)fdiv((uint32_t)row, A.div_group);
    return (((long)b * A.t + i) * A.hq + h * A.group + (row - i * A.group)) * A.c.d;
}

// LDS of the combine: what each split's row counts for, and the sums of the thread groups.
struct CombineLds {
    float share[KV4_MAX_SPLITS * 16];
    float m[16][16], l[16][16];
    float4 sum[64 * WAVES];
};

// Adds the active workgroups' partials of a unit, in order, and writes its rows.  Threads share the splits: all
// loads of a thread are independent.
template <int DT>
__device__ __forceinline__ void combine(const Kv4AttnArgs& A, CombineLds& L, int unit, int b, int h, int tile, int active) {
    const int D = A.c.d, cols = min(A.cols, A.rows - 16 * tile), tid = threadIdx.x;
    {
        const int c = tid & 15, s0 = tid >> 4;
        const float* r = part_rows(A, unit, 0) + 2 * c;
        float m = LOW, l = 0.f;
        if (c < cols)
            for (int s = s0; s < active; s += 16) m = fmaxf(m, partial_get(r + (long)s * A.cols * 2));
        L.m[s0][c] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; ++i) m = fmaxf(m, L.m[i][c]);
        if (c < cols)
            for (int s = s0; s < active; s += 16) {
                const float* q = r + (long)s * A.cols * 2;
                const float f = __builtin_amdgcn_exp2f(partial_get(q) - m);
                L.share[s * cols + c] = f;
                l += f * partial_get(q + 1);
            }
        L.l[s0][c] = l;
        __syncthreads();
    }
    const int items = cols * (D >> 2), stride = A.cols * D * 4;
    const int groups = max(1, 64 * WAVES / items);               // thread groups that share the splits
    const __amdgpu_buffer_rsrc_t buf = buffer_of(A.partial + part_sums(A, unit, 0), (long)active * A.cols * D);
    for (int x0 = 0; x0 < items; x0 += 64 * WAVES) {
        const int grp = groups > 1 ? tid / items : 0, x = groups > 1 ? tid - grp * items : x0 + tid;
        const int c = x / (D >> 2), d = (x - c * (D >> 2)) * 4;
        float4 o = {0.f, 0.f, 0.f, 0.f};
        if (x < items && grp < groups) {
            const int at = (c * D + d) * 4;
#pragma unroll 8
            for (int s = grp; s < active; s += groups) {
                const u4 v = __builtin_amdgcn_raw_buffer_load_b128(buf, at + s * stride, 0, SC1);
                const float f = L.share[s * cols + c];
                o.x += f * __uint_as_float(v[0]), o.y += f * __uint_as_float(v[1]);
                o.z += f * __uint_as_float(v[2]), o.w += f * __uint_as_float(v[3]);
            }
        }
        if (groups > 1) {
            L.sum[tid] = o;
            __syncthreads();
            if (grp != 0) return;
            for (int g = 1; g < groups; ++g) {
                const float4 v = L.sum[g * items + x];
                o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
            }
        }
        if (x >= items) continue;
        float l = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) l += L.l[i][c];
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const long at = out_at<DT>(A, b, h, 16 * tile + c) + d;
        store_f<DT>(A.out, at, o.x * inv), store_f<DT>(A.out, at + 1, o.y * inv);
        store_f<DT>(A.out, at + 2, o.z * inv), store_f<DT>(A.out, at + 3, o.w * inv);
    }
}

template <int NS, int DT>
__global__ __launch_bounds__(64 * WAVES) void kv4_attn_kernel(Kv4AttnArgs A) {
    constexpr int TILES = 2 * NS, DP = 32 * NS;
    constexpr bool EXACT = DT == DT_F32;
    constexpr int TERMS = EXACT ? 2 : 1;
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
    const int split = blockIdx.x, tile = blockIdx.y / C.heads, h = blockIdx.y - tile * C.heads, b = blockIdx.z;
    const int len = C.lens[b];
    int blocks, per, active;
    shares(A, len, blocks, per, active);
    if (split >= active) return;
    const int first = split * per, last = min(first + per, blocks);
    const int D = C.d;

    // this lane's query row; its newest visible token
    const int row = 16 * tile + n;
    const int tok = (int)fdiv((uint32_t)row, A.div_group);
    const bool real = row < A.rows;
    const int newest = real ? len - A.t + tok : -1;
    const int all_see = len - A.t + (int)fdiv((uint32_t)(16 * tile), A.div_group);    // every row sees tokens up to here

    // q scaled to below 2^11, and its sum
    Op q[TERMS][NS];
    float cc, qsum = 0.f;
    {
        float x[NS][8];
        float top = 0.f;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int d = 8 * (g * NS + s);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[s][j] = 0.f;
            if (real && d < D) load8<DT>(A.q, out_at<DT>(A, b, h, row) + d, x[s]);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, __builtin_fabsf(x[s][j]));
        }
        top = group_max(top);
        const int e = top > 0.f && top < __builtin_inff() ? __builtin_amdgcn_frexp_expf(top) : 0;   // top < 2^e
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float v = __builtin_ldexpf(x[s][j], 11 - e);
                const float u = !EXACT && (j & 2) ? v * 0.0625f : v;
                const _Float16 hi = (_Float16)u;
                q[0][s].h[j] = hi;
                float held = (float)hi;
                if constexpr (TERMS == 2) {
                    const _Float16 lo = (_Float16)(u - held);
                    q[1][s].h[j] = lo;
                    held += (float)lo;
                }
                if constexpr (!EXACT) qsum += (j & 2) ? held * 16.f : held;
            }
        if constexpr (!EXACT) qsum = group_sum(qsum) * 0x1p-22f;
        cc = __builtin_ldexpf(A.scale * 1.44269504088896341f, UP - 11 + e);
    }

    f4 acc[TILES], accz = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < TILES; ++i) acc[i] = f4{0.f, 0.f, 0.f, 0.f};
    float M = LOW, la = 0.f, lb = 0.f;

    auto step = [&](const Block<NS, EXACT>& B, int blk) {
        // scores of 8 tokens: y = s (dot - z sum q), and log2 of the probability's factor = cc y
        float y[8], sv[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < NS; ++st) {
                if constexpr (EXACT) {
                    const _Float16 z = (_Float16)(float)(B.kz[i] & 15u);
                    const h2 lo = h2{(_Float16)-256.f, (_Float16)-256.f} - h2{z, z};
                    const h2 hi = h2{(_Float16)-16.f, (_Float16)-16.f} - h2{z, z};
                    const h8 kc = decode_exact(B.k[i][st], lo, hi, lo, hi);
                    s = mfma(kc, q[0][st].v, s);
                    s = mfma(kc, q[1][st].v, s);
                } else {
                    s = mfma(decode(B.k[i][st]), q[0][st].v, s);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t w = B.km[i][j];
                y[4 * i + j] = __uint_as_float(w) * (EXACT ? s[j] : __builtin_fmaf(-(float)(w & 15u), qsum, s[j]));
                sv[4 * i + j] = __uint_as_float(B.vm[i][j]);
            }
        }
        const int base = 32 * blk + 4 * g;
        if (32 * blk + 31 > all_see) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool seen = base + (j & 3) + 16 * (j >> 2) <= newest;
                y[j] = seen ? y[j] : -__builtin_inff();
                sv[j] = seen ? sv[j] : 0.f;
            }
        }
        float ym = y[0], sm = sv[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) ym = fmaxf(ym, y[j]), sm = fmaxf(sm, sv[j]);
        // score + log2 s' is below this for every token of the lane
        float bound = ym * cc + (float)max(__builtin_amdgcn_frexp_expf(sm), -90);
        bound = group_max(bound);
        if (__builtin_amdgcn_ballot_w64(bound > M + SLACK) != 0) {
            const float to = bound > M + SLACK ? bound : M;
            const float f = __builtin_amdgcn_exp2f(M - to);
            M = to;
            la *= f, lb *= f;
#pragma unroll
            for (int i = 0; i < TILES; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] *= f;
#pragma unroll
            for (int j = 0; j < 4; ++j) accz[j] *= f;
        }
        const float ma = HEADROOM - M, mb = EXACT ? ma : HEADROOM - 4.f - M;
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(y[j], cc, (j & 2) ? mb : ma));
            if (j & 2) lb += p;
            else la += p;
            w[j] = p * sv[j];
        }
        Op wo[TERMS], zo;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            wo[0].h[j] = (_Float16)w[j];
            if constexpr (TERMS == 2) wo[1].h[j] = (_Float16)(w[j] - (float)wo[0].h[j]);
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
                acc[i] = mfma(vc, wo[1].v, acc[i]);
            }
        } else {
            // zero points as codes: pairs (0,1), (4,5) plain, (2,3), (6,7) 16-fold
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                zo.u[2 * i] = (__builtin_amdgcn_perm(B.vm[i][1], B.vm[i][0], 0x0C040C00u) & 0x000F000Fu) << 2;
                zo.u[2 * i + 1] = (__builtin_amdgcn_perm(B.vm[i][3], B.vm[i][2], 0x0C040C00u) & 0x000F000Fu) << 6;
            }
            accz = mfma(zo.v, wo[0].v, accz);
#pragma unroll
            for (int i = 0; i < TILES; ++i) acc[i] = mfma(decode(B.v[i]), wo[0].v, acc[i]);
        }
    };

    // the wave's blocks in turn, two sets of registers; a block without a page is left out
    {
        Block<NS, EXACT> one, two;
        auto fetch = [&](Block<NS, EXACT>& B, int blk) {
            const uint32_t* p = blk < last ? kv4_block(C, b, blk, h) : nullptr;
            if (p) B.load(p, lane);
            return p != nullptr;
        };
        int blk = first + wave;
        bool has_one = fetch(one, blk), has_two;
        while (blk < last) {
            has_two = fetch(two, blk + WAVES);
            if (has_one) step(one, blk);
            blk += WAVES;
            if (blk >= last) break;
            has_one = fetch(one, blk + WAVES);
            if (has_two) step(two, blk);
            blk += WAVES;
        }
    }

    // the waves' rows meet
    float l = group_sum(EXACT ? la + lb : __builtin_fmaf(16.f, lb, la));
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
    const int unit = (b * C.heads + h) * A.tiles + tile;
    const int cols = min(16, A.rows - 16 * tile);
    for (int x = threadIdx.x; x < cols * (D >> 2); x += 64 * WAVES) {
        const int c = x / (D >> 2), d = (x - c * (D >> 2)) * 4;
        float o[4], ls = 0.f, mt = red_m[0][c];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) mt = fmaxf(mt, red_m[w][c]);
#pragma unroll
        for (int w = 0; w < WAVES; ++w) ls += red_l[w][c] * __builtin_amdgcn_exp2f(red_m[w][c] - mt);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = red[0][c][d + i] + red[1][c][d + i];
        if (active == 1) {
            const float inv = ls == 0.f ? 0.f : 1.f / ls;
            const long at = out_at<DT>(A, b, h, 16 * tile + c) + d;
#pragma unroll
            for (int i = 0; i < 4; ++i) store_f<DT>(A.out, at + i, o[i] * inv);
        } else {
            const __amdgpu_buffer_rsrc_t buf = buffer_of(A.partial + part_sums(A, unit, split), (long)A.cols * D);
            const u4 v = {__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3])};
            __builtin_amdgcn_raw_buffer_store_b128(v, buf, (c * D + d) * 4, 0, SC1);
            if (d == 0) {
                float* r = part_rows(A, unit, split) + 2 * c;
                partial_put(r, mt), partial_put(r + 1, ls);
            }
        }
    }
    if (active == 1 || !A.split_cnt) return;
    if (split_arrive(A.split_cnt + unit, active, &flag)) combine<DT>(A, lds.combine, unit, b, h, tile, active);
}

// The combine as a launch of its own, for calls without counters.
template <int DT>
__global__ __launch_bounds__(64 * WAVES) void kv4_combine_kernel(Kv4AttnArgs A) {
    __shared__ __align__(16) CombineLds lds;
    const int tile = blockIdx.y / A.c.heads, h = blockIdx.y - tile * A.c.heads, b = blockIdx.z;
    int blocks, per, active;
    shares(A, A.c.lens[b], blocks, per, active);
    if (active > 1) combine<DT>(A, lds, (b * A.c.heads + h) * A.tiles + tile, b, h, tile, active);
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
    const dim3 units(1, A.c.heads * A.tiles, A.c.seqs);
    hipError_t e = launch(f, dim3(A.splits, units.y, units.z), dim3(64 * WAVES), args, 0, stream);
    if (e != hipSuccess || A.splits == 1 || A.split_cnt) return e;
    f = dt == DT_F16 ? (const void*)kv4_combine_kernel<DT_F16>
      : dt == DT_BF16 ? (const void*)kv4_combine_kernel<DT_BF16> : (const void*)kv4_combine_kernel<DT_F32>;
    return launch(f, units, dim3(64 * WAVES), args, 0, stream);
}

}  // namespace cbk
