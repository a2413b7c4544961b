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

__device__ __forceinline__ f4 mfma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// The largest over the four lane groups (lanes l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float group_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float group_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// One block's words as a lane holds them.
template <int NS>
struct Block {
    uint32_t k[2][NS];
    uint32_t v[2 * NS];
    u4 km[2], vm[2];

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

// The partials of a (sequence, head, row tile): A.splits times [cols][D + 2], the row's sums, its
// reference M and its sum of p.
__device__ __forceinline__ float* partial_of(const Kv4AttnArgs& A, int unit, int split) {
    return A.partial + ((long)unit * A.splits + split) * A.cols * (A.c.d + 2);
}

template <int DT>
__device__ __forceinline__ long out_at(const Kv4AttnArgs& A, int b, int h, int row) {
    const int i = (int)fdiv((uint32_t)row, A.div_group);
    return (((long)b * A.t + i) * A.hq + h * A.group + (row - i * A.group)) * A.c.d;
}

// Adds the active workgroups' partials of a unit, in order, and writes its rows.
template <int DT>
__device__ __forceinline__ void combine(const Kv4AttnArgs& A, int unit, int b, int h, int tile, int active) {
    const int D = A.c.d, cols = min(A.cols, A.rows - 16 * tile);
    const long stride = (long)A.cols * (D + 2);
    for (int x = threadIdx.x; x < cols * (D >> 2); x += blockDim.x) {
        const int c = x / (D >> 2), d = (x - c * (D >> 2)) * 4;
        const float* p = partial_of(A, unit, 0) + (long)c * (D + 2);
        float m = LOW;
        for (int s = 0; s < active; ++s) m = fmaxf(m, partial_get(p + s * stride + D));
        float o[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
        for (int s = 0; s < active; ++s) {
            const float* q = p + s * stride;
            const float f = __builtin_amdgcn_exp2f(partial_get(q + D) - m);
            l += f * partial_get(q + D + 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += f * partial_get(q + d + i);
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const long at = out_at<DT>(A, b, h, 16 * tile + c) + d;
#pragma unroll
        for (int i = 0; i < 4; ++i) store_f<DT>(A.out, at + i, o[i] * inv);
    }
}

template <int NS, int DT>
__global__ __launch_bounds__(64 * WAVES) void kv4_attn_kernel(Kv4AttnArgs A) {
    constexpr int TILES = 2 * NS, DP = 32 * NS;
    constexpr int TERMS = DT == DT_F32 ? 2 : 1;
    __shared__ __align__(16) float red[2][16][DP + 4];
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
                const float u = (j & 2) ? v * 0.0625f : v;
                const _Float16 hi = (_Float16)u;
                q[0][s].h[j] = hi;
                float held = (float)hi;
                if constexpr (TERMS == 2) {
                    const _Float16 lo = (_Float16)(u - held);
                    q[1][s].h[j] = lo;
                    held += (float)lo;
                }
                qsum += (j & 2) ? held * 16.f : held;
            }
        qsum = group_sum(qsum) * 0x1p-22f;
        cc = __builtin_ldexpf(A.scale * 1.44269504088896341f, 22 - 11 + e);
    }

    f4 acc[TILES], accz = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < TILES; ++i) acc[i] = f4{0.f, 0.f, 0.f, 0.f};
    float M = LOW, la = 0.f, lb = 0.f;

    auto step = [&](const Block<NS>& B, int blk) {
        // scores of 8 tokens: y = s (dot - z sum q), and log2 of the probability's factor = cc y
        float y[8], sv[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < NS; ++st) {
                const h8 kc = decode(B.k[i][st]);
                s = mfma(kc, q[0][st].v, s);
                if constexpr (TERMS == 2) s = mfma(kc, q[1][st].v, s);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t w = B.km[i][j];
                y[4 * i + j] = __uint_as_float(w) * __builtin_fmaf(-(float)(w & 15u), qsum, s[j]);
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
        const float ma = HEADROOM - M, mb = HEADROOM - 4.f - M;
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
        // zero points as codes: pairs (0,1), (4,5) plain, (2,3), (6,7) 16-fold
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            zo.u[2 * i] = (__builtin_amdgcn_perm(B.vm[i][1], B.vm[i][0], 0x0C040C00u) & 0x000F000Fu) << 2;
            zo.u[2 * i + 1] = (__builtin_amdgcn_perm(B.vm[i][3], B.vm[i][2], 0x0C040C00u) & 0x000F000Fu) << 6;
        }
#pragma unroll
        for (int t = 0; t < TERMS; ++t) accz = mfma(zo.v, wo[t].v, accz);
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            const h8 vc = decode(B.v[i]);
#pragma unroll
            for (int t = 0; t < TERMS; ++t) acc[i] = mfma(vc, wo[t].v, acc[i]);
        }
    };

    // the wave's blocks, one ahead; a block without a page is left out
    {
        Block<NS> cur, nxt;
        int blk = first + wave;
        const uint32_t* p = blk < last ? kv4_block(C, b, blk, h) : nullptr;
        if (p) cur.load(p, lane);
        while (blk < last) {
            const int ahead = blk + WAVES;
            const uint32_t* pn = ahead < last ? kv4_block(C, b, ahead, h) : nullptr;
            if (pn) nxt.load(pn, lane);
            if (p) step(cur, blk);
            cur = nxt;
            p = pn;
            blk = ahead;
        }
    }

    // the waves' rows meet
    float l = group_sum(__builtin_fmaf(16.f, lb, la));
    if (g == 0) red_m[wave][n] = M, red_l[wave][n] = l;
    __syncthreads();
    float top = red_m[0][n];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) top = fmaxf(top, red_m[w][n]);
    const float f = __builtin_amdgcn_exp2f(M - top) * 0x1p22f;
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
            float* p = partial_of(A, unit, split) + (long)c * (D + 2);
#pragma unroll
            for (int i = 0; i < 4; ++i) partial_put(p + d + i, o[i]);
            if (d == 0) partial_put(p + D, mt), partial_put(p + D + 1, ls);
        }
    }
    if (active == 1 || !A.split_cnt) return;
    if (split_arrive(A.split_cnt + unit, active, &flag)) combine<DT>(A, unit, b, h, tile, active);
}

// The combine as a launch of its own, for calls without counters.
template <int DT>
__global__ __launch_bounds__(64 * WAVES) void kv4_combine_kernel(Kv4AttnArgs A) {
    const int tile = blockIdx.y / A.c.heads, h = blockIdx.y - tile * A.c.heads, b = blockIdx.z;
    int blocks, per, active;
    shares(A, A.c.lens[b], blocks, per, active);
    if (active > 1) combine<DT>(A, (b * A.c.heads + h) * A.tiles + tile, b, h, tile, active);
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
