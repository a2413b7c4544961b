// prompt_attn.hip -- causal attention over packed prompts, fp16 / bf16, on the 16-bit matrix cores.
//
// Row i of a sequence sees its rows 0 .. i; query head h reads kv head h / group.  One pass over the keys with
// the running maximum and sum of the softmax: per tile of 64 tokens
//   S^T[token, row] = K q^T,  w = 2^(scale log2e S - M),  O^T[d, row] += V^T w
// A workgroup has 128 rows of one head (32 a wave) and stages K and V tiles in LDS, the next tile's loads under
// way.  v_mfma_f32_32x32x16 gives a lane one row's column of S^T (tokens 8 i + 4 (lane / 32) + 0..3), which is the
// operand layout of w for the tokens in that order, so w stays in its lane; V^T is read transposed from LDS
// (ds_read_b64_tr_b16) in the same token order.  The running reference M of a row moves only when a tile's
// largest score exceeds it by 8 (w <= 2^8 then, 2^15 in fp16, in range; sums are fp32), and stays a whole number, so that what it
// scales is exact.  w is rounded to the type (nearest even), as the products take both operands in V's type: an output's
// error is 2.1e-3 then in bf16 and 2.5e-4 in fp16, its own rounding alone 1.6e-3 and 2.0e-4; a second term would be half as many
// products again, of a kernel bound by them.  l sums the rounded w, so that the rounding cancels where values agree.
//
// Bound: a tile of a wave costs 32 matrix instructions of 32 cycles (D = 128) and about as many cycles of vector
// instructions (the softmax's, the same for any D); two waves a SIMD overlap them in part.  8192 rows, 32/8 heads, bf16:
// 560 us, 0.98 PFLOP/s of the 1.22 that a large matrix product reaches (554 to 573 by card); three waves a SIMD (six a
// workgroup) were a tenth slower.
//
// Masked places take no part whatever they hold: scores there are selected away, and a V tile on the diagonal
// that has infinities or NaN (a product 0 x inf would reach rows that do not see it) is left for a second pass, with those
// values zeroed, and what a row sees of them is added at the end.  (A visible infinity whose weight is below the type's
// smallest gives NaN in a whole tile, 0 x inf, and the infinity in one on the diagonal: not finite either way.)
#include "kv4.hpp"
#include "cbk_kernels.hpp"

namespace cbk {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int WAVES = 4;
constexpr int ROWS = 32 * WAVES;       // query rows of a workgroup
constexpr int KT = 64;                 // tokens of a tile
constexpr float LOW = -0x1.fffffep127f;        // reference of a row that has seen nothing
constexpr float SLACK = 8.f;
// Weights stand 2^UP above their reference: fp16 uses its range up to 2^15, so that what is denormal, or lost, lies 2^-20, or
// 2^-31, below the largest weight rather than 2^-13 and 2^-24 (thirty thousand tokens of 2^-25 each count)
template <int DT>
constexpr float UP = DT == DT_F16 ? 7.f : 0.f;

template <int DT>
__device__ __forceinline__ f16v mfma(u4 a, u4 b, f16v c) {
    if constexpr (DT == DT_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// Two values rounded to the type (nearest even), packed.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    if constexpr (DT == DT_F16) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, h2{(_Float16)x, (_Float16)y});
    } else {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, b2{(__bf16)x, (__bf16)y});
    }
}

// A value of the type (in the low half) as a float.
template <int DT>
__device__ __forceinline__ float half_of(uint32_t v) {
    return Dt<DT>::to_f(__builtin_bit_cast(typename Dt<DT>::S, (uint16_t)v));
}

// l plus the two values of a packed pair, in one instruction (fp32, denormals kept).
template <int DT>
__device__ __forceinline__ float plus_both(uint32_t pair, float l) {
    if constexpr (DT == DT_F16) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, pair), h2{(_Float16)1.f, (_Float16)1.f}, l, false);
    } else {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, pair), b2{(__bf16)1.f, (__bf16)1.f}, l, false);
    }
}

__device__ __forceinline__ f16v zero16() {
    f16v z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}

typedef __attribute__((address_space(3))) void* lds_ptr;
typedef const __attribute__((address_space(3))) u4* lds_u4;
typedef __attribute__((address_space(3))) s4* lds_s4;

// Where a tile's row r keeps its 16-byte chunk c, in chunks.  A wave reads, of K, two neighbouring chunks of 32 rows at
// once, of V four neighbouring chunks of eight rows: either way the places cover the 64 banks evenly.  Rows have CP
// chunks, a power of two, turned against each other by an exclusive or, or twelve (80 and 96 values: three
// workgroups' tiles fit the LDS instead of two), whose pitch sets four rows apart by itself.
template <int CP>
__device__ __forceinline__ int k_place(int r, int c) {
    if constexpr (CP == 12) return r * 12 + (c + 2 * (r >> 2 & 1)) % 12;
    return r * CP + (c ^ (CP >= 16 ? (r & 7) << 1 : CP == 8 ? (r >> 1 & 3) << 1 : (r >> 2 & 1) << 1));
}
template <int CP>
__device__ __forceinline__ int v_place(int r, int c) {
    return r * CP + (c ^ (CP >= 16 ? (r & 3) << 2 : CP == 8 ? (r >> 1 & 1) << 2 : 0));
}

// A buffer over a sequence's rows (len of them, `stride` elements apart, D values each) from tile t on.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_from(const uint16_t* base, long stride, int t, int len, int D) {
    const long left = len - t * KT;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base + (long)t * KT * stride), 0,
                                             (int)min(((left - 1) * stride + D) * 2, 0x7FFFFF00l), 0x00020000);
}

// 16 bytes a lane from the buffer to LDS, the lanes' behind each other from `to` on.  All of the offset is the lane's: the
// range check need not count a scalar offset.
__device__ __forceinline__ void load_chunks(__amdgpu_buffer_rsrc_t from, uint32_t to, uint32_t offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_ptr)to, 16, offset, 0, 0, 0);
}

// KS: steps of 16 of the head's values, DT32: tiles of 32, CP: chunks of a row in LDS.
template <int DT, int KS, int CP>
__global__ __launch_bounds__(64 * WAVES, CP == 32 ? 1 : CP == 16 ? 2 : 3) void prompt_attn_kernel(PromptArgs A, int row_tiles) {
    constexpr int DT32 = (KS + 1) / 2;
    constexpr int TILE = KT * CP * 16;                 // bytes of a K or V tile
    auto not_finite = [](uint32_t v) {                 // all ones in each 16-bit half that is an infinity or NaN
        constexpr uint32_t EX = DT == DT_F16 ? 0x7C00u : 0x7F80u;
        return ((v & EX) == EX ? 0xFFFFu : 0u) | ((v >> 16 & EX) == EX ? 0xFFFF0000u : 0u);
    };
    extern __shared__ __align__(16) char lds[];        // [2][K tile, V tile]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, hf = lane >> 5;

    // kv heads innermost: with the workgroups dealt out to the XCDs in turn, a kv head's tiles stay on one; the
    // longest rows' tiles first
    int id = blockIdx.x;
    const int hk = id % A.hkv;
    id /= A.hkv;
    const int h = hk * A.group + id % A.group;
    id /= A.group;
    const int b = id % (A.seqs + A.zero_tail);
    const int tile = row_tiles - 1 - id / (A.seqs + A.zero_tail);
    if (b == A.seqs) {                                 // rows of no sequence, before the first and behind the last
        const int a = min(max(A.cu[0], 0), A.rows), z = min(max(A.cu[A.seqs], a), A.rows);
        const int none = a + A.rows - z;
        for (int r = tile * ROWS + (threadIdx.x >> 5); r < none; r += 8) {
            if (r >= tile * ROWS + ROWS && tile != row_tiles - 1) break;
            uint16_t* o = reinterpret_cast<uint16_t*>(A.out) + ((long)(r < a ? r : z + r - a) * A.hq + h) * A.d;
            for (int d = threadIdx.x & 31; d < A.d; d += 32) o[d] = 0;
        }
        return;
    }
    const int start = min(max(A.cu[b], 0), A.rows), end = min(max(A.cu[b + 1], start), A.rows);
    const int len = end - start;
    const int q0 = tile * ROWS;
    if (q0 >= len) return;
    const int D = A.d, chunks = D >> 3;
    const uint16_t* kp = reinterpret_cast<const uint16_t*>(A.k) + (long)start * A.k_row + hk * A.k_head;
    const uint16_t* vp = reinterpret_cast<const uint16_t*>(A.v) + (long)start * A.v_row + hk * A.v_head;

    // this wave's rows of q
    const int wq = q0 + 32 * wave, row = wq + n;
    u4 q[KS];
    {
        const uint16_t* qp = reinterpret_cast<const uint16_t*>(A.q) + (long)(start + min(row, len - 1)) * A.q_row +
                             h * A.q_head;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int c = 2 * s + hf;
            q[s] = c < chunks ? *reinterpret_cast<const u4*>(qp + 8 * c) : u4{0, 0, 0, 0};
        }
    }
    // Staging: each lane brings 16-byte chunks, its place in the tile fixed by the lane; rows behind the sequence and chunks
    // behind the head's values are out of the buffer's range and come as zeros.
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr)lds;
    // A lane's loads; where its chunks come from: the first's place, and the rows from one load to the next (turns are the
    // same in all of them, twelve-chunk rows have a place for each).
    constexpr int LOADS = KT * CP / (64 * WAVES), PLACES = CP == 12 ? LOADS : 1, STEP = CP == 12 ? 0 : 64 * WAVES / CP;
    const uint32_t k_bytes = (uint32_t)A.k_row * 2, v_bytes = (uint32_t)A.v_row * 2;
    uint32_t k_off[PLACES], v_off[PLACES];
#pragma unroll
    for (int i = 0; i < PLACES; ++i) {
        const int pos = (i * WAVES + wave) * 64 + lane, r = pos / CP, c = pos % CP;
        // the chunk that is kept at place `pos`: a turn undoes itself, the rotation goes back
        const int ck = CP == 12 ? (c + 12 - 2 * (r >> 2 & 1)) % 12 : k_place<CP>(r, c) - r * CP;
        const int cv = v_place<CP>(r, c) - r * CP;
        k_off[i] = ck < chunks ? r * k_bytes + 16 * ck : 0x7FFFFFF0u;
        v_off[i] = cv < chunks ? r * v_bytes + 16 * cv : 0x7FFFFFF0u;
    }
    auto stage = [&](int t, int buf) {
        const __amdgpu_buffer_rsrc_t kr = rows_from(kp, A.k_row, t, len, D), vr = rows_from(vp, A.v_row, t, len, D);
        const uint32_t to = lds0 + buf * 2 * TILE + wave * 1024;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            load_chunks(kr, to + i * WAVES * 1024, k_off[i % PLACES] + i * STEP * k_bytes);
            load_chunks(vr, to + TILE + i * WAVES * 1024, v_off[i % PLACES] + i * STEP * v_bytes);
        }
    };

    f16v acc[DT32];
#pragma unroll
    for (int i = 0; i < DT32; ++i) acc[i] = zero16();
    float M = LOW, l = 0.f;
    const float cc = A.scale * 1.44269504088896341f;
    // Exponents are s ca + at, in one FMA.  Where M is FAR from zero its product is not a float to within the exponents' range:
    // there the rounded product minus M takes s's place.
    float ca = cc, at = 0.f;
    bool far = false;                                             // some row of the wave is so

    // LDS addresses of this lane's operands: K row n (32 rows on: the same places) at step s; V^T of d tile i, two
    // transposed reads of four tokens a token step.  An exclusive or takes a turned row from step to step.
    const uint32_t k_lds = lds0 + 16 * k_place<CP>(n, hf);
    uint32_t k_step[CP == 12 ? KS : 1];
    if constexpr (CP == 12)
#pragma unroll
        for (int s = 0; s < KS; ++s) k_step[s] = lds0 + 16 * k_place<CP>(n, 2 * s + hf);
    const int tr_row = 4 * hf + ((lane & 15) >> 2), tr_chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const uint32_t v_lds = lds0 + TILE + 16 * v_place<CP>(tr_row, tr_chunk) + 8 * (lane & 1);
    auto k_operand = [&](uint32_t buf, int i, int s) {            // buf: the tile's buffer, in bytes
        uint32_t at;
        if constexpr (CP == 12) at = k_step[s] + buf;
        else at = (k_lds + buf) ^ (32 * s);
        return *reinterpret_cast<lds_u4>(at + i * 32 * CP * 16);
    };
    auto v_operand = [&](uint32_t buf, int i, int s) {
        const uint32_t at = CP == 12 ? v_lds + buf + 64 * i : (v_lds + buf) ^ (64 * i);
        union { s4 h[2]; u4 v; } o;
#pragma unroll
        for (int p = 0; p < 2; ++p)
            o.h[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s4>(at + (16 * s + 8 * p) * CP * 16));
        return o.v;
    };

    const int tiles = (min(q0 + ROWS, len) + KT - 1) / KT;       // the workgroup's last row sees up to itself
    const int whole = (wq + 1) / KT;                              // tiles that every row of this wave sees all of
    uint32_t odd = 0;                                             // tiles from `whole` on whose V is not all finite
    auto tile_step = [&](int t, auto edge_tag) {
        const uint32_t BUF = (t & 1) * 2 * TILE;
        constexpr bool EDGE = decltype(edge_tag)::value;          // some row does not see all of the tile
        if constexpr (EDGE) {
            // V times zeros: NaN where some value is an infinity or NaN
            f16v test = zero16();
#pragma unroll
            for (int i = 0; i < DT32; ++i)
#pragma unroll
                for (int st = 0; st < 4; ++st) test = mfma<DT>(v_operand(BUF, i, st), u4{0, 0, 0, 0}, test);
            float any = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) any += test[j];
            if (__builtin_amdgcn_ballot_w64(any != any) != 0) {
                odd |= 1u << (t - whole);
                return;
            }
        }
        // Two halves of 32 tokens: the second half's scores may run beside the first's weights, the first's sums beside the
        // second's weights, and half a tile of scores is live at a time.
        u4 w[4];                                                  // weights, 16 tokens a step
        auto scores = [&](int i) {
            f16v s = zero16();
#pragma unroll
            for (int st = 0; st < KS; ++st) s = mfma<DT>(k_operand(BUF, i, st), q[st], s);
            return s;
        };
        // masks what is not seen and moves M where a score is past it; `done`: steps of w that are scaled by it already
        auto reference = [&](f16v& s, int i, int done) {
            if constexpr (EDGE) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int tok = t * KT + 32 * i + 8 * (j >> 2) + 4 * hf + (j & 3);
                    s[j] = tok <= row ? s[j] : -__builtin_inff();
                }
            }
            float top = s[0];
#pragma unroll
            for (int j = 1; j < 16; ++j) top = fmaxf(top, s[j]);
            const uint32_t u = __float_as_uint(top);
            const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
            top = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])) * cc;
            if (far || __builtin_amdgcn_ballot_w64(top > M + SLACK) != 0) {
                const float to = top > M + SLACK ? __builtin_ceilf(top) : M;       // whole: what it scales stays exact
                const float f = __builtin_amdgcn_exp2f(M - to);
                M = to;
                l *= f;
#pragma unroll
                for (int d = 0; d < DT32; ++d)
#pragma unroll
                    for (int j = 0; j < 16; ++j) acc[d][j] *= f;
#pragma unroll
                for (int k = 0; k < done; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        w[k][e] = pack2<DT>(half_of<DT>(w[k][e]) * f, half_of<DT>(w[k][e] >> 16) * f);
                const bool apart = !(__builtin_fabsf(M) < FAR);
                ca = apart ? 1.f : cc;
                at = apart ? UP<DT> : UP<DT> - M;
                far = __builtin_amdgcn_ballot_w64(apart) != 0;
                if (far) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) s[j] = apart ? less_rounded(s[j], cc, M) : s[j];
                }
            }
        };
        auto weights = [&](const f16v& s, int i) {
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j], ca, at));
                const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j + 1], ca, at));
                const uint32_t both = pack2<DT>(x, y);
                w[2 * i + (j >> 3)][(j & 7) >> 1] = both;
                l = plus_both<DT>(both, l);
            }
        };
        auto sums = [&](int i) {
#pragma unroll
            for (int st = 2 * i; st < 2 * i + 2; ++st)
#pragma unroll
                for (int d = 0; d < DT32; ++d) acc[d] = mfma<DT>(v_operand(BUF, d, st), w[st], acc[d]);
        };
        f16v s0 = scores(0);
        reference(s0, 0, 0);
        f16v s1 = scores(1);
        weights(s0, 0);
        reference(s1, 1, 2);
        sums(0);
        weights(s1, 1);
        sums(1);
    };

    // All tiles, then, where some wave left tiles out, the diagonal ones again with V's infinities and NaN as zeros.
    // Every turn has one barrier, so that waves may be in different loops.
    bool again = false;
    auto turn = [&](int t) {
        landed_barrier();                                         // tile t has landed; tile t - 1 has been read
        if (t + 1 < tiles) stage(t + 1, (t + 1) & 1);
    };
    for (int t0 = 0;;) {
        stage(t0, t0 & 1);
        int t = t0;
        for (; !again && t < min(whole, tiles); ++t) {
            turn(t);
            tile_step(t, std::integral_constant<bool, false>{});
        }
        for (; t < tiles; ++t) {
            if (again) {
                landed_barrier();
                for (int x = threadIdx.x; x < KT * CP; x += 64 * WAVES) {
                    u4* at = reinterpret_cast<u4*>(lds + (2 * (t & 1) + 1) * TILE) + x;
                    u4 v = *at;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] &= ~not_finite(v[e]);
                    *at = v;
                }
            }
            turn(t);
            if (t >= whole && (again ? odd >> (t - whole) & 1 : t * KT <= wq + 31))
                tile_step(t, std::integral_constant<bool, true>{});
        }
        if (again) break;
        __syncthreads();                                          // the tiles have been read: the waves' marks go there
        uint32_t* marks = reinterpret_cast<uint32_t*>(lds);
        if (lane == 0) marks[wave] = odd;
        __syncthreads();
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) any |= marks[i];
        if (!any) break;
        __syncthreads();
        again = true;
        t0 = (q0 + 1) / KT;
    }

    l += __shfl_xor(l, 32);
    if (row >= len) return;
    const float inv = 1.f / l;
    uint16_t* o = reinterpret_cast<uint16_t*>(A.out) + ((long)(start + row) * A.hq + h) * D;
#pragma unroll
    for (int i = 0; i < DT32; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = 32 * i + 8 * j + 4 * hf;
            if (d < D) {
                uint2 v;
                v.x = pack2<DT>(acc[i][4 * j] * inv, acc[i][4 * j + 1] * inv);
                v.y = pack2<DT>(acc[i][4 * j + 2] * inv, acc[i][4 * j + 3] * inv);
                *reinterpret_cast<uint2*>(o + d) = v;
            }
        }
    if (odd) {                                                    // what the row sees of them
#pragma unroll 1
        for (int tok = whole * KT; tok <= row; ++tok)
#pragma unroll 1
            for (int d = 4 * hf; d < D; d += (d & 3) == 3 ? 5 : 1) {
                const uint16_t x = vp[(long)tok * A.v_row + d];
                if (not_finite(x) != 0) store_f<DT>(o, d, load_f<DT>(o, d) + load_f<DT>(&x, 0));
            }
    }
}

struct Built {
    const void* f;
    int cp;
};

template <int DT>
Built kernel_for(int d) {
    switch ((d + 15) / 16) {
        case 1: case 2: return {(const void*)prompt_attn_kernel<DT, 2, 4>, 4};
        case 3: return {(const void*)prompt_attn_kernel<DT, 3, 8>, 8};
        case 4: return {(const void*)prompt_attn_kernel<DT, 4, 8>, 8};
        case 5: return {(const void*)prompt_attn_kernel<DT, 5, 12>, 12};
        case 6: return {(const void*)prompt_attn_kernel<DT, 6, 12>, 12};
        case 7: return {(const void*)prompt_attn_kernel<DT, 7, 16>, 16};
        case 8: return {(const void*)prompt_attn_kernel<DT, 8, 16>, 16};
        case 9: case 10: case 11: case 12: return {(const void*)prompt_attn_kernel<DT, 12, 32>, 32};
        default: return {(const void*)prompt_attn_kernel<DT, 16, 32>, 32};
    }
}

}  // namespace

hipError_t launch_prompt_attn(const PromptArgs& A, int dt, hipStream_t stream) {
    const Built k = dt == DT_F16 ? kernel_for<DT_F16>(A.d) : kernel_for<DT_BF16>(A.d);
    PromptArgs a = A;
    int row_tiles = (A.longest + ROWS - 1) / ROWS;
    const int lds = 4 * KT * k.cp * 16;
    if (hipError_t e = lds_limit_raise(k.f, lds); e != hipSuccess) return e;
    void* args[] = {&a, &row_tiles};
    const long grid = (long)row_tiles * (A.seqs + A.zero_tail) * A.hq;
    return launch(k.f, dim3((unsigned)grid), dim3(64 * WAVES), args, lds, stream);
}

}  // namespace cbk
