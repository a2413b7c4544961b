// prompt_attn_f32.hip -- causal attention over packed prompts, fp32, on the fp32 matrix cores.
//
// prompt_attn.hip's arithmetic with nothing rounded below fp32: S^T = K q^T and O^T += V^T w on
// v_mfma_f32_32x32x2_f32, whose S^T layout (column = row, tokens 8 i + 4 (lane / 32) + 0..3) again gives the
// operand of w without moving it: step i of the second product takes the two tokens that lanes l and l + 32
// hold in register i.  A workgroup has 128 rows of one head (32 a wave); tiles of 32 tokens are staged in LDS as in
// prompt_attn.hip, the next one's loads under way.  The order of a product's steps is free: lanes l and l + 32 take four
// neighbouring values each, so that K comes in 16-byte reads.
// Bound: the fp32 matrix instructions, a sixteenth of the 16-bit rate, each waiting for the one before: a tile is one chain
// of D / 2 products and D / 32 of sixteen, and one or two waves share a SIMD.  Measured: 1024 rows, 32 heads of 128, 255 us
// (34 TFLOP/s; with loads through registers and two waves a workgroup 561); 4 x 100..700 rows, 16 / 4 heads of 80, 131 us
// (216).  The scores in two sums instead of one: 260 and 129.  1500 rows, 8 heads of 256: 750 us (2143), 96 workgroups on
// 256 CUs, the last with 47 tiles in a row.
#include "kv4.hpp"
#include "cbk_kernels.hpp"

namespace cbk {
namespace {

typedef float f16v __attribute__((ext_vector_type(16)));

constexpr int WAVES = 4;
constexpr int ROWS = 32 * WAVES;
constexpr int KT = 32;
constexpr float LOW = -0x1.fffffep127f;        // reference of a row that has seen nothing

typedef float f4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef const __attribute__((address_space(3))) f4* lds_f4;
typedef const __attribute__((address_space(3))) float* lds_f1;

// The chunk of K's row r that lies at chunk c (and the other way round): a wave reads two neighbouring chunks of 32 rows.
template <int CP>
__device__ __forceinline__ int k_turn(int r, int c) { return c ^ (CP % 16 == 0 ? (r & 7) << 1 : (r >> 1 & 3) << 1); }

// A buffer over a sequence's rows (len of them, `stride` elements apart, D values each) from tile t on.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_from(const float* base, long stride, int t, int len, int D) {
    const long left = len - t * KT;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base + (long)t * KT * stride), 0,
                                             (int)min(((left - 1) * stride + D) * 4, 0x7FFFFF00l), 0x00020000);
}

__device__ __forceinline__ void load_chunks(__amdgpu_buffer_rsrc_t from, uint32_t to, uint32_t offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_ptr)to, 16, offset, 0, 0, 0);
}

// DP: the head's values rounded up to 32 (64 above 128).
template <int DP>
__global__ __launch_bounds__(64 * WAVES, 1) void prompt_attn_f32_kernel(PromptArgs A, int row_tiles) {
    constexpr int DT32 = DP / 32, CP = DP / 4;         // d tiles, 16-byte chunks of a row
    constexpr int TILE = KT * CP * 16;                 // bytes of a K or V tile
    extern __shared__ __align__(16) char lds[];        // [2][K tile, V tile]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, hf = lane >> 5;
    int id = blockIdx.x;
    const int hk = id % A.hkv;
    id /= A.hkv;
    const int h = hk * A.group + id % A.group;
    id /= A.group;
    const int b = id % (A.seqs + A.zero_tail);
    const int tile = row_tiles - 1 - id / (A.seqs + A.zero_tail);
    const int D = A.d;
    float* out = reinterpret_cast<float*>(A.out);
    if (b == A.seqs) {                                 // rows of no sequence, before the first and behind the last
        const int a = min(max(A.cu[0], 0), A.rows), z = min(max(A.cu[A.seqs], a), A.rows);
        const int none = a + A.rows - z;
        for (int r = tile * ROWS + wave; r < none; r += WAVES) {
            if (r >= tile * ROWS + ROWS && tile != row_tiles - 1) break;
            float* o = out + ((long)(r < a ? r : z + r - a) * A.hq + h) * D;
            for (int d = lane; d < D; d += 64) o[d] = 0.f;
        }
        return;
    }
    const int start = min(max(A.cu[b], 0), A.rows), end = min(max(A.cu[b + 1], start), A.rows);
    const int len = end - start;
    const int q0 = tile * ROWS;
    if (q0 >= len) return;
    const float* kp = reinterpret_cast<const float*>(A.k) + (long)start * A.k_row + hk * A.k_head;
    const float* vp = reinterpret_cast<const float*>(A.v) + (long)start * A.v_row + hk * A.v_head;
    const int wq = q0 + 32 * wave, row = wq + n;

    f4 q[DP / 8];                                      // values 8 u + 4 hf ..
    {
        const float* qp = reinterpret_cast<const float*>(A.q) + (long)(start + min(row, len - 1)) * A.q_row + h * A.q_head;
#pragma unroll
        for (int u = 0; u < DP / 8; ++u) {
            const int d = 8 * u + 4 * hf;
            q[u] = d < D ? *reinterpret_cast<const f4*>(qp + d) : f4{0.f, 0.f, 0.f, 0.f};
        }
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr)lds;
    constexpr int LOADS = KT * CP / (64 * WAVES);      // a lane's loads of a tile, and where its chunks come from
    uint32_t k_off[LOADS], v_off[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int pos = (i * WAVES + wave) * 64 + lane, r = pos / CP, c = pos % CP, ck = k_turn<CP>(r, c);
        k_off[i] = 4 * ck < D ? r * (uint32_t)A.k_row * 4 + 16 * ck : 0x7FFFFFF0u;
        v_off[i] = 4 * c < D ? r * (uint32_t)A.v_row * 4 + 16 * c : 0x7FFFFFF0u;
    }
    auto stage = [&](int t) {
        const __amdgpu_buffer_rsrc_t kr = rows_from(kp, A.k_row, t, len, D), vr = rows_from(vp, A.v_row, t, len, D);
        const uint32_t to = lds0 + (t & 1) * 2 * TILE + wave * 1024;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            load_chunks(kr, to + i * WAVES * 1024, k_off[i]);
            load_chunks(vr, to + TILE + i * WAVES * 1024, v_off[i]);
        }
    };
    f16v acc[DT32];
#pragma unroll
    for (int i = 0; i < DT32; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i][j] = 0.f;
    float M = LOW, l = 0.f;
    // scale log2 e in two terms: its rounding would bend every score by 2^-24 of itself
    const double c2 = (double)A.scale * 1.44269504088896340736;
    const float cc = (float)c2, cl = (float)(c2 - (double)cc);
    bool odd_values = false;

    const int tiles = (min(q0 + ROWS, len) + KT - 1) / KT;
    stage(0);
    for (int t = 0; t < tiles; ++t) {
        landed_barrier();                              // tile t has landed; tile t - 1 has been read
        if (t + 1 < tiles) stage(t + 1);
        const int t0 = t * KT;
        if (t0 > wq + 31) continue;
        const uint32_t kt = lds0 + (t & 1) * 2 * TILE, vt = kt + TILE;
        f16v s;
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = 0.f;
#pragma unroll
        for (int u = 0; u < DP / 8; ++u) {
            const f4 k = *reinterpret_cast<lds_f4>(kt + 16 * (n * CP + k_turn<CP>(n, 2 * u + hf)));
#pragma unroll
            for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e], q[u][e], s, 0, 0, 0);
        }
        const bool edge = t0 + KT - 1 > wq;
        float top = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            if (edge && t0 + 8 * (j >> 2) + 4 * hf + (j & 3) > row) s[j] = -__builtin_inff();
            top = fmaxf(top, s[j]);
        }
        top = fmaxf(top, __shfl_xor(top, 32)) * cc;
        if (top > M) {
            top = __builtin_ceilf(top);                 // whole: scores minus M and what M scales stay exact
            const float f = __builtin_amdgcn_exp2f(M - top);
            M = top;
            l *= f;
#pragma unroll
            for (int i = 0; i < DT32; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[i][j] *= f;
        }
        float ca = cc, cb = cl, m = -M;
        const bool apart = !(__builtin_fabsf(M) < FAR);
        if (__builtin_amdgcn_ballot_w64(apart) != 0) {  // as in prompt_attn.hip: the rounded product minus M for s
            ca = apart ? 1.f : cc, cb = apart ? 0.f : cl, m = apart ? 0.f : m;
#pragma unroll
            for (int j = 0; j < 16; ++j) s[j] = apart ? less_rounded(s[j], cc, M) : s[j];
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float at = s[j] > -__builtin_inff() ? __builtin_fmaf(s[j], cb, m) : m;
            s[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j], ca, at));
            l += s[j];
        }
        // masked places take no part whatever they hold: on the diagonal, infinities and NaN go in as zeros and
        // what a row sees of them is added at the end
#pragma unroll
        for (int i = 0; i < DT32; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                float v = *reinterpret_cast<lds_f1>(vt + ((8 * (j >> 2) + 4 * hf + (j & 3)) * DP + 32 * i + n) * 4);
                if (edge && !(__builtin_fabsf(v) < __builtin_inff())) v = 0.f, odd_values = true;
                acc[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, s[j], acc[i], 0, 0, 0);
            }
    }
    const bool any_odd = __builtin_amdgcn_ballot_w64(odd_values) != 0;
    l += __shfl_xor(l, 32);
    if (row >= len) return;
    const float inv = 1.f / l;
    float* o = out + ((long)(start + row) * A.hq + h) * D;
#pragma unroll
    for (int i = 0; i < DT32; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int d = 32 * i + 8 * (j >> 2) + 4 * hf + (j & 3);
            if (d < D) o[d] = acc[i][j] * inv;
        }
    if (any_odd) {                                     // what the row sees of them
#pragma unroll 1
        for (int tok = (wq + 1) / KT * KT; tok <= row; ++tok)
#pragma unroll 1
            for (int d = 4 * hf; d < D; d += (d & 3) == 3 ? 5 : 1) {
                const float x = vp[(long)tok * A.v_row + d];
                if (!(__builtin_fabsf(x) < __builtin_inff())) o[d] += x;
            }
    }
}

template <int DP>
const void* built(int& lds) {
    lds = 4 * KT * DP * 4;
    return (const void*)prompt_attn_f32_kernel<DP>;
}

}  // namespace

hipError_t launch_prompt_attn_f32(const PromptArgs& A, hipStream_t stream) {
    int lds = 0;
    const void* f = A.d <= 32 ? built<32>(lds) : A.d <= 64 ? built<64>(lds) : A.d <= 96 ? built<96>(lds)
                  : A.d <= 128 ? built<128>(lds) : A.d <= 192 ? built<192>(lds) : built<256>(lds);
    PromptArgs a = A;
    int row_tiles = (A.longest + ROWS - 1) / ROWS;
    if (hipError_t e = lds_limit_raise(f, lds); e != hipSuccess) return e;
    void* args[] = {&a, &row_tiles};
    const long grid = (long)row_tiles * (A.seqs + A.zero_tail) * A.hq;
    return launch(f, dim3((unsigned)grid), dim3(64 * WAVES), args, lds, stream);
}

}  // namespace cbk
