// prompt_attn_f32.hip -- causal attention over packed prompts, fp32, on the fp32 matrix cores.
//
// prompt_attn.hip's arithmetic with nothing rounded below fp32: S^T = K q^T and O^T += V^T w on
// v_mfma_f32_32x32x2_f32, whose S^T layout (column = row, tokens 8 i + 4 (lane / 32) + 0..3) again gives the
// operand of w without moving it: step i of the second product takes the two tokens that lanes l and l + 32
// hold in register i.  A workgroup has 64 rows of one head (32 a wave); tiles of 32 tokens pass through LDS.  Bound: the fp32
// matrix instructions, a sixteenth of the 16-bit rate, and the tile's staging, which nothing hides.
#include "kv4.hpp"
#include "cbk_kernels.hpp"

namespace cbk {
namespace {

typedef float f16v __attribute__((ext_vector_type(16)));

constexpr int WAVES = 2;
constexpr int ROWS = 32 * WAVES;
constexpr int KT = 32;
constexpr float LOW = -1e30f;

// DP: the head's values rounded up to 32 (64 above 128).
template <int DP>
__global__ __launch_bounds__(64 * WAVES, 1) void prompt_attn_f32_kernel(PromptArgs A, int row_tiles) {
    constexpr int DT32 = DP / 32;
    constexpr int PITCH = DP + 1;                      // odd: a wave reads 32 rows' values of one column
    extern __shared__ __align__(16) float lds_f[];     // K tile [KT][PITCH], V tile [KT][DP]
    float* kt = lds_f;
    float* vt = lds_f + KT * PITCH;
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

    float q[DP / 2];                                   // values 2 s + hf
    {
        const float* qp = reinterpret_cast<const float*>(A.q) + (long)(start + min(row, len - 1)) * A.q_row + h * A.q_head;
#pragma unroll
        for (int s = 0; s < DP / 2; ++s) q[s] = 2 * s + hf < D ? qp[2 * s + hf] : 0.f;
    }
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

    const int last = min(q0 + ROWS, len);
    for (int t0 = 0; t0 < last; t0 += KT) {
        __syncthreads();
        for (int x = threadIdx.x; x < KT * DP; x += 64 * WAVES) {
            const int r = x / DP, d = x % DP;
            const long tok = min(t0 + r, len - 1);
            kt[r * PITCH + d] = d < D ? kp[tok * A.k_row + d] : 0.f;
            vt[x] = d < D ? vp[tok * A.v_row + d] : 0.f;
        }
        __syncthreads();
        if (t0 > wq + 31) continue;
        f16v s;
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = 0.f;
#pragma unroll
        for (int st = 0; st < DP / 2; ++st)
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(kt[n * PITCH + 2 * st + hf], q[st], s, 0, 0, 0);
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
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float at = s[j] > -__builtin_inff() ? __builtin_fmaf(s[j], cl, -M) : -M;
            s[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j], cc, at));
            l += s[j];
        }
        // masked places take no part whatever they hold: on the diagonal, infinities and NaN go in as zeros and
        // what a row sees of them is added at the end
#pragma unroll
        for (int i = 0; i < DT32; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                float v = vt[(8 * (j >> 2) + 4 * hf + (j & 3)) * DP + 32 * i + n];
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
    lds = (KT * (DP + 1) + KT * DP) * 4;
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
