// kv4_store.hip -- new tokens' keys and values into the paged 4-bit cache, and back out of it.
//
// Quantizing a vector x of a token and head (kv4.hpp's format): over lo = min(0, min x) and
// hi = max(0, max x), r = hi - lo and z = rint(-15 lo / r) in 64 bits, the word
// (bits(max(float(r / 15), 2^-100)) & ~15) | z, whose float is s, and c = clamp(rint(x / s) + z, 0, 15)
// with x / s at its exact value (halves to even).  The codes follow the definition exactly, at borders too:
// a rounded quotient would move a whole step.  x * (1 / s) is off by less than 2e-6, so its rint is right
// unless it lies within 4e-6 of a half; where some lane's does (one wave pass in a few hundred) e = x - q s decides,
// exact in one FMA there (a multiple of half x's last place below 2^24 of them).  z is found the same way.
//
// A wave has one block of 32 tokens of one head.  K: 16 lanes (32 above 128 values) hold a token, eight
// values each, and write one word each; the next four tokens' loads are under way meanwhile.  V's words hold eight
// tokens of one value: the codes pass through LDS as bytes [value][token], and a word is two dwords of them folded
// together.  A block that is not all new keeps the other tokens' codes (read ahead of the rest).
// Bound: the vector instructions of quantizing (6545 tokens of 32 heads of 128 in fp16, 136 MB with the codes: 48 us, 2.8 TB/s, 38 us of
// vector issue), for a decode step's tokens the latencies of table, values and old words (64 tokens of 8 heads: 8 us).
// The read moves as many bytes in 41 us.
#include "kv4.hpp"
#include "cbk_kernels.hpp"

namespace cbk {
namespace {

constexpr int WAVES = 4;

// Which sequence virtual block `u` belongs to, and which of its touched blocks it is.  Sequence b has
// the virtual blocks [cu[b] / 32 + 2 b, cu[b + 1] / 32 + 2 (b + 1)): at least as many as its new tokens
// touch.  Lanes look at 64 sequences at once.  b = seqs: u lies before the first sequence or behind the
// last, `n` rows from row0 on.
struct Where {
    int b, i;          // sequence, virtual block within it
    int row0, n;       // first new row, new rows
    int pos0;          // the first one's position in the sequence
};

__device__ __forceinline__ Where where_of(const Kv4View& C, const Kv4Rows& R, int u, int lane) {
    Where w;
    if (!R.cu) {       // one row a sequence: one virtual block each
        w.b = u, w.i = 0, w.row0 = u, w.n = 1;
    } else {
        int below = 0;
        for (int b0 = 0; b0 < C.seqs; b0 += 64) {
            const int b = b0 + lane;
            const bool in = b < C.seqs && (min(max(R.cu[b], 0), R.rows) >> 5) + 2 * b <= u;
            const uint64_t m = __builtin_amdgcn_ballot_w64(in);
            below += __builtin_popcountll(m);
            if (m != ~0ull) break;
        }
        const int b = __builtin_amdgcn_readfirstlane(below - 1);
        if (b < 0) {                                   // before the first sequence
            w.b = C.seqs, w.i = u, w.row0 = 0, w.n = min(max(R.cu[0], 0), R.rows), w.pos0 = 0;
            return w;
        }
        const int a = min(max(R.cu[b], 0), R.rows), z = min(max(R.cu[b + 1], a), R.rows);
        w.b = b, w.i = u - (a >> 5) - 2 * b, w.row0 = a, w.n = z - a;
        if (b == C.seqs - 1 && w.i >= (z >> 5) - (a >> 5) + 2) {       // behind the last sequence
            w.i -= (z >> 5) - (a >> 5) + 2;
            w.b = C.seqs, w.row0 = z, w.n = R.rows - z, w.pos0 = 0;
            return w;
        }
    }
    w.pos0 = w.b < C.seqs ? C.lens[w.b] - w.n : 0;
    return w;
}

// The smaller, and the larger, of a value over the W lanes of a token.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xF, 0xF, true));
}
template <int W, bool MAX>
__device__ __forceinline__ float row_best(float v) {
    auto best = [](float a, float b) { return MAX ? fmaxf(a, b) : fminf(a, b); };
    v = best(v, dpp<0xB1>(v));          // lanes 1 apart, 2 apart, the other four of eight, the other eight
    v = best(v, dpp<0x4E>(v));
    v = best(v, dpp<0x141>(v));
    v = best(v, dpp<0x140>(v));
    if constexpr (W == 32) {
        const uint32_t u = __float_as_uint(v);
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        v = best(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    return v;
}

constexpr float NEAR_HALF = 0.5f - 4e-6f;

// Eight values of a vector spread over W lanes -> their codes and the vector's word.
template <int W>
__device__ __forceinline__ uint32_t quantize8(const float (&x)[8], int lane, int (&c)[8]) {
    float lo = 0.f, hi = 0.f;
    bool fine = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        lo = fminf(lo, x[j]);
        hi = fmaxf(hi, x[j]);
        fine &= __builtin_fabsf(x[j]) < __builtin_inff();
    }
    lo = row_best<W, false>(lo);
    hi = row_best<W, true>(hi);
    const uint64_t odd = __builtin_amdgcn_ballot_w64(!fine);
    const double r = (double)hi - (double)lo;
    // z = rint(-15 lo / r), near 0 .. 15, in fp32 of the halves (no overflow): off by three roundings, 15 x 3 x 2^-24 < 3e-6,
    // where r is not so small that halves lose bits; r / 15 by its reciprocal and one correction, which rounds as the division
    const float rh = 0.5f * hi - 0.5f * lo;
    const float zt = -15.f * (0.5f * lo / rh);
    float zr = r > 0.0 ? __builtin_rintf(zt) : 0.f;
    if (__builtin_amdgcn_ballot_w64(r > 0.0 && !(__builtin_fabsf(zt - zr) < NEAR_HALF && rh >= 0x1p-100f)) != 0)
        zr = r > 0.0 ? (float)__builtin_rint(-15.0 * (double)lo / r) : 0.f;
    const double fifteenth = 1.0 / 15.0, q0 = r * fifteenth;
    const double fifth = __builtin_fma(__builtin_fma(-15.0, q0, r), fifteenth, q0);
    const float step = fmaxf((float)fifth, KV4_MIN_SCALE);
    const int z = (int)zr;
    uint32_t word = (__float_as_uint(step) & ~15u) | (uint32_t)z;
    const float s = __uint_as_float(word), inv = 1.0f / s;
    float q[8], far = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float t = x[j] * inv;
        q[j] = __builtin_rintf(t);
        far = fmaxf(far, __builtin_fabsf(t - q[j]));
    }
    if (__builtin_amdgcn_ballot_w64(!(far < NEAR_HALF)) != 0) {
        const float half = 0.5f * s;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float e = __builtin_fmaf(-q[j], s, x[j]);
            const bool uneven = ((int)q[j] & 1) != 0;
            const bool up = e > half || (e == half && uneven), down = e < -half || (e == -half && uneven);
            q[j] += up ? 1.f : down ? -1.f : 0.f;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = (int)fminf(fmaxf(q[j] + zr, 0.f), 15.f);
    if (odd) {
        const uint64_t own = (W == 32 ? 0xFFFFFFFFull : 0xFFFFull) << (lane & ~(W - 1));
        if (odd & own) {
            word = 0x7FC00000u;
#pragma unroll
            for (int j = 0; j < 8; ++j) c[j] = 0;
        }
    }
    return word;
}

template <int DT>
__device__ __forceinline__ void load8(const void* p, long i, float (&x)[8]) {
    if constexpr (DT == DT_F32) {
        const float4* s = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
        const float4 a = s[0], b = s[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        using S = typename Dt<DT>::S;
        struct alignas(16) V { S v[8]; };
        const V v = *reinterpret_cast<const V*>(reinterpret_cast<const S*>(p) + i);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = Dt<DT>::to_f(v.v[j]);
    }
}

template <int DT>
__device__ __forceinline__ void store8(void* p, long i, const float (&x)[8]) {
    using S = typename Dt<DT>::S;
    struct alignas(16) V { S v[8]; };
    V v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v.v[j] = Dt<DT>::from_f(x[j]);
    *reinterpret_cast<V*>(reinterpret_cast<S*>(p) + i) = v;
}

// s (c - z) as an fp32 product: it is rounded to the output's type after (the empty asm keeps the compiler from
// rounding once, to fp16, with a mixed-precision multiply).
__device__ __forceinline__ float value_of(uint32_t word, uint32_t code) {
    float p = __uint_as_float(word) * (float)((int)code - (int)(word & 15u));
    asm("" : "+v"(p));
    return p;
}

// W lanes a token: 16 for up to 128 values, 32 beyond.
template <int DT, int W>
__global__ __launch_bounds__(64 * WAVES) void kv4_append_kernel(Kv4StoreArgs A, int units) {
    constexpr int TOK = 64 / W;                        // tokens of a pass
    constexpr int PITCH = KV4_BLOCK + 4;               // bytes of a value's tokens in LDS
    __shared__ __align__(16) uint8_t codes[WAVES][8 * W * PITCH];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = blockIdx.y * WAVES + wave;
    const int u = blockIdx.x;
    const Kv4View& C = A.c;
    if (h >= C.heads || u >= units) return;
    const Where w = where_of(C, A.r, u, lane);
    if (w.b >= C.seqs || w.n <= 0) return;
    const int first = max(w.pos0, 0);                  // a sequence shorter than its new rows: the rest is left out
    const int blk = (first >> 5) + w.i;
    const int lo = max(first, 32 * blk), hi = min(w.pos0 + w.n, 32 * blk + 32);
    if (lo >= hi) return;
    uint32_t* base = kv4_block(C, w.b, blk, h);
    if (!base) return;
    const int ns = C.ns, sub = lane / W, i8 = lane % W;      // token of the pass, word of the token
    const bool mine = 8 * i8 < C.d;
    const int psh = ns & 1 ? 1 : 2;                    // log2 of the words of a piece
    uint32_t* meta = base + 256 * ns;
    uint32_t* vc = base + 128 * ns;
    uint8_t* lds = codes[wave];
    const bool part = hi - lo < 32;
    uint32_t old[KV4_MAX_D / 16 * W / 32];             // V's words of a block that keeps some (2 ns of them a lane)
    if (part) {
#pragma unroll
        for (int i = 0; i < KV4_MAX_D / 16 * W / 32; ++i)
            if (i < 2 * ns) old[i] = vc[lane + 64 * i];
    }
    // values of the pass at t0 (the nearest rows that are new where the lane's own is not)
    const long k0 = h * A.k_head + (mine ? 8 * i8 : 0), v0 = h * A.v_head + (mine ? 8 * i8 : 0);
    auto fetch = [&](int t0, float (&xk)[8], float (&xv)[8]) {
        const long row = w.row0 + (min(max(t0 + sub, lo), hi - 1) - w.pos0);
        load8<DT>(A.k, row * A.k_row + k0, xk);
        load8<DT>(A.v, row * A.v_row + v0, xv);
    };
    const int from = 32 * blk + (lo - 32 * blk) / TOK * TOK;
    float xk[8], xv[8], nk[8], nv[8];
    fetch(from, xk, xv);
    for (int t0 = from; t0 < hi; t0 += TOK) {
        fetch(t0 + TOK, nk, nv);
        const int pos = t0 + sub, tok = pos - 32 * blk;
        const bool is_new = pos >= lo && pos < hi;
        int c[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) xk[j] = mine ? xk[j] : 0.f, xv[j] = mine ? xv[j] : 0.f;
        const uint32_t kw = quantize8<W>(xk, lane, c);
        if (is_new) {
            if (i8 < 4 * ns) {
                uint32_t word = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) word |= mine ? kv4_put((uint32_t)c[j], j) : 0u;
                base[tok * 4 * ns + i8] = word;
            }
            if (i8 == 0) meta[tok] = kw;
        }
        const uint32_t vw = quantize8<W>(xv, lane, c);
        if (is_new && i8 == 0) meta[32 + tok] = vw;
        if (is_new && i8 < 4 * ns) {
#pragma unroll
            for (int j = 0; j < 8; ++j) lds[(8 * i8 + j) * PITCH + tok] = (uint8_t)(mine ? c[j] : 0);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) xk[j] = nk[j], xv[j] = nv[j];
    }
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_s_waitcnt(0xF | (0x3 << 14) | (0x7 << 4));    // lgkmcnt(0): the wave's own bytes
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < KV4_MAX_D / 16 * W / 32; ++i) {
        if (i >= 2 * ns) break;
        const int x = lane + 64 * i;
        const int e = x & ((1 << psh) - 1), y = x >> psh;
        const int m = y & 15, g = (y >> 4) & 3, piece = y >> 6;
        const int d = 16 * ((piece << psh) + e) + m;
        // tokens 4 g + 0..3 and 16 + 4 g + 0..3 of value d, a byte each: fold them to nibbles (0, 2, 1, 3), and the
        // two to the word's (0, 2, 4, 6, 1, 3, 5, 7), turned by two bits
        auto fold = [](uint32_t a, uint32_t b) {
            a &= 0x0F0F0F0Fu, b &= 0x0F0F0F0Fu;        // bytes of tokens that are not new hold anything
            a |= a >> 12, b |= b >> 12;
            const uint32_t v = __builtin_amdgcn_perm(b, a, 0x05010400u);
            return __builtin_amdgcn_alignbit(v, v, 30);
        };
        const uint32_t* at = reinterpret_cast<const uint32_t*>(lds + d * PITCH + 4 * g);
        uint32_t word = fold(at[0], at[4]);
        if (part) {
            uint32_t na = 0, nb = 0;                   // which of the tokens are new
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int pa = 32 * blk + 4 * g + j, pb = pa + 16;
                na |= pa >= lo && pa < hi ? 15u << (8 * j) : 0u;
                nb |= pb >= lo && pb < hi ? 15u << (8 * j) : 0u;
            }
            const uint32_t fresh = fold(na, nb);
            if (fresh == 0) continue;
            word = (word & fresh) | (old[i] & ~fresh);
        }
        vc[x] = word;
    }
}

template <int DT, int W>
__global__ __launch_bounds__(64 * WAVES) void kv4_read_kernel(Kv4StoreArgs A, int units) {
    constexpr int TOK = 64 / W;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = blockIdx.y * WAVES + wave;
    const int u = blockIdx.x;
    const Kv4View& C = A.c;
    if (h >= C.heads || u >= units) return;
    const Where w = where_of(C, A.r, u, lane);
    const int ns = C.ns, sub = lane / W, i8 = lane % W;
    const bool mine = 8 * i8 < C.d;
    const float zeros[8] = {};
    if (w.b >= C.seqs) {                               // rows of no sequence
        for (int r = 32 * w.i + sub; r < min(32 * w.i + 32, w.n); r += TOK)
            if (mine) {
                const long at = ((long)(w.row0 + r) * C.heads + h) * C.d + 8 * i8;
                store8<DT>(A.k_out, at, zeros);
                store8<DT>(A.v_out, at, zeros);
            }
        return;
    }
    if (w.b == 0 && w.i == 0 && A.r.cu)                // rows before the first sequence, this side of its block
        for (int r = (w.row0 & ~31) + sub; r < w.row0; r += TOK)
            if (mine) {
                const long at = ((long)r * C.heads + h) * C.d + 8 * i8;
                store8<DT>(A.k_out, at, zeros);
                store8<DT>(A.v_out, at, zeros);
            }
    if (w.n <= 0) return;
    // blocks counted from the first new token's, which may lie before position 0 (floor)
    const int blk = (w.pos0 >> 5) + w.i;
    const int lo = max(w.pos0, 32 * blk), hi = min(w.pos0 + w.n, 32 * blk + 32);
    if (lo >= hi) return;
    const uint32_t* base = kv4_block(C, w.b, blk, h);
    const int psh = ns & 1 ? 1 : 2, pw = 1 << psh;
#pragma unroll 4
    for (int t0 = 32 * blk; t0 < 32 * blk + 32; t0 += TOK) {
        const int pos = t0 + sub, tok = pos - 32 * blk;
        if (pos < lo || pos >= hi || !mine) continue;
        const long at = ((long)(w.row0 + (pos - w.pos0)) * C.heads + h) * C.d + 8 * i8;
        if (!base) {
            store8<DT>(A.k_out, at, zeros);
            store8<DT>(A.v_out, at, zeros);
            continue;
        }
        const uint32_t kw = base[256 * ns + tok], vw = base[256 * ns + 32 + tok];
        const uint32_t kc = base[tok * 4 * ns + i8];
        const int g = kv4_group(tok), bit = kv4_bit(kv4_value(tok));
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            x[j] = value_of(kw, kv4_get(kc, kv4_bit(j)));
        store8<DT>(A.k_out, at, x);
        // eight values of one 16-value tile
        const int tile = i8 >> 1, m0 = 8 * (i8 & 1);
        const uint32_t* vc = base + 128 * ns + (((tile >> psh) * 4 + g) * 16 + m0) * pw + (tile & (pw - 1));
#pragma unroll
        for (int j = 0; j < 8; ++j)
            x[j] = value_of(vw, kv4_get(vc[j * pw], bit));
        store8<DT>(A.v_out, at, x);
    }
}

template <int DT>
const void* kernel_for(bool read, bool wide) {
    if (read) return wide ? (const void*)kv4_read_kernel<DT, 32> : (const void*)kv4_read_kernel<DT, 16>;
    return wide ? (const void*)kv4_append_kernel<DT, 32> : (const void*)kv4_append_kernel<DT, 16>;
}

hipError_t launch_store(const Kv4StoreArgs& A, int dt, bool read, hipStream_t stream) {
    const bool wide = A.c.d > 128;
    const void* f = dt == DT_F16 ? kernel_for<DT_F16>(read, wide)
                  : dt == DT_BF16 ? kernel_for<DT_BF16>(read, wide) : kernel_for<DT_F32>(read, wide);
    // one more unit than the sequences can touch: the rows behind the last
    int units = A.r.cu ? A.r.rows / 32 + 2 * A.c.seqs + 1 : A.c.seqs;
    Kv4StoreArgs a = A;
    void* args[] = {&a, &units};
    return launch(f, dim3(units, (A.c.heads + WAVES - 1) / WAVES), dim3(64 * WAVES), args, 0, stream);
}

}  // namespace

hipError_t launch_kv4_append(const Kv4StoreArgs& A, int dt, hipStream_t stream) {
    return launch_store(A, dt, false, stream);
}
hipError_t launch_kv4_read(const Kv4StoreArgs& A, int dt, hipStream_t stream) {
    return launch_store(A, dt, true, stream);
}

}  // namespace cbk
