// kv4_store.hip -- new tokens' keys and values into the paged 4-bit cache, and back out of it.
//
// Quantizing a vector x of a token and head (kv4.hpp's format): over lo = min(0, min x) and
// hi = max(0, max x), r = hi - lo and z = rint(-15 lo / r) in 64 bits, the word
// (bits(max(float(r / 15), 2^-100)) & ~15) | z, whose float is s, and c = clamp(rint(x / s) + z, 0, 15)
// with x / s at its exact value (halves to even).  The codes follow the definition exactly, at borders too:
// a rounded quotient would move a whole step.  rint(x * (1 / s)) is off by at most one, and
// e = x - q s, exact in one FMA where it matters (near s / 2 it is a multiple of half x's last place
// below 2^24 of them), says which way.
//
// A wave has one block of 32 tokens of one head.  K: 16 lanes (32 above 128 values) hold a token, eight
// values each, and write one word each.  V's words hold eight tokens of one value: the codes pass
// through LDS as bytes [value][token].  A block that is not all new keeps the other tokens' codes.
// Bound: the bytes (the 16-bit values in, codes out).
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

// x / s rounded to the nearest whole number (halves to even), exactly, for |x / s| < 2^22.
__device__ __forceinline__ float exact_quotient(float x, float s, float inv) {
    float q = __builtin_rintf(x * inv);
    const float e = __builtin_fmaf(-q, s, x), half = 0.5f * s;
    const bool odd = ((int)q & 1) != 0;
    if (e > half || (e == half && odd)) q += 1.f;
    if (e < -half || (e == -half && odd)) q -= 1.f;
    return q;
}

template <int W>
__device__ __forceinline__ float row_min(float v) {
#pragma unroll
    for (int m = 1; m < W; m <<= 1) v = fminf(v, __shfl_xor(v, m));
    return v;
}
template <int W>
__device__ __forceinline__ float row_max(float v) {
#pragma unroll
    for (int m = 1; m < W; m <<= 1) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}

// Eight values of a vector spread over W lanes -> their codes and the vector's word.
template <int W>
__device__ __forceinline__ uint32_t quantize8(const float (&x)[8], int (&c)[8]) {
    float lo = 0.f, hi = 0.f;
    bool fine = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        lo = fminf(lo, x[j]);
        hi = fmaxf(hi, x[j]);
        fine &= __builtin_fabsf(x[j]) < __builtin_inff();
    }
    lo = row_min<W>(lo);
    hi = row_max<W>(hi);
    const float bad = row_max<W>(fine ? 0.f : 1.f);
    const double r = (double)hi - (double)lo;
    const int z = r > 0.0 ? (int)__builtin_rint(-15.0 * (double)lo / r) : 0;
    const float step = fmaxf((float)(r / 15.0), KV4_MIN_SCALE);
    uint32_t word = (__float_as_uint(step) & ~15u) | (uint32_t)z;
    const float s = __uint_as_float(word), inv = 1.0f / s;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float q = exact_quotient(x[j], s, inv) + (float)z;
        c[j] = (int)fminf(fmaxf(q, 0.f), 15.f);
    }
    if (bad != 0.f) {
        word = 0x7FC00000u;
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = 0;
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
    uint32_t* meta = base + 256 * ns;
    uint8_t* lds = codes[wave];
    for (int t0 = 32 * blk; t0 < 32 * blk + 32; t0 += TOK) {
        if (t0 + TOK <= lo || t0 >= hi) continue;
        const int pos = t0 + sub, tok = pos - 32 * blk;
        const bool is_new = pos >= lo && pos < hi;
        float xk[8] = {}, xv[8] = {};
        if (is_new && mine) {
            const long row = w.row0 + (pos - w.pos0);
            load8<DT>(A.k, row * A.k_row + h * A.k_head + 8 * i8, xk);
            load8<DT>(A.v, row * A.v_row + h * A.v_head + 8 * i8, xv);
        }
        int c[8];
        const uint32_t kw = quantize8<W>(xk, c);
        if (!mine) {
#pragma unroll
            for (int j = 0; j < 8; ++j) c[j] = 0;
        }
        if (is_new) {
            if (i8 < 4 * ns) {
                uint32_t word = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) word |= kv4_put((uint32_t)c[j], j);
                base[tok * 4 * ns + i8] = word;
            }
            if (i8 == 0) meta[tok] = kw;
        }
        const uint32_t vw = quantize8<W>(xv, c);
        if (!mine) {
#pragma unroll
            for (int j = 0; j < 8; ++j) c[j] = 0;
        }
        if (is_new && i8 == 0) meta[32 + tok] = vw;
        if (is_new && i8 < 4 * ns) {
#pragma unroll
            for (int j = 0; j < 8; ++j) lds[(8 * i8 + j) * PITCH + tok] = (uint8_t)c[j];
        }
    }
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_s_waitcnt(0xF | (0x3 << 14) | (0x7 << 4));    // lgkmcnt(0): the wave's own bytes
    asm volatile("" ::: "memory");
    const int psh = ns & 1 ? 1 : 2;                    // log2 of the words of a piece
    uint32_t* vc = base + 128 * ns;
    for (int x = lane; x < 128 * ns; x += 64) {
        const int e = x & ((1 << psh) - 1), y = x >> psh;
        const int m = y & 15, g = (y >> 4) & 3, piece = y >> 6;
        const int d = 16 * ((piece << psh) + e) + m;
        uint32_t keep = 0, word = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int tok = 4 * g + (j & 3) + 16 * (j >> 2), pos = 32 * blk + tok;
            if (pos >= lo && pos < hi) word |= kv4_put(lds[d * PITCH + tok], j);
            else keep |= kv4_put(15u, j);
        }
        if (keep == 0xFFFFFFFFu) continue;
        if (keep) word |= vc[x] & keep;
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
