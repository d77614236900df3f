// The 8-bit activation checkpoint (act8.hip, rmsnorm.hip): vector loads and stores of any alignment, the group's exponent,
// the conversion both ways.
//
// A row is cut into groups of 32 columns, the last one possibly shorter.  A group shares one power of two, 2^e, with e the
// smallest exponent for which round(max |x| 2^-e) <= 127 (and >= -126); element x is kept as q = round(x 2^-e), ties to
// even, in int8, and reads back as q 2^e.  Powers of two make the scaling exact: the one rounding is q's, off by at most
// 2^(e-1), which is at most max |x| / 127 (2^-127 where e = -126), and q 2^e is exact in fp32, bf16 and (inside its range)
// fp16.  A group of fp16 numbers whose largest is 65 280 or more keeps it as 64 * 2^10, one step over fp16's range: unpacking
// to fp16 writes +-2^16 as +-65 504, so finite fp16 values read back finite.  The byte kept per group is code = e + 127, the
// exponent field of 2^e as a float: 1 .. 247.  A group that holds a NaN, an infinity or a magnitude of
// 255 * 2^119 or more gets code 255, q = 0: 2^e is then infinity as a float and every element reads back as NaN, so an
// overflow still reaches the gradients (a loss scaler's check sees it).
#pragma once
#include "common.h"

#define ACT8_GROUP 32

// How a kernel reads rows in vectors of V elements.  ALIGNED: rows begin at addresses aligned to a vector (at most 16 bytes)
// and hold whole vectors.  ANY: rows of at least V elements anywhere; the vector at a row's end is read V elements in front
// of the end -- global memory takes unaligned 16-byte accesses on this target -- and moved down in registers, so an odd width
// costs split cache lines and some vector instructions, but no branch and no element-wise loads (20 000 x 1 155 bf16, RMS
// norm backward: 43 us, element by element 57).  TINY: shorter rows, element by element.
enum { ROWS_TINY = 0, ROWS_ANY = 1, ROWS_ALIGNED = 2 };

// w moved down by `bytes` (0 .. 4 W), zeros from above; `bytes` may differ from lane to lane
template <int W> __device__ __forceinline__ void shift_down(unsigned (&w)[W], int bytes) {
#pragma unroll
    for (int step = W; step >= 1; step >>= 1) {                // words
        const bool by = bytes & (4 * step);
#pragma unroll
        for (int k = 0; k < W; ++k) w[k] = by ? (k + step < W ? w[k + step] : 0u) : w[k];
    }
#pragma unroll
    for (int k = 0; k < W; ++k) w[k] = __builtin_amdgcn_alignbyte(k + 1 < W ? w[k + 1] : 0u, w[k], (unsigned)bytes & 3u);
}

// V elements of a row as they lie in memory, n of them (<= 0: none) in front of the row's end.  Nothing waits for the load
// until the values are taken: a conversion behind each of several loads, as a branch on a run-time type makes it, waits for
// one after the other.
template <typename T, int V, int A> struct Chunk {
    static constexpr int W = V * (int)sizeof(T) / 4;
    unsigned w[W];
    // ONCE: the kernel reads these words once and aligned rows take non-temporal loads, which leave the caches' lines to
    // others.  36 928 x 1 024 fp16 behind a producer that wrote the operands last / behind 1 GiB of other writes: RMS norm
    // forward with an add 47 / 58 us (ordinary loads 49 / 74), backward from the checkpoint 53 / 60 (54 / 94), GELU with its
    // checkpoint 32 / 35 (38 / 47).  Rows of ROWS_ANY share cache lines between lanes and lose by it where the operands were
    // written last (20 000 x 1 155 bf16 forward 41 instead of 36 us), so they keep ordinary loads.  Non-temporal stores gain
    // nothing and cost the unpacking of 73 728 x 768 fp32 84 us instead of 46.
    template <bool ONCE = false> __device__ __forceinline__ void load(const void* base, size_t off, int n) {
        const T* p = (const T*)base + off;
        if constexpr (A == ROWS_ANY) {
            get<false, sizeof(T)>(p + min(0, n - V));
        } else if constexpr (A == ROWS_ALIGNED) {
#pragma unroll
            for (int k = 0; k < W; ++k) w[k] = 0;
            if (n >= V) get<ONCE, sizeof(w) < 16 ? sizeof(w) : 16>(p);
        } else {
            T t[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                t[j] = T(0);
                if (j < n) t[j] = p[j];
            }
            __builtin_memcpy(w, t, sizeof(w));
        }
    }
    template <bool ONCE, int ALIGN> __device__ __forceinline__ void get(const T* p) {
        typedef unsigned piece __attribute__((ext_vector_type(W > 4 ? 4 : W), aligned(ALIGN)));
#pragma unroll
        for (int k = 0; k < W; k += 4) {
            piece q;
            if constexpr (ONCE) q = __builtin_nontemporal_load((const piece*)p + k / 4);
            else q = *((const piece*)p + k / 4);
            __builtin_memcpy(w + k, &q, sizeof(w) < 16 ? sizeof(w) : 16);
        }
    }
    // the words, zeros behind the row's end
    __device__ __forceinline__ void words(unsigned (&o)[W], int n) const {
#pragma unroll
        for (int k = 0; k < W; ++k) o[k] = w[k];
        if constexpr (A == ROWS_ANY) shift_down<W>(o, (V - max(0, min(n, V))) * (int)sizeof(T));
    }
    __device__ __forceinline__ void take(float (&o)[V], int n) const {
        typedef T vec __attribute__((ext_vector_type(V)));
        unsigned u[W];
        words(u, n);
        vec r;
        __builtin_memcpy(&r, u, sizeof(u));
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = to_f32<T>(r[j]);
    }
    // The load is complete behind this point.  (Stores count in vmcnt too: a wait that the compiler places between stores
    // which may or may not happen is a wait for those stores.)
    __device__ __forceinline__ void arrived() {
#pragma unroll
        for (int k = 0; k < W; ++k) asm volatile("" : "+v"(w[k]));
    }
};
template <typename T, int V, int A, bool ONCE = false> __device__ __forceinline__ void vec_load_n(const T* p, int n, float (&o)[V]) {
    Chunk<T, V, A> c;
    c.template load<ONCE>(p, 0, n);
    c.take(o, n);
}
template <typename T, int V, int A> __device__ __forceinline__ void vec_store_n(T* p, int n, const float (&v)[V]) {
    typedef T vec __attribute__((ext_vector_type(V)));
    vec r;
#pragma unroll
    for (int j = 0; j < V; ++j) r[j] = from_f32<T>(v[j]);
    if (n >= V) {
        if constexpr (A == ROWS_ALIGNED) __builtin_memcpy(__builtin_assume_aligned(p, sizeof(r) < 16 ? sizeof(r) : 16), &r, sizeof(r));
        else __builtin_memcpy(p, &r, sizeof(r));
    } else if constexpr (A != ROWS_ALIGNED) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < n) p[j] = r[j];
    }
}
// V bytes from V / 4 words
template <int V, int A> __device__ __forceinline__ void bytes_store_n(uint8_t* p, int n, const unsigned (&w)[V / 4]) {
    if (n >= V) {
        if constexpr (A == ROWS_ALIGNED) __builtin_memcpy(__builtin_assume_aligned(p, V), w, V);
        else __builtin_memcpy(p, w, V);
    } else if constexpr (A != ROWS_ALIGNED) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < n) p[j] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
    }
}
// the wave's number in its workgroup, as the scalar it is: rows, tokens and branches that depend on it stay scalar too
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

// Largest magnitude of V elements as the bits of a non-negative float: an integer maximum, so a NaN (whose bits lie above
// infinity's) is kept where fmaxf would drop it.
template <int V>
__device__ __forceinline__ unsigned magnitude_bits(const float (&x)[V]) {
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const unsigned b = __float_as_uint(x[j]) & 0x7FFFFFFFu;
        m = m > b ? m : b;
    }
    return m;
}
// maximum over the 32 / V neighbouring lanes that hold one group (V = 8: a quad, V = 4: two quads).  All lanes of the group
// must be active.
template <int V>
__device__ __forceinline__ unsigned group_max(unsigned v) {
    static_assert(V == 8 || V == 4, "a group is a quad of 8-element lanes or eight 4-element lanes");
    unsigned o = (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true);       // quad_perm [1, 0, 3, 2]
    v = v > o ? v : o;
    o = (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true);                // quad_perm [2, 3, 0, 1]
    v = v > o ? v : o;
    if constexpr (V == 4) {
        o = (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true);           // row_half_mirror: the other quad
        v = v > o ? v : o;
    }
    return v;
}

// The group's byte.  With max |x| = m 2^k, 1 <= m < 2, e = k - 6 puts it into [64, 128); where it would round to 128
// (m >= 255 / 128, mantissa field >= 0x7F0000) adding 0x10000 carries into the exponent field.
__device__ __forceinline__ unsigned act8_code(unsigned amax_bits) {
    const int c = (int)((amax_bits + 0x10000u) >> 23) - 6;
    return c >= 248 ? 255u : c < 1 ? 1u : (unsigned)c;
}
__device__ __forceinline__ float act8_step(unsigned code) { return __uint_as_float(code << 23); }      // 2^e; 255: infinity

// Four elements to four bytes: x 2^-e + 1.5 * 2^23 rounds to an integer (ties to even) whose two's complement is the low
// byte of the sum's bits; two byte permutes join them.
__device__ __forceinline__ unsigned act8_quant4(float a, float b, float c, float d, float inv) {
    const float magic = 12582912.0f;
    const unsigned ia = __float_as_uint(fmaf(a, inv, magic)), ib = __float_as_uint(fmaf(b, inv, magic));
    const unsigned ic = __float_as_uint(fmaf(c, inv, magic)), id = __float_as_uint(fmaf(d, inv, magic));
    const unsigned lo = __builtin_amdgcn_perm(ib, ia, 0x0c0c0400u), hi = __builtin_amdgcn_perm(id, ic, 0x0c0c0400u);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}
template <int V>
__device__ __forceinline__ void act8_quant(const float (&x)[V], unsigned code, unsigned (&w)[V / 4]) {
    const float inv = __uint_as_float((254u - code) << 23);                              // 2^-e (not used for code 255)
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
        const unsigned q = act8_quant4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3], inv);
        w[j] = code == 255u ? 0u : q;
    }
}
// q 2^e = (u - 128) 2^e with u = q + 128 unsigned (one conversion instruction per byte); both terms and the sum are exact.
template <int V>
__device__ __forceinline__ void act8_dequant(const unsigned (&w)[V / 4], unsigned code, float (&x)[V]) {
    const float s = act8_step(code), off = -128.0f * s;
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
        const unsigned u = w[j] ^ 0x80808080u;
        x[4 * j] = fmaf((float)(u & 255u), s, off);
        x[4 * j + 1] = fmaf((float)((u >> 8) & 255u), s, off);
        x[4 * j + 2] = fmaf((float)((u >> 16) & 255u), s, off);
        x[4 * j + 3] = fmaf((float)(u >> 24), s, off);
    }
}
