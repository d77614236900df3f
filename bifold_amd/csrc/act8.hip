// Activation checkpoints in 8 bits (format: act8.h) and their use in the backward pass:
//   bf_act8_pack       x -> q, code                       what a training step keeps instead of a 16- or 32-bit activation
//   bf_act8_unpack     q, code -> x
//   bf_act8_gelu_fwd   pre -> y = act(pre), and the checkpoint of pre, in one pass
//   bf_act8_gelu_bwd   dy, checkpoint -> dpre = dy act'(q 2^e)
// All four stream: every byte is touched once and nothing is reused, so HBM bounds them (the 16-bit erf forward, at 4.8 TB/s,
// its vector instructions) and the layout is chosen for it.  A
// lane holds V = 8 consecutive elements (one 16-byte access of a 16-bit tensor, 8 bytes of q) or 4 of an fp32 tensor; a group
// of 32 is a quad of lanes (or two), its maximum two (three) cross-lane moves without LDS.  One vector a lane and many
// workgroups: 36 928 x 4 096 fp16 forward and backward 123 and 132 us, 6.2 and 5.8 TB/s (a copy of 2 GiB reaches 4.9, one of
// 256 MiB 5.5); with four vectors a lane in flight 129 and 159 where one took 119 and 137, both with ordinary loads.
#include "act8.h"

namespace {

enum { A8_PACK = 0, A8_UNPACK = 1, A8_FWD = 2, A8_BWD = 3 };

// ---- the activations.  s = 1 / (1 + e^-u):  quick GELU x s(1.702 x);  tanh GELU x s(2 c (x + 0.044715 x^3)), which is
// 0.5 x (1 + tanh) without its cancellation at negative x;  erf GELU x Phi(x).  Derivative of x s(u): s + x u' s (1 - s).
// fp32 tensors take the accurate exponential and division; 16-bit ones v_exp / v_rcp: the exponential of u is off by some
// (2 + |u|) 2^-23 of itself, under 2^-16 wherever it is a normal number, and the result is rounded to 2^-8 or 2^-11.  Where
// e^-u overflows (u < -88.7) the gate is 0: results under |x| 2^-127 are lost.  |x| is cut at 100 in their derivative (in
// fp32 it is 0 or 1 from there on), a NaN stays.
template <int ACT> __device__ __forceinline__ float gate_at(float x) {
    return ACT == BF_ACT_QUICK_GELU ? 1.702f * x : 1.5957691216057308f * fmaf(0.044715f * x * x, x, x);
}
template <int ACT, bool EXACT> __device__ __forceinline__ float gate(float x) {
    const float u = gate_at<ACT>(x);
    if constexpr (EXACT) return 1.0f / (1.0f + expf(-u));
    else return __builtin_amdgcn_rcpf(1.0f + __expf(-u));
}
// Phi(-|x|) and e^(-x^2/2) in fp32, without branches; the GELU's value is right to 7 units of 2^-24, its slope's terms to 5
// (73 728 x 768, forward 81 us, backward 83; with erfcf, whose lanes part at |x|, 89 and 93).  Phi(-a) = e^(-a^2/2) R(a), and
// R(a) (a + 3.75) is smooth and bounded: a polynomial of degree 8 in (a - 3.75) / (a + 3.75), the form Shepherd and Laframboise
// published for erfc (1981), fitted here by least squares of the relative error at 400 Chebyshev nodes on 0 <= a <= 15, to
// 4.6e-8 of the value.  The rounding of a^2 is made good behind the exponential.  From |x| = 15 on e^(-x^2/2)
// is under fp32's smallest number; |x| is cut at 20, where it is 0.
__device__ __forceinline__ float normal_tail(float x, float& e) {
    const float a = fminf(fabsf(x), 20.0f), h = a * a;
    e = expf(-0.5f * h);
    e = fmaf(e, -0.5f * fmaf(a, a, -h), e);
    const float q = __builtin_amdgcn_rcpf(a + 3.75f), u = (a - 3.75f) * q;
    float r = 4.4473037e-04f;
    r = fmaf(r, u, 5.11906e-04f);
    r = fmaf(r, u, -4.1687856e-03f);
    r = fmaf(r, u, 1.198799e-03f);
    r = fmaf(r, u, 3.7492145e-02f);
    r = fmaf(r, u, -1.5152062e-01f);
    r = fmaf(r, u, 3.5293967e-01f);
    r = fmaf(r, u, -5.881883e-01f);
    r = fmaf(r, u, 7.502941e-01f);
    return e * (r * q);
}
// The same for 16-bit tensors, whose squares are exact in fp32: right to (32 + x^2) 2^-24 of itself wherever e^(-x^2/2) is a
// normal number (|x| < 13.2).  1 + erf with an erf right to 1.5e-7 has no digits left from x = -5.5 on.  R(a) as a polynomial
// in q = 1 / (a + 3.75) without a constant term, fitted to 8.0e-7 of the value on 0 <= a <= 14.3 by least squares of the
// relative error whose weights are multiplied by the error again and again (Lawson's method for the least maximum).  36 928 x 4 096 fp16: forward 157 us, backward 134 (quick GELU 123 and 127: here the vector
// instructions bound the forward; with 1 + erf it took 149, the backward 138).
__device__ __forceinline__ float normal_tail_fast(float x, float& e) {
    const float a = fminf(fabsf(x), 20.0f);
    e = __builtin_amdgcn_exp2f(-0.72134752044448170368f * (a * a));          // -log2(e) / 2
    const float q = __builtin_amdgcn_rcpf(a + 3.75f);
    float r = -6.82312e+02f;
    r = fmaf(r, q, 5.075025e+02f);
    r = fmaf(r, q, -3.803952e+01f);
    r = fmaf(r, q, 2.6375841e+01f);
    r = fmaf(r, q, 4.5656223e+00f);
    r = fmaf(r, q, 1.5183665e+00f);
    r = fmaf(r, q, 3.9862776e-01f);
    return e * (r * q);
}
template <int ACT, bool EXACT> __device__ __forceinline__ float act_value(float x) {
    if constexpr (ACT == BF_ACT_ERF_GELU) {
        float e;
        const float t = EXACT ? normal_tail(x, e) : normal_tail_fast(x, e);
        return x * (x < 0.0f ? t : 1.0f - t);
    } else {
        return x * gate<ACT, EXACT>(x);
    }
}
template <int ACT, bool EXACT> __device__ __forceinline__ float act_slope(float x) {
    if constexpr (ACT == BF_ACT_ERF_GELU) {                    // a checkpoint's values are finite or NaN
        float e;
        const float t = EXACT ? normal_tail(x, e) : normal_tail_fast(x, e);
        return fmaf(x * 0.39894228040143267794f, e, x < 0.0f ? t : 1.0f - t);
    } else {
        x = fabsf(x) > 100.0f ? copysignf(100.0f, x) : x;
        const float du = ACT == BF_ACT_QUICK_GELU ? 1.702f : 1.5957691216057308f * fmaf(0.134145f * x, x, 1.0f);
        if constexpr (EXACT) {
            // s and 1 - s from one exponential, without the cancellation that an fp32 result could show: with v = e^-|u| the
            // larger is 1 / (1 + v), the smaller v / (1 + v)
            const float u = gate_at<ACT>(x), v = expf(-fabsf(u)), large = 1.0f / (1.0f + v), small = v * large;
            return fmaf(x * du, large * small, u < 0.0f ? small : large);
        } else {
            const float s = gate<ACT, EXACT>(x), r = 1.0f - s;
            return fmaf(x * du, s * r, s);
        }
    }
}

// One kernel body for the four: MODE picks what is read and written.  DENSE: cols is a multiple of 32, all rows follow each
// other and are 16-byte aligned, so vector v lies at element 8 v.  Otherwise a row owns a whole number of quads of lanes
// (the last ones partly or wholly empty), `vpr` vectors of 8 per row, and accesses may be unaligned: one division per vector.
struct A8Args {
    const void* x; int64_t ldx;             // A8_PACK / A8_FWD: the activation;  A8_BWD: dy
    void* y; int64_t ldy;                   // A8_FWD: act(pre);  A8_BWD: dpre;  A8_UNPACK: the tensor
    uint8_t* q; uint8_t* code;
    unsigned nvec; unsigned vpr; int cols; int gpr;
};

template <typename T, int MODE, int ACT, int A, int V>
__global__ __launch_bounds__(256) void act8_kernel(const A8Args a) {
    constexpr bool EXACT = sizeof(T) == 4;
    constexpr unsigned PER = ACT8_GROUP / V;                   // lanes per group
    const unsigned v = blockIdx.x * 256u + threadIdx.x;
    const bool live = v < a.nvec;
    int n;                                                     // elements of the row from here on (at most V; <= 0: behind it)
    size_t off_x, off_y, off_q, off_c;
    bool first;
    if constexpr (A == ROWS_ALIGNED) {
        if (MODE == A8_UNPACK && !live) return;                // no lane needs another: one branch around everything
        n = MODE == A8_UNPACK || live ? V : 0;
        off_x = off_y = off_q = (size_t)v * V;
        off_c = v / PER;
        first = v % PER == 0;
    } else {                                                   // lanes behind the last vector read it again
        const unsigned w = min(v, a.nvec - 1), row = w / a.vpr, c = (w - row * a.vpr) * V;
        n = min(V, a.cols - (int)c);
        off_x = (size_t)row * a.ldx + c;
        off_y = (size_t)row * a.ldy + c;
        off_q = (size_t)row * a.cols + c;
        off_c = (size_t)row * a.gpr + c / ACT8_GROUP;
        first = c % ACT8_GROUP == 0;
    }
    const int put = live ? n : 0;                              // elements to write
    const T* x = (const T*)a.x + off_x;
    T* y = (T*)a.y + off_y;
    float f[V];
    unsigned w[V / 4], code;
    if constexpr (MODE == A8_PACK || MODE == A8_FWD) {
        vec_load_n<T, V, A, true>(x, n, f);
        code = act8_code(group_max<V>(magnitude_bits<V>(f)));
        act8_quant<V>(f, code, w);
        bytes_store_n<V, A>(a.q + off_q, put, w);
        if (first && put > 0) a.code[off_c] = (uint8_t)code;
        if constexpr (MODE == A8_FWD) {
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = act_value<ACT, EXACT>(f[j]);
            vec_store_n<T, V, A>(y, put, f);
        }
    } else {
        Chunk<T, V, A> dy;
        Chunk<uint8_t, V, A> q;
        q.template load<true>(a.q, off_q, n);
        code = n > 0 ? a.code[off_c] : 1u;
        if constexpr (MODE == A8_BWD) dy.template load<true>(x, 0, n);
        q.words(w, n);
        act8_dequant<V>(w, code, f);
        if constexpr (MODE == A8_UNPACK && __is_same(T, f16_t)) {
            // 2^16 is what fp16's numbers from 65 280 on are kept as, and the one value of theirs that fp16 does not hold; a wave
            // seldom has a step of 2^10 or more
            if (__ballot(code >= 137u) != 0) {
#pragma unroll
                for (int j = 0; j < V; ++j) f[j] = fabsf(f[j]) == 65536.0f ? copysignf(65504.0f, f[j]) : f[j];
            }
        }
        if constexpr (MODE == A8_BWD) {
            float d[V];
            dy.take(d, n);
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = d[j] * act_slope<ACT, EXACT>(f[j]);
        }
        vec_store_n<T, V, A>(y, put, f);
    }
}

template <typename T, int MODE, int ACT>
void act8_launch(const A8Args& a, bool dense, hipStream_t s) {
    if (dense) {
        // fp32 writers of q take 4 elements a lane (whole lines per load instruction): 50 432 x 768 packed in 36 us,
        // with 8 in 38, GELU with its checkpoint 57 and 61; the read-back takes 8 (73 728 x 768 in 45 us, with 4 in 48)
        constexpr int V = sizeof(T) == 4 && MODE != A8_UNPACK ? 4 : 8;
        A8Args b = a;
        b.nvec = a.nvec * (8 / V);
        hipLaunchKernelGGL((act8_kernel<T, MODE, ACT, ROWS_ALIGNED, V>), dim3((unsigned)(((size_t)b.nvec + 255) / 256)), dim3(256), 0, s, b);
    } else {
        const dim3 grid((unsigned)(((size_t)a.nvec + 255) / 256));
        if (a.cols >= 8) hipLaunchKernelGGL((act8_kernel<T, MODE, ACT, ROWS_ANY, 8>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((act8_kernel<T, MODE, ACT, ROWS_TINY, 8>), grid, dim3(256), 0, s, a);
    }
}

template <int MODE, int ACT>
void act8_by_type(const A8Args& a, int dtype, bool dense, hipStream_t s) {
    if (dtype == BF_BF16) act8_launch<bf16_t, MODE, ACT>(a, dense, s);
    else if (dtype == BF_F16) act8_launch<f16_t, MODE, ACT>(a, dense, s);
    else act8_launch<float, MODE, ACT>(a, dense, s);
}

template <int MODE>
int act8_run(const char* name, const void* x, int64_t ldx, void* y, int64_t ldy, void* q, void* code, int dtype, int act,
             int64_t rows, int cols, bf_stream_t stream) {
    BF_REQUIRE(dtype == BF_F32 || bf_is_half(dtype), BF_EINVAL, "%s: bad dtype %d", name, dtype);
    BF_REQUIRE(rows >= 0 && cols > 0 && cols <= (1 << 30), BF_EINVAL, "%s: bad shape (rows=%lld cols=%d)", name, (long long)rows, cols);
    constexpr bool HAS_X = MODE != A8_UNPACK, HAS_Y = MODE != A8_PACK;
    BF_REQUIRE((!HAS_X || ldx >= cols) && (!HAS_Y || ldy >= cols), BF_EINVAL, "%s: a leading dimension is under cols=%d", name, cols);
    if (MODE == A8_FWD || MODE == A8_BWD)
        BF_REQUIRE(act == BF_ACT_QUICK_GELU || act == BF_ACT_ERF_GELU || act == BF_ACT_TANH_GELU, BF_EINVAL,
                   "%s: act must be BF_ACT_QUICK_GELU, BF_ACT_ERF_GELU or BF_ACT_TANH_GELU (got %d)", name, act);
    if (rows == 0) return BF_OK;
    BF_REQUIRE((!HAS_X || x) && (!HAS_Y || y) && q && code, BF_EINVAL, "%s: null pointer", name);
    const size_t esz = bf_dtype_size(dtype);
    BF_REQUIRE((!HAS_X || (uintptr_t)x % esz == 0) && (!HAS_Y || (uintptr_t)y % esz == 0), BF_EALIGN,
               "%s: a tensor is not aligned to its element", name);
    A8Args a;
    a.x = x; a.ldx = ldx; a.y = y; a.ldy = ldy; a.q = (uint8_t*)q; a.code = (uint8_t*)code;
    a.cols = cols; a.gpr = (cols + ACT8_GROUP - 1) / ACT8_GROUP;
    a.vpr = (unsigned)a.gpr * 4;
    BF_REQUIRE(rows <= (int64_t)(0x7FFFF000u / a.vpr), BF_EINVAL, "%s: rows=%lld x cols=%d is over 2^34 elements", name,
               (long long)rows, cols);
    a.nvec = (unsigned)rows * a.vpr;
    const bool dense = cols % ACT8_GROUP == 0 && (!HAS_X || (ldx == cols && bf_aligned16(x))) &&
                       (!HAS_Y || (ldy == cols && bf_aligned16(y))) && ((uintptr_t)q & 7u) == 0;
    hipStream_t s = (hipStream_t)stream;
    if (MODE == A8_PACK || MODE == A8_UNPACK) act8_by_type<MODE, BF_ACT_NONE>(a, dtype, dense, s);
    else if (act == BF_ACT_QUICK_GELU) act8_by_type<MODE, MODE == A8_FWD || MODE == A8_BWD ? BF_ACT_QUICK_GELU : 0>(a, dtype, dense, s);
    else if (act == BF_ACT_ERF_GELU) act8_by_type<MODE, MODE == A8_FWD || MODE == A8_BWD ? BF_ACT_ERF_GELU : 0>(a, dtype, dense, s);
    else act8_by_type<MODE, MODE == A8_FWD || MODE == A8_BWD ? BF_ACT_TANH_GELU : 0>(a, dtype, dense, s);
    BF_CHECK_LAUNCH(name);
    return BF_OK;
}

}  // namespace

extern "C" int bf_act8_pack(const void* x, int64_t ldx, int dtype, void* q, void* code, int64_t rows, int cols, bf_stream_t stream) {
    return act8_run<A8_PACK>("bf_act8_pack", x, ldx, nullptr, 0, q, code, dtype, 0, rows, cols, stream);
}
extern "C" int bf_act8_unpack(const void* q, const void* code, void* x, int64_t ldx, int dtype, int64_t rows, int cols,
                              bf_stream_t stream) {
    return act8_run<A8_UNPACK>("bf_act8_unpack", nullptr, 0, x, ldx, (void*)q, (void*)code, dtype, 0, rows, cols, stream);
}
extern "C" int bf_act8_gelu_fwd(const void* pre, int64_t ld_pre, void* y, void* q, void* code, int dtype, int act, int64_t rows,
                                int cols, bf_stream_t stream) {
    return act8_run<A8_FWD>("bf_act8_gelu_fwd", pre, ld_pre, y, cols, q, code, dtype, act, rows, cols, stream);
}
extern "C" int bf_act8_gelu_bwd(const void* dy, int64_t ld_dy, const void* q, const void* code, void* dpre, int64_t ld_dpre,
                                int dtype, int act, int64_t rows, int cols, bf_stream_t stream) {
    return act8_run<A8_BWD>("bf_act8_gelu_bwd", dy, ld_dy, dpre, ld_dpre, (void*)q, (void*)code, dtype, act, rows, cols, stream);
}
