// Root-mean-square norm with the residual's addition (forward, to 16 / 32 bits or to e4m3 with a row scale) and its backward.
//   forward:   t = x + delta;  r = 1 / sqrt(mean t^2 + eps);  y = t r gamma
//              e4m3: s = max |y| / 448 (1 for a row of zeros, NaN for one that holds a NaN or an infinity), y8 = e4m3(y / s)
//   backward:  h = t r;  b = dy gamma;  dx = dres + r (b - h mean(b h));  dgamma = sum over rows of dy h
// The forward can leave the 8-bit checkpoint of t (act8.h) from the registers that hold the row; the backward takes t as a
// tensor or as that checkpoint.  Statistics and sums are fp32.  t enters y, r and the checkpoint unrounded; x_out is t
// rounded once to the stream's type.
//
// HBM bounds both: each tensor is read once and written once, the row stays in registers between the sum and the output.  A
// lane holds V consecutive elements per chunk: 4 of an fp32 stream, 8 of a 16-bit one (16 bytes either way).  Rows up to
// 1 024 columns belong to one wave (reductions without LDS or barriers, four rows per workgroup); up to 16 384 to one
// workgroup (of four waves, over 8 192 of sixteen); longer ones are walked two or three times.  Measured: 50 432 x 768, fp32
// stream + fp16 branch to e4m3, sum written: 68 us, 6.3 TB/s; 36 928 x 1 024 to fp16 with the checkpoint 84 us, 5.9 TB/s, and
// its backward from the checkpoint 46 + 5 us, 5.8 TB/s (a copy of 2 GiB reaches 4.9, one of 256 MiB 5.5).
#include "act8.h"

namespace {

enum { Y_E4M3 = 3 };                            // beside BF_F32 / BF_BF16 / BF_F16 as a store format
#define RMS_FP8_MAX 448.0f

struct RmsFwd {
    const void* x; int64_t ldx;
    const void* delta; int64_t ldd; int d_dtype;
    const float* gamma;
    void* x_out; int64_t ldo;
    void* y; int y_dtype; float* y_scale; float* rstd;
    uint8_t* q; uint8_t* code;
    int rows, cols, gpr; float eps;
};
struct RmsBwd {
    const void* dy; int64_t ldy;
    const void* x; int64_t ldx; int x_dtype; const uint8_t* q; const uint8_t* code;
    const float* gamma; const float* rstd;
    const void* dres; int64_t ldr;
    void* dx; int dx_dtype;
    float* part;
    int rows, cols, gpr, nblk;
};

template <int V, int A> __device__ __forceinline__ void load_as(const void* p, int dtype, size_t off, int n, float (&o)[V]) {
    if (dtype == BF_F32) vec_load_n<float, V, A>((const float*)p + off, n, o);
    else if (dtype == BF_BF16) vec_load_n<bf16_t, V, A>((const bf16_t*)p + off, n, o);
    else vec_load_n<f16_t, V, A>((const f16_t*)p + off, n, o);
}
template <int V, int A> __device__ __forceinline__ void store_as(void* p, int dtype, size_t off, int n, const float (&v)[V]) {
    if (dtype == BF_F32) vec_store_n<float, V, A>((float*)p + off, n, v);
    else if (dtype == BF_BF16) vec_store_n<bf16_t, V, A>((bf16_t*)p + off, n, v);
    else vec_store_n<f16_t, V, A>((f16_t*)p + off, n, v);
}
template <int V> __device__ __forceinline__ void to_e4m3(const float (&y)[V], float inv, unsigned (&w)[V / 4]) {
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
        float f[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = fminf(RMS_FP8_MAX, fmaxf(-RMS_FP8_MAX, y[4 * j + k] * inv));
        int p = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
        w[j] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], p, true);
    }
}
// a row's scale from the bits of its largest magnitude (infinity and NaN lie at 0x7F800000 and above)
__device__ __forceinline__ float e4m3_scale(unsigned amax_bits) {
    if (amax_bits >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
    return amax_bits ? fmaxf(__uint_as_float(amax_bits) / RMS_FP8_MAX, 1.17549435e-38f) : 1.0f;    // 1 / s stays finite
}
__device__ __forceinline__ unsigned wave_max_bits(unsigned v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned w = (unsigned)__shfl_xor((int)v, o, 64);
        v = v > w ? v : w;
    }
    return v;
}
// sum / maximum over the WPR waves that share a row; `red` has one slot per wave and is used once between barriers
template <int WPR> __device__ __forceinline__ float row_sum(float v, float* red) {
    v = wave_sum(v);
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < WPR; ++w) v += red[w];
    }
    return v;
}
template <int WPR> __device__ __forceinline__ unsigned row_max(unsigned v, unsigned* red) {
    v = wave_max_bits(v);
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int w = 0; w < WPR; ++w) v = v > red[w] ? v : red[w];
    }
    return v;
}
template <int V, int A>
__device__ __forceinline__ void keep8(const RmsFwd& a, int row, int c, int n, const float (&t)[V]) {
    const unsigned code = act8_code(group_max<V>(magnitude_bits<V>(t)));
    unsigned w[V / 4];
    act8_quant<V>(t, code, w);
    bytes_store_n<V, A>(a.q + (size_t)row * a.cols + c, n, w);
    if ((c & 31) == 0 && n > 0) a.code[(size_t)row * a.gpr + (c >> 5)] = (uint8_t)code;
}

template <typename TD, int V, int T, int NV, int A>
__device__ __forceinline__ void add_row(const RmsFwd& a, int row, int slot, float (&t)[NV][V]) {
    const TD* p = (const TD*)a.delta + (size_t)row * a.ldd;
    float d[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * T + slot) * V;
        vec_load_n<TD, V, A, true>(p + c, a.cols - c, d[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) t[i][j] += d[i][j];
}

// ------------------------------------------------------------------ forward, the row in registers (cols <= 64 WPR V NV)
template <typename TX, int V, int WPR, int NV, int A>
__global__ __launch_bounds__(WPR == 16 ? 1024 : 256) void rms_fwd_kernel(const RmsFwd a) {
    constexpr int T = 64 * WPR;
    __shared__ float red_s[WPR];
    __shared__ unsigned red_m[WPR];
    const int row = WPR == 1 ? blockIdx.x * 4 + wave_id() : blockIdx.x;
    if (row >= a.rows) return;
    const int slot = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
    const TX* x = (const TX*)a.x + (size_t)row * a.ldx;
    float t[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * T + slot) * V;
        vec_load_n<TX, V, A, true>(x + c, a.cols - c, t[i]);
    }
    if (a.delta) {                              // all chunks' loads first: a conversion between them would wait for each
        if (a.d_dtype == BF_F32) add_row<float, V, T, NV, A>(a, row, slot, t);
        else if (a.d_dtype == BF_BF16) add_row<bf16_t, V, T, NV, A>(a, row, slot, t);
        else add_row<f16_t, V, T, NV, A>(a, row, slot, t);
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) s = fmaf(t[i][j], t[i][j], s);
    if (a.x_out) {
        TX* o = (TX*)a.x_out + (size_t)row * a.ldo;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * T + slot) * V;
            vec_store_n<TX, V, A>(o + c, a.cols - c, t[i]);
        }
    }
    if (a.q) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * T + slot) * V;
            keep8<V, A>(a, row, c, a.cols - c, t[i]);
        }
    }
    const float r = 1.0f / sqrtf(row_sum<WPR>(s, red_s) / (float)a.cols + a.eps);
    if (a.rstd && slot == 0) a.rstd[row] = r;
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * T + slot) * V;
        float g[V];
        vec_load_n<float, V, A>(a.gamma + c, a.cols - c, g);
#pragma unroll
        for (int j = 0; j < V; ++j) t[i][j] = t[i][j] * r * g[j];
        const unsigned b = magnitude_bits<V>(t[i]);
        m = m > b ? m : b;
    }
    const size_t yo = (size_t)row * a.cols;
    if (a.y_dtype == Y_E4M3) {
        const float sc = e4m3_scale(row_max<WPR>(m, red_m)), inv = 1.0f / sc;
        if (slot == 0) a.y_scale[row] = sc;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * T + slot) * V;
            unsigned w[V / 4];
            to_e4m3<V>(t[i], inv, w);
            bytes_store_n<V, A>((uint8_t*)a.y + yo + c, a.cols - c, w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * T + slot) * V;
            store_as<V, A>(a.y, a.y_dtype, yo + c, a.cols - c, t[i]);
        }
    }
}

// ------------------------------------------------------------------ forward, any width: one workgroup walks the row
template <typename TX, int A>
__global__ __launch_bounds__(256) void rms_fwd_long_kernel(const RmsFwd a) {
    constexpr int V = 8;
    __shared__ float red_s[4];
    __shared__ unsigned red_m[4];
    const int row = blockIdx.x;
    const TX* x = (const TX*)a.x + (size_t)row * a.ldx;
    // t of this thread's chunk; x is read before x_out (which may be x) is written, and only by this thread
    auto chunk = [&](int c, float (&t)[V]) __attribute__((always_inline)) {
        vec_load_n<TX, V, A>(x + c, a.cols - c, t);
        if (a.delta) {
            float d[V];
            load_as<V, A>(a.delta, a.d_dtype, (size_t)row * a.ldd + c, a.cols - c, d);
#pragma unroll
            for (int j = 0; j < V; ++j) t[j] += d[j];
        }
    };
    auto scaled = [&](int c, float r, float (&t)[V]) __attribute__((always_inline)) {
        float g[V];
        vec_load_n<float, V, A>(a.gamma + c, a.cols - c, g);
#pragma unroll
        for (int j = 0; j < V; ++j) t[j] = t[j] * r * g[j];
    };
    float t[V], s = 0.f;
    for (int base = 0; base < a.cols; base += 256 * V) {
        const int c = base + threadIdx.x * V;
        chunk(c, t);
#pragma unroll
        for (int j = 0; j < V; ++j) s = fmaf(t[j], t[j], s);
        if (a.q) keep8<V, A>(a, row, c, a.cols - c, t);
    }
    const float r = 1.0f / sqrtf(row_sum<4>(s, red_s) / (float)a.cols + a.eps);
    if (a.rstd && threadIdx.x == 0) a.rstd[row] = r;
    float inv = 1.0f;
    if (a.y_dtype == Y_E4M3) {
        unsigned m = 0;
        for (int c = threadIdx.x * V; c < a.cols; c += 256 * V) {
            chunk(c, t);
            scaled(c, r, t);
            const unsigned b = magnitude_bits<V>(t);
            m = m > b ? m : b;
        }
        const float sc = e4m3_scale(row_max<4>(m, red_m));
        if (threadIdx.x == 0) a.y_scale[row] = sc;
        inv = 1.0f / sc;
    }
    const size_t yo = (size_t)row * a.cols;
    for (int c = threadIdx.x * V; c < a.cols; c += 256 * V) {
        chunk(c, t);
        if (a.x_out) vec_store_n<TX, V, A>((TX*)a.x_out + (size_t)row * a.ldo + c, a.cols - c, t);
        scaled(c, r, t);
        if (a.y_dtype == Y_E4M3) {
            unsigned w[V / 4];
            to_e4m3<V>(t, inv, w);
            bytes_store_n<V, A>((uint8_t*)a.y + yo + c, a.cols - c, w);
        } else {
            store_as<V, A>(a.y, a.y_dtype, yo + c, a.cols - c, t);
        }
    }
}

// ------------------------------------------------------------------ backward
struct Kept {};                                 // the stream is a checkpoint

template <typename TX, int V, int A> struct StreamChunk {
    Chunk<TX, V, A> x;
    __device__ __forceinline__ void load(const RmsBwd& a, int row, int c, int n) { x.template load<true>(a.x, (size_t)row * a.ldx + c, n); }
    __device__ __forceinline__ void take(int n, float (&t)[V]) const { x.take(t, n); }
};
template <int V, int A> struct StreamChunk<Kept, V, A> {
    Chunk<uint8_t, V, A> q;
    unsigned code;
    __device__ __forceinline__ void load(const RmsBwd& a, int row, int c, int n) {
        q.template load<true>(a.q, (size_t)row * a.cols + c, n);
        code = a.code[(size_t)row * a.gpr + (n > 0 ? c >> 5 : 0)];
    }
    __device__ __forceinline__ void take(int n, float (&t)[V]) const {
        unsigned w[V / 4];
        q.words(w, n);
        act8_dequant<V>(w, code, t);
        if (n < V) {                            // a NaN group's missing columns are no part of the row
#pragma unroll
            for (int j = 0; j < V; ++j) t[j] = j < n ? t[j] : 0.f;
        }
    }
};

// Workgroups walk rows (nblk of them side by side); a lane keeps its columns' share of dgamma over all its rows in
// registers, the workgroup writes one row of partial sums and rms_dgamma_kernel adds those in a fixed order.  A row's three
// loads are issued together, in the types they have (template: a branch on a type at run time would convert, and so wait,
// between them).
template <typename TDY, typename TX, typename TD, int V, int WPR, int NV, int A>
__global__ __launch_bounds__(WPR == 16 ? 1024 : 256) void rms_bwd_kernel(const RmsBwd a) {
    constexpr int T = 64 * WPR;
    __shared__ float red[2][WPR];
    extern __shared__ float fold[];             // WPR == 1: [4][cols]
    const int wave = wave_id();
    const int slot = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int stride = WPR == 1 ? a.nblk * 4 : a.nblk;
    float g[NV][V], acc[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * T + slot) * V;
        vec_load_n<float, V, A>(a.gamma + c, a.cols - c, g[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) acc[i][j] = 0.f;
    }
    int turn = 0;
    for (int row = WPR == 1 ? blockIdx.x * 4 + wave : blockIdx.x; row < a.rows; row += stride, turn ^= 1) {
        Chunk<TDY, V, A> dy[NV];
        StreamChunk<TX, V, A> x[NV];
        Chunk<TD, V, A> dres[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * T + slot) * V;
            dy[i].template load<true>(a.dy, (size_t)row * a.ldy + c, a.cols - c);
            x[i].load(a, row, c, a.cols - c);
        }
        if (a.dres) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * T + slot) * V;
                dres[i].template load<true>(a.dres, (size_t)row * a.ldr + c, a.cols - c);
            }
        }
        const float r = a.rstd[row];
        float b[NV][V], h[NV][V], s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int n = a.cols - (i * T + slot) * V;
            dy[i].take(b[i], n);
            x[i].take(n, h[i]);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                h[i][j] *= r;
                acc[i][j] = fmaf(b[i][j], h[i][j], acc[i][j]);
                b[i][j] *= g[i][j];
                s = fmaf(b[i][j], h[i][j], s);
            }
        }
        const float m = row_sum<WPR>(s, red[turn]) / (float)a.cols;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * T + slot) * V, n = a.cols - c;
#pragma unroll
            for (int j = 0; j < V; ++j) b[i][j] = r * (b[i][j] - h[i][j] * m);
            if (a.dres) {
                float d[V];
                dres[i].take(d, n);
#pragma unroll
                for (int j = 0; j < V; ++j) b[i][j] += d[j];
            }
            vec_store_n<TD, V, A>((TD*)a.dx + (size_t)row * a.cols + c, n, b[i]);
        }
    }
    float* part = a.part + (size_t)blockIdx.x * a.cols;
    if constexpr (WPR == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * T + slot) * V;
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (c + j < a.cols) fold[wave * a.cols + c + j] = acc[i][j];
        }
        __syncthreads();
        for (int c = threadIdx.x; c < a.cols; c += 256)
            part[c] = (fold[c] + fold[a.cols + c]) + (fold[2 * a.cols + c] + fold[3 * a.cols + c]);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * T + slot) * V;
            vec_store_n<float, V, A>(part + c, a.cols - c, acc[i]);
        }
    }
}

// t of one chunk, its type chosen at run time
template <int V, int A>
__device__ __forceinline__ void stream_load(const RmsBwd& a, int row, int c, int n, float (&t)[V]) {
    if (a.q) {
        StreamChunk<Kept, V, A> k;
        k.load(a, row, c, n);
        k.take(n, t);
    } else {
        load_as<V, A>(a.x, a.x_dtype, (size_t)row * a.ldx + c, n, t);
    }
}

// any width and any mixture of types: dx by one workgroup per row, two walks; dgamma by columns, a thread per column and
// chunk of rows
template <typename TDY, int A>
__global__ __launch_bounds__(256) void rms_bwd_long_kernel(const RmsBwd a) {
    constexpr int V = 8;
    __shared__ float red[4];
    for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const TDY* dy = (const TDY*)a.dy + (size_t)row * a.ldy;
        const float r = a.rstd[row];
        auto chunk = [&](int c, float (&b)[V], float (&h)[V]) __attribute__((always_inline)) {
            float g[V];
            vec_load_n<TDY, V, A>(dy + c, a.cols - c, b);
            vec_load_n<float, V, A>(a.gamma + c, a.cols - c, g);
            stream_load<V, A>(a, row, c, a.cols - c, h);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                b[j] *= g[j];
                h[j] *= r;
            }
        };
        float b[V], h[V], s = 0.f;
        for (int c = threadIdx.x * V; c < a.cols; c += 256 * V) {
            chunk(c, b, h);
#pragma unroll
            for (int j = 0; j < V; ++j) s = fmaf(b[j], h[j], s);
        }
        const float m = row_sum<4>(s, red) / (float)a.cols;
        for (int c = threadIdx.x * V; c < a.cols; c += 256 * V) {
            chunk(c, b, h);
#pragma unroll
            for (int j = 0; j < V; ++j) b[j] = r * (b[j] - h[j] * m);
            if (a.dres) {
                float d[V];
                load_as<V, A>(a.dres, a.dx_dtype, (size_t)row * a.ldr + c, a.cols - c, d);
#pragma unroll
                for (int j = 0; j < V; ++j) b[j] += d[j];
            }
            store_as<V, A>(a.dx, a.dx_dtype, (size_t)row * a.cols + c, a.cols - c, b);
        }
        __syncthreads();                        // red is written again
    }
}
// Launched in front of rms_bwd_long_kernel, which may write dx over dy.
template <typename TDY>
__global__ __launch_bounds__(256) void rms_dgamma_long_kernel(const RmsBwd a) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.cols) return;
    float s = 0.f;
    for (int row = blockIdx.y; row < a.rows; row += a.nblk) {
        float t[1];
        if (a.q) {
            const float step = act8_step(a.code[(size_t)row * a.gpr + (c >> 5)]);
            t[0] = (float)(int8_t)a.q[(size_t)row * a.cols + c] * step;
        } else {
            t[0] = a.x_dtype == BF_F32 ? ((const float*)a.x)[(size_t)row * a.ldx + c]
                 : a.x_dtype == BF_BF16 ? to_f32<bf16_t>(((const bf16_t*)a.x)[(size_t)row * a.ldx + c])
                                        : to_f32<f16_t>(((const f16_t*)a.x)[(size_t)row * a.ldx + c]);
        }
        s = fmaf(to_f32<TDY>(((const TDY*)a.dy)[(size_t)row * a.ldy + c]), t[0] * a.rstd[row], s);
    }
    a.part[(size_t)blockIdx.y * a.cols + c] = s;
}

// dgamma[c] = sum of nparts rows of partial sums: 32 columns x 32 row lanes per workgroup, joined in a fixed order
__global__ __launch_bounds__(1024) void rms_dgamma_kernel(const float* __restrict__ part, float* __restrict__ out, int nparts,
                                                          int cols) {
    __shared__ float red[32][33];
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + cl;
    float s = 0.f;
    if (c < cols) {
#pragma unroll 8
        for (int p = rl; p < nparts; p += 32) s += part[(size_t)p * cols + c];
    }
    red[rl][cl] = s;
    __syncthreads();
    if (rl == 0 && c < cols) {
        s = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) s += red[k][cl];
        out[c] = s;
    }
}

// ------------------------------------------------------------------ dispatch
#define RMS_LONG 16384                          /* widest row kept in the registers of one workgroup */
#define RMS_SLICE (1 << 21)                     /* rows of one forward launch; a multiple of every alignment */
static_assert((unsigned long long)RMS_SLICE * 1024 < 1ull << 32, "a grid counts threads in 32 bits");
#define RMS_MOST (1 << 30)                      /* rows, columns */

template <typename TX, int V, int A> void rms_fwd_launch(const RmsFwd& a, hipStream_t s) {
    const dim3 wave((unsigned)((a.rows + 3) / 4)), wg((unsigned)a.rows), block(256);
    const int chunks = (a.cols + V - 1) / V;
#define RMS_FWD(W, N) hipLaunchKernelGGL((rms_fwd_kernel<TX, V, W, N, A>), W == 1 ? wave : wg, W == 16 ? dim3(1024) : block, 0, s, a)
    if constexpr (V == 4) {                      // 1 024 columns to a wave, 8 192 to four, 16 384 to sixteen
        if (chunks <= 64) RMS_FWD(1, 1);
        else if (chunks <= 128) RMS_FWD(1, 2);
        else if (chunks <= 192) RMS_FWD(1, 3);
        else if (chunks <= 256) RMS_FWD(1, 4);
        else if (chunks <= 512) RMS_FWD(4, 2);
        else if (chunks <= 1024) RMS_FWD(4, 4);
        else if (chunks <= 2048) RMS_FWD(4, 8);
        else RMS_FWD(16, 4);
    } else {
        if (chunks <= 64) RMS_FWD(1, 1);
        else if (chunks <= 128) RMS_FWD(1, 2);
        else if (chunks <= 192) RMS_FWD(1, 3);  // 40 000 x 1 536 with an add: 77 us, as a workgroup per row 85; 16 384 x 2 048: 36 and 32
        else if (chunks <= 256) RMS_FWD(4, 1);
        else if (chunks <= 512) RMS_FWD(4, 2);
        else if (chunks <= 1024) RMS_FWD(4, 4);
        else RMS_FWD(16, 2);
    }
#undef RMS_FWD
}
template <typename TDY, typename TX, typename TD, int V, int A> void rms_bwd_launch(const RmsBwd& a, hipStream_t s) {
    const dim3 grid((unsigned)a.nblk), block(256);
    const int chunks = (a.cols + V - 1) / V;
    const size_t lds = (size_t)16 * a.cols;     // WPR == 1: at most 16 KB
#define RMS_BWD(W, N) hipLaunchKernelGGL((rms_bwd_kernel<TDY, TX, TD, V, W, N, A>), grid, W == 16 ? dim3(1024) : block, W == 1 ? lds : 0, s, a)
    if constexpr (V == 4) {                      // 1 024 columns to a wave, 8 192 to four, 16 384 to sixteen
        if (chunks <= 64) RMS_BWD(1, 1);
        else if (chunks <= 128) RMS_BWD(1, 2);
        else if (chunks <= 192) RMS_BWD(1, 3);
        else if (chunks <= 256) RMS_BWD(1, 4);
        else if (chunks <= 512) RMS_BWD(4, 2);
        else if (chunks <= 1024) RMS_BWD(4, 4);
        else if (chunks <= 2048) RMS_BWD(4, 8);
        else RMS_BWD(16, 4);
    } else {
        if (chunks <= 64) RMS_BWD(1, 1);
        else if (chunks <= 128) RMS_BWD(1, 2);
        else if (chunks <= 256) RMS_BWD(4, 1);
        else if (chunks <= 512) RMS_BWD(4, 2);
        else if (chunks <= 1024) RMS_BWD(4, 4);
        else RMS_BWD(16, 2);
    }
#undef RMS_BWD
}

template <typename TX> void rms_fwd_any(const RmsFwd& a, bool al, hipStream_t s) {
    constexpr int V = sizeof(TX) == 4 ? 4 : 8;
    if (a.cols < 8) hipLaunchKernelGGL((rms_fwd_long_kernel<TX, ROWS_TINY>), dim3((unsigned)a.rows), dim3(256), 0, s, a);
    else if (a.cols > RMS_LONG) hipLaunchKernelGGL((rms_fwd_long_kernel<TX, ROWS_ANY>), dim3((unsigned)a.rows), dim3(256), 0, s, a);
    else if (al) rms_fwd_launch<TX, V, ROWS_ALIGNED>(a, s);
    else rms_fwd_launch<TX, V, ROWS_ANY>(a, s);
}
template <typename TDY, typename TX, typename TD> void rms_bwd_types(const RmsBwd& a, bool al, hipStream_t s) {
    constexpr int V = sizeof(TDY) == 4 ? 4 : 8;
    if (al) rms_bwd_launch<TDY, TX, TD, V, ROWS_ALIGNED>(a, s);
    else rms_bwd_launch<TDY, TX, TD, V, ROWS_ANY>(a, s);
}
// dy, x and dx of one 16-bit type or fp32, with dy fp32 only beside fp32: what training steps have.  Wider rows, rows under 8
// columns and other mixtures take the kernels that walk.
template <typename TDY> constexpr int dtype_of() { return sizeof(TDY) == 4 ? BF_F32 : __is_same(TDY, bf16_t) ? BF_BF16 : BF_F16; }
bool rms_bwd_walks(int dy_dtype, int x_dtype, bool kept, int dx_dtype, int cols) {
    const bool x_ok = kept || x_dtype == BF_F32 || x_dtype == dy_dtype, d_ok = dx_dtype == BF_F32 || dx_dtype == dy_dtype;
    return cols < 8 || cols > RMS_LONG || !x_ok || !d_ok;
}
template <typename TDY> void rms_bwd_any(const RmsBwd& a, bool al, hipStream_t s) {
    constexpr int dt = dtype_of<TDY>();
    if (rms_bwd_walks(dt, a.x_dtype, a.q != nullptr, a.dx_dtype, a.cols)) {
        hipLaunchKernelGGL((rms_dgamma_long_kernel<TDY>), dim3((unsigned)((a.cols + 255) / 256), (unsigned)a.nblk), dim3(256), 0, s, a);
        const dim3 grid((unsigned)(a.rows < RMS_SLICE ? a.rows : RMS_SLICE));
        if (a.cols < 8) hipLaunchKernelGGL((rms_bwd_long_kernel<TDY, ROWS_TINY>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((rms_bwd_long_kernel<TDY, ROWS_ANY>), grid, dim3(256), 0, s, a);
    } else if (a.dx_dtype == dt) {
        if (a.q) rms_bwd_types<TDY, Kept, TDY>(a, al, s);
        else if (a.x_dtype == dt) rms_bwd_types<TDY, TDY, TDY>(a, al, s);
        else rms_bwd_types<TDY, float, TDY>(a, al, s);
    } else {
        if (a.q) rms_bwd_types<TDY, Kept, float>(a, al, s);
        else if (a.x_dtype == dt) rms_bwd_types<TDY, TDY, float>(a, al, s);
        else rms_bwd_types<TDY, float, float>(a, al, s);
    }
}

// may rows of this tensor be read in whole aligned vectors of V elements?
bool rows_aligned(const void* p, int64_t ld, size_t esz, int V) {
    const size_t vec = esz * V < 16 ? esz * V : 16;
    return p == nullptr || ((uintptr_t)p % vec == 0 && ((size_t)ld * esz) % vec == 0);
}
bool any_float(int dt) { return dt == BF_F32 || bf_is_half(dt); }

int rms_fwd(const char* name, RmsFwd& a, int x_dtype, bf_stream_t stream) {
    BF_REQUIRE(any_float(x_dtype), BF_EINVAL, "%s: bad x_dtype %d", name, x_dtype);
    BF_REQUIRE(!a.delta || any_float(a.d_dtype), BF_EINVAL, "%s: bad delta_dtype %d", name, a.d_dtype);
    BF_REQUIRE(a.rows >= 0 && a.rows <= RMS_MOST && a.cols > 0 && a.cols <= RMS_MOST, BF_EINVAL, "%s: bad shape (rows=%d cols=%d)",
               name, a.rows, a.cols);
    BF_REQUIRE(a.ldx >= a.cols && (!a.delta || a.ldd >= a.cols) && (!a.x_out || a.ldo >= a.cols), BF_EINVAL,
               "%s: a leading dimension is under cols=%d", name, a.cols);
    BF_REQUIRE((a.q == nullptr) == (a.code == nullptr), BF_EINVAL, "%s: a checkpoint is q and code, or neither", name);
    BF_REQUIRE(a.eps >= 0.f, BF_EINVAL, "%s: eps must not be negative", name);
    if (a.rows == 0) return BF_OK;
    BF_REQUIRE(a.x && a.gamma && a.y && (a.y_dtype != Y_E4M3 || a.y_scale), BF_EINVAL, "%s: null pointer", name);
    const size_t xs = bf_dtype_size(x_dtype), ds = bf_dtype_size(a.d_dtype), ys = a.y_dtype == Y_E4M3 ? 1 : bf_dtype_size(a.y_dtype);
    BF_REQUIRE((uintptr_t)a.x % xs == 0 && (uintptr_t)a.x_out % xs == 0 && (uintptr_t)a.delta % ds == 0 && (uintptr_t)a.y % ys == 0 &&
               (uintptr_t)a.gamma % 4 == 0 && (uintptr_t)a.rstd % 4 == 0 && (uintptr_t)a.y_scale % 4 == 0, BF_EALIGN,
               "%s: a tensor is not aligned to its element", name);
    a.gpr = (a.cols + ACT8_GROUP - 1) / ACT8_GROUP;
    const int V = x_dtype == BF_F32 ? 4 : 8;
    const bool al = a.cols % V == 0 && rows_aligned(a.x, a.ldx, xs, V) && rows_aligned(a.delta, a.ldd, ds, V) &&
                    rows_aligned(a.x_out, a.ldo, xs, V) && rows_aligned(a.y, a.cols, ys, V) && rows_aligned(a.q, a.cols, 1, V) &&
                    rows_aligned(a.gamma, a.cols, 4, V);
    // a grid counts threads in 32 bits: very many rows are taken in slices
    hipStream_t s = (hipStream_t)stream;
    const int rows = a.rows;
    for (int r0 = 0; r0 < rows; r0 += RMS_SLICE) {
        RmsFwd b = a;
        b.rows = rows - r0 < RMS_SLICE ? rows - r0 : RMS_SLICE;
        b.x = (const char*)a.x + (size_t)r0 * a.ldx * xs;
        if (a.delta) b.delta = (const char*)a.delta + (size_t)r0 * a.ldd * ds;
        if (a.x_out) b.x_out = (char*)a.x_out + (size_t)r0 * a.ldo * xs;
        b.y = (char*)a.y + (size_t)r0 * a.cols * ys;
        if (a.y_scale) b.y_scale = a.y_scale + r0;
        if (a.rstd) b.rstd = a.rstd + r0;
        if (a.q) {
            b.q = a.q + (size_t)r0 * a.cols;
            b.code = a.code + (size_t)r0 * a.gpr;
        }
        if (x_dtype == BF_F32) rms_fwd_any<float>(b, al, s);
        else if (x_dtype == BF_BF16) rms_fwd_any<bf16_t>(b, al, s);
        else rms_fwd_any<f16_t>(b, al, s);
        BF_CHECK_LAUNCH(name);
    }
    return BF_OK;
}

}  // namespace

extern "C" int bf_rmsnorm_fwd(const void* x, int64_t ldx, int x_dtype, const void* delta, int64_t ld_delta, int delta_dtype,
                              const float* gamma, void* x_out, int64_t ld_out, void* y, int y_dtype, float* rstd, void* q,
                              void* code, int rows, int cols, float eps, bf_stream_t stream) {
    BF_REQUIRE(any_float(y_dtype), BF_EINVAL, "bf_rmsnorm_fwd: bad y_dtype %d", y_dtype);
    RmsFwd a = {x, ldx, delta, ld_delta, delta_dtype, gamma, x_out, ld_out, y, y_dtype, nullptr, rstd, (uint8_t*)q,
                (uint8_t*)code, rows, cols, 0, eps};
    return rms_fwd("bf_rmsnorm_fwd", a, x_dtype, stream);
}

extern "C" int bf_rmsnorm_fwd_fp8(const void* x, int64_t ldx, int x_dtype, const void* delta, int64_t ld_delta, int delta_dtype,
                                  const float* gamma, void* x_out, int64_t ld_out, void* y_fp8, float* row_scale, float* rstd,
                                  void* q, void* code, int rows, int cols, float eps, bf_stream_t stream) {
    RmsFwd a = {x, ldx, delta, ld_delta, delta_dtype, gamma, x_out, ld_out, y_fp8, Y_E4M3, row_scale, rstd, (uint8_t*)q,
                (uint8_t*)code, rows, cols, 0, eps};
    return rms_fwd("bf_rmsnorm_fwd_fp8", a, x_dtype, stream);
}

extern "C" int bf_rmsnorm_bwd_parts(int rows, int cols) {
    if (rows <= 0 || cols <= 0) return 0;
    if (cols > RMS_LONG) return rows < 64 ? rows : 64;
    // As many workgroups as stay resident side by side: their registers grow with the row.  From the checkpoint with dres,
    // operands just written: 36 928 x 1 024 fp32 85 us with 768, 106 with 1 024, 95 with 512 (fp16 51, 52, 51); 50 432 x 768
    // fp16 51 with 768, 55 with 1 024; 60 000 x 512 fp16 45 and 43; 30 000 x 1 536 fp16 67 with 1 280, 72 with 1 024, 79 with
    // 768; 9 000 x 4 096 fp32 86 with 768, 106 with 1 024, 101 with 512 (fp16 49, 53, 51); 4 096 x 8 192 fp32 98 with 512, 110
    // with 768.
    if (cols <= 1024) {                          // a wave per row
        const int most = cols <= 512 ? 1024 : 768, want = rows / 4 + (rows % 4 != 0);
        return want < most ? want : most;
    }
    const int most = cols <= 2048 ? 1280 : cols <= 4096 ? 768 : cols <= 8192 ? 512 : 256;
    return rows < most ? rows : most;
}

extern "C" int bf_rmsnorm_bwd(const void* dy, int64_t ld_dy, int dy_dtype, const void* x, int64_t ldx, int x_dtype, const void* q,
                              const void* code, const float* gamma, const float* rstd, const void* dres, int64_t ld_dres,
                              void* dx, int dx_dtype, float* dgamma, float* parts_ws, int rows, int cols, bf_stream_t stream) {
    const char* name = "bf_rmsnorm_bwd";
    BF_REQUIRE(any_float(dy_dtype) && any_float(dx_dtype), BF_EINVAL, "%s: bad dy_dtype %d or dx_dtype %d", name, dy_dtype, dx_dtype);
    BF_REQUIRE(rows >= 0 && rows <= RMS_MOST && cols > 0 && cols <= RMS_MOST, BF_EINVAL, "%s: bad shape (rows=%d cols=%d)", name,
               rows, cols);
    BF_REQUIRE((q == nullptr) == (code == nullptr), BF_EINVAL, "%s: a checkpoint is q and code, or neither", name);
    BF_REQUIRE(dgamma && (uintptr_t)dgamma % 4 == 0, BF_EINVAL, "%s: null dgamma", name);
    hipStream_t s = (hipStream_t)stream;
    if (rows == 0) {
        hipError_t e = bf_zero_f32_async(dgamma, (size_t)cols, s);
        BF_REQUIRE(e == hipSuccess, BF_ELAUNCH, "%s: launch failed", name);
        return BF_OK;
    }
    BF_REQUIRE((x == nullptr) != (q == nullptr), BF_EINVAL, "%s: the stream is x, or a checkpoint q / code: exactly one", name);
    BF_REQUIRE(!x || any_float(x_dtype), BF_EINVAL, "%s: bad x_dtype %d", name, x_dtype);
    BF_REQUIRE(dy && gamma && rstd && dx && parts_ws, BF_EINVAL, "%s: null pointer", name);
    BF_REQUIRE(ld_dy >= cols && (!x || ldx >= cols) && (!dres || ld_dres >= cols), BF_EINVAL,
               "%s: a leading dimension is under cols=%d", name, cols);
    BF_REQUIRE(dx != dy || (ld_dy == cols && dx_dtype == dy_dtype), BF_EINVAL, "%s: dx may be dy only where their rows coincide", name);
    BF_REQUIRE(dx != dres || ld_dres == cols, BF_EINVAL, "%s: dx may be dres only where their rows coincide", name);
    const size_t ys = bf_dtype_size(dy_dtype), xs = bf_dtype_size(x_dtype), os = bf_dtype_size(dx_dtype);
    BF_REQUIRE((uintptr_t)dy % ys == 0 && (!x || (uintptr_t)x % xs == 0) && (uintptr_t)dres % os == 0 && (uintptr_t)dx % os == 0 &&
               (uintptr_t)gamma % 4 == 0 && (uintptr_t)rstd % 4 == 0 && (uintptr_t)parts_ws % 4 == 0, BF_EALIGN,
               "%s: a tensor is not aligned to its element", name);
    RmsBwd a = {dy, ld_dy, x, ldx, x_dtype, (const uint8_t*)q, (const uint8_t*)code, gamma, rstd, dres, ld_dres, dx, dx_dtype,
                parts_ws, rows, cols, (cols + ACT8_GROUP - 1) / ACT8_GROUP, bf_rmsnorm_bwd_parts(rows, cols)};
    const int V = dy_dtype == BF_F32 ? 4 : 8;
    const bool al = cols % V == 0 && rows_aligned(dy, ld_dy, ys, V) && (!x || rows_aligned(x, ldx, xs, V)) &&
                    rows_aligned(q, cols, 1, V) && rows_aligned(dres, ld_dres, os, V) && rows_aligned(dx, cols, os, V) &&
                    rows_aligned(gamma, cols, 4, V) && rows_aligned(parts_ws, cols, 4, V);
    if (a.nblk == 1) a.part = dgamma;           // one row of partial sums is the result
    if (dy_dtype == BF_F32) rms_bwd_any<float>(a, al && rows_aligned(a.part, cols, 4, V), s);
    else if (dy_dtype == BF_BF16) rms_bwd_any<bf16_t>(a, al && rows_aligned(a.part, cols, 4, V), s);
    else rms_bwd_any<f16_t>(a, al && rows_aligned(a.part, cols, 4, V), s);
    BF_CHECK_LAUNCH(name);
    if (a.nblk > 1) {
        hipLaunchKernelGGL(rms_dgamma_kernel, dim3((unsigned)((cols + 31) / 32)), dim3(1024), 0, s, parts_ws, dgamma, a.nblk, cols);
        BF_CHECK_LAUNCH(name);
    }
    return BF_OK;
}
