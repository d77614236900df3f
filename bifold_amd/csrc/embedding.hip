// Embedding lookup with scaling, and its gradient by sorted tokens.
//   bf_embed_scaled_fwd   out[i, :] = scale * table[id_i, :]
//   bf_embed_scaled_bwd   grad[v, :] (+)= scale * sum over { i : id_i = v } of dy[i, :]
// The gradient is a sum over rows that share a token.  Rows are brought together by a stable radix sort of (id, i), summed in
// runs of equal ids in the order of i, each in fp32; nothing is added with atomics, so the result is the same on every call.
// HBM bounds both for real batches (dy read once, the table's gradient written once).  The sort marks the tokens that occur in a
// table of bytes, and the launch that sums the runs also writes the zeros of a dense gradient's other rows: its gathers wait for
// latency, the zeros for bandwidth.
#include "act8.h"

namespace {

// ------------------------------------------------------------------ lookup
template <typename TT, int A, int U>
__global__ __launch_bounds__(256) void embed_scaled_kernel(const int32_t* __restrict__ ids, const TT* __restrict__ table,
                                                           void* __restrict__ out, int out_dtype, float scale, unsigned nvec,
                                                           unsigned vpr, int cols, int vocab, int* __restrict__ err_flag) {
    constexpr int V = sizeof(TT) == 4 ? 4 : 8;
    // two dependent loads: all ids first, then all rows, no branch between (which would wait for each)
    unsigned row[U], c[U];
    int id[U];
    Chunk<TT, V, A> x[U];
    const unsigned v0 = blockIdx.x * (256u * U) + threadIdx.x;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned v = min(v0 + u * 256u, nvec - 1);
        row[u] = v / vpr;
        c[u] = (v - row[u] * vpr) * V;
        id[u] = ids[row[u]];
    }
    bool bad = false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const bool out_of = id[u] < 0 || id[u] >= vocab;
        bad |= out_of;
        x[u].load(table, (size_t)(out_of ? 0 : id[u]) * cols + c[u], cols - (int)c[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (v0 + u * 256u >= nvec) break;
        float f[V];
        const int n = cols - (int)c[u];
        x[u].take(f, n);
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] *= scale;
        const size_t off = (size_t)row[u] * cols + c[u];
        if (out_dtype == BF_F32) vec_store_n<float, V, A>((float*)out + off, n, f);
        else if (out_dtype == BF_BF16) vec_store_n<bf16_t, V, A>((bf16_t*)out + off, n, f);
        else vec_store_n<f16_t, V, A>((f16_t*)out + off, n, f);
    }
    if (bad && err_flag) atomicExch(err_flag, 1);
}

// ------------------------------------------------------------------ the sort: least significant digit first, stable
// A pass is two launches: counts of each digit per tile, then every tile finds its places -- for each digit the tokens of
// smaller digits, of earlier tiles and of earlier waves -- and moves its tokens.  (Counting the next pass's digits by global
// atomics while moving saves a launch and costs more: 131 072 tokens 74 instead of 59 us.)  Digits of up to 9 bits put a
// vocabulary of 2^18 into two passes.  Ids outside the table and the padding token become the key `vocab`, which sorts
// behind the others.  131 072 tokens take 28 us in four short dependent launches, bound by their latencies; few tokens need
// no count launch (embed_scatter_kernel): 8 192 take 11.6 us, with them 14.6.
#define SORT_THREADS 512
#define SORT_WAVES 8
#define SORT_MAX_BINS 512
#define SORT_MAX_TILES 64
#define SORT_SELF 12288                         /* tokens; a digit's counts are kept in 16 bits */

struct SortArgs {
    const int32_t* ids; int n; int vocab; int pad;
    const int2* in; int2* out;                  // (key, token's place)
    int* hist; int* owner_count; int* err_flag;
    uint8_t* present;                           // [v]: token v occurs; NULL where nobody asks
    int rounds, tiles, dbits, shift;
};
template <bool FIRST>
__device__ __forceinline__ int2 sort_item(const SortArgs& a, int i, int* err_flag) {
    if constexpr (FIRST) {
        const int id = a.ids[i];
        if (id < 0 || id >= a.vocab) {
            if (err_flag) atomicExch(err_flag, 1);
            return make_int2(a.vocab, i);
        }
        return make_int2(id == a.pad ? a.vocab : id, i);
    } else {
        return a.in[i];
    }
}
__device__ __forceinline__ void sort_clear(const SortArgs& a) {
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.owner_count = 0;
    if (a.present) {
        unsigned* words = (unsigned*)a.present;
        const int many = (int)(((unsigned)a.vocab + 3u) >> 2);
        for (int i = blockIdx.x * SORT_THREADS + threadIdx.x; i < many; i += a.tiles * SORT_THREADS) words[i] = 0;
    }
}
template <bool FIRST>
__global__ __launch_bounds__(SORT_THREADS) void embed_hist_kernel(const SortArgs a) {
    __shared__ int bins[SORT_MAX_BINS];
    if (FIRST) sort_clear(a);
    bins[threadIdx.x] = 0;
    __syncthreads();
    const int base = blockIdx.x * SORT_THREADS * a.rounds, mask = (1 << a.dbits) - 1;
    for (int r = 0; r < a.rounds; ++r) {
        const int i = base + r * SORT_THREADS + threadIdx.x;
        if (i < a.n) atomicAdd(&bins[(sort_item<FIRST>(a, i, a.err_flag).x >> a.shift) & mask], 1);
    }
    __syncthreads();
    a.hist[blockIdx.x * SORT_MAX_BINS + threadIdx.x] = bins[threadIdx.x];
}
// SELF: no count launch, every workgroup counts all tokens itself.  The whole gradient of n tokens x 64 fp16, added, with and
// without: 2 049 21 and 25 us, 4 096 22 and 25, 8 192 26 and 28, 12 288 28 and 30, 16 384 36 and 36, so up to 12 288 tokens.
template <bool FIRST, bool SELF>
__global__ __launch_bounds__(SORT_THREADS) void embed_scatter_kernel(const SortArgs a) {
    __shared__ int cnt[SORT_WAVES][SORT_MAX_BINS];
    __shared__ int wave_tot[SORT_WAVES];
    // lanes of one digit wait for each other at its counter, and padding makes one token frequent: copies on different banks
    // (8 192 times one token: 25 us with 8, 29 with 2, 35 with one)
    constexpr int COPIES = 8, SKEW = 4;
    __shared__ unsigned all[SELF ? COPIES * (SORT_MAX_BINS + SKEW) : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int mask = (1 << a.dbits) - 1, span = SORT_THREADS * a.rounds;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) cnt[w][tid] = 0;
    if constexpr (SELF) {
#pragma unroll
        for (int k = 0; k < COPIES; ++k) all[k * (SORT_MAX_BINS + SKEW) + tid] = 0;
        if (FIRST) sort_clear(a);
    }
    __syncthreads();
    // a wave owns `rounds` x 64 consecutive tokens of the tile
    const int first = blockIdx.x * span + wave * 64 * a.rounds + lane;
#pragma unroll 4
    for (int r = 0; r < a.rounds; ++r) {
        const int i = first + r * 64;
        if (i < a.n) atomicAdd(&cnt[wave][(sort_item<FIRST>(a, i, nullptr).x >> a.shift) & mask], 1);
    }
    // all tokens of this thread's digit, and those in earlier tiles: sixteen tiles' counts in flight
    int tot = 0, before = 0;
    if constexpr (SELF) {                       // a digit's tokens in the low half of a word, those in earlier tiles in the high
        const int start = blockIdx.x * span;
        unsigned* const copy = all + (lane & (COPIES - 1)) * (SORT_MAX_BINS + SKEW);
        for (int i0 = tid; i0 < a.n; i0 += 8 * SORT_THREADS) {
            int key[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) key[u] = sort_item<FIRST>(a, min(i0 + u * SORT_THREADS, a.n - 1), nullptr).x;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int i = i0 + u * SORT_THREADS;
                if (i < a.n) atomicAdd(&copy[(key[u] >> a.shift) & mask], i < start ? 0x10001u : 1u);
            }
        }
        __syncthreads();
        unsigned both = 0;
#pragma unroll
        for (int k = 0; k < COPIES; ++k) both += all[k * (SORT_MAX_BINS + SKEW) + tid];
        tot = (int)(both & 0xFFFFu);
        before = (int)(both >> 16);
    }
    for (int t0 = 0; !SELF && t0 < a.tiles; t0 += 16) {
        int h[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) h[u] = a.hist[min(t0 + u, a.tiles - 1) * SORT_MAX_BINS + tid];
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            tot += t0 + u < a.tiles ? h[u] : 0;
            before += t0 + u < (int)blockIdx.x ? h[u] : 0;
        }
    }
    int scan = tot;                             // inclusive over the digits
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(scan, o, 64);
        if (lane >= o) scan += up;
    }
    if (lane == 63) wave_tot[wave] = scan;
    __syncthreads();
    for (int w = 0; w < wave; ++w) scan += wave_tot[w];
    int place = scan - tot + before;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) {
        const int c = cnt[w][tid];
        cnt[w][tid] = place;
        place += c;
    }
    __syncthreads();
    // cnt[wave][d] is where this wave's next token of digit d goes.  Within 64 tokens the lanes of one digit find each other
    // by a ballot per digit bit; the first of them moves the place on.  LDS accesses of one wave complete in order; the
    // relaxed atomics keep the compiler from holding a place in a register.
    int* mine = cnt[wave];
    int* const flag = SELF ? a.err_flag : nullptr;
    int2 item = first < a.n ? sort_item<FIRST>(a, first, flag) : make_int2(0, 0);
    for (int r = 0; r < a.rounds; ++r) {
        const int i = first + r * 64;
        const bool live = i < a.n;
        const int2 it = item;
        if (r + 1 < a.rounds && i + 64 < a.n) item = sort_item<FIRST>(a, i + 64, flag);
        const int d = (it.x >> a.shift) & mask;
        unsigned long long same = __ballot(live);
        for (int b = 0; b < a.dbits; ++b) {
            const bool bit = (d >> b) & 1;
            const unsigned long long votes = __ballot(bit);
            same &= bit ? votes : ~votes;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1ull));
        if (live) {
            const int at = __hip_atomic_load(&mine[d], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
            a.out[at + rank] = it;
            if (rank == 0) __hip_atomic_store(&mine[d], at + __popcll(same), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
            // whoever stores it, it is the same byte; a launch after the one that cleared the table
            if (FIRST != SELF && a.present && it.x < a.vocab) a.present[it.x] = 1;
        }
    }
}

// Up to 2 048 tokens of a vocabulary under 2^18: the same sort by one workgroup, in LDS, one launch (the whole gradient of
// 2 048 x 64 fp16, added into one that is there: 19 us instead of 22, of 1 024 17.5 instead of 20.5; 8 192 x 1 024 fp32 37,
// by four launches 33: one CU is not enough there).  A token is one word, its key over its place (11 bits; a larger vocabulary would fit, but one workgroup
// also clears its table of bytes); a thread holds R of them, a wave R x 64 consecutive ones.  Places behind the last token
// hold the largest word, which stays behind.
#define ONE_THREADS 1024
#define ONE_WAVES 16
#define ONE_BITS 11
#define ONE_MAX (1 << ONE_BITS)
#define ONE_BINS 256
template <int R>
__global__ __launch_bounds__(ONE_THREADS) void embed_sort_one_kernel(const SortArgs a, int passes) {
    __shared__ unsigned buf[ONE_THREADS * R];
    __shared__ int cnt[ONE_WAVES][ONE_BINS];
    __shared__ int wave_tot[ONE_BINS / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int first = wave * 64 * R + lane, mask = (1 << a.dbits) - 1;
    if (tid == 0) *a.owner_count = 0;
    if (a.present) {
        unsigned* words = (unsigned*)a.present;
        const int many = (int)(((unsigned)a.vocab + 3u) >> 2);
        for (int i = tid; i < many; i += ONE_THREADS) words[i] = 0;
    }
    unsigned item[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = first + r * 64;
        item[r] = i < a.n ? (unsigned)sort_item<true>(a, i, a.err_flag).x << ONE_BITS | (unsigned)i : 0xFFFFFFFFu;
    }
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = ONE_BITS + pass * a.dbits;
#pragma unroll
        for (int k = 0; k < ONE_WAVES * ONE_BINS / ONE_THREADS; ++k) (&cnt[0][0])[k * ONE_THREADS + tid] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; ++r) atomicAdd(&cnt[wave][(item[r] >> shift) & mask], 1);
        __syncthreads();
        int tot = 0, scan = 0;
        if (tid < ONE_BINS) {
#pragma unroll
            for (int w = 0; w < ONE_WAVES; ++w) tot += cnt[w][tid];
            scan = tot;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int up = __shfl_up(scan, o, 64);
                if (lane >= o) scan += up;
            }
            if (lane == 63) wave_tot[wave] = scan;
        }
        __syncthreads();
        if (tid < ONE_BINS) {
            for (int w = 0; w < wave; ++w) scan += wave_tot[w];
            int place = scan - tot;
#pragma unroll
            for (int w = 0; w < ONE_WAVES; ++w) {
                const int c = cnt[w][tid];
                cnt[w][tid] = place;
                place += c;
            }
        }
        __syncthreads();
        int* mine = cnt[wave];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int d = (item[r] >> shift) & mask;
            unsigned long long same = ~0ull;
            for (int b = 0; b < a.dbits; ++b) {
                const bool bit = (d >> b) & 1;
                const unsigned long long votes = __ballot(bit);
                same &= bit ? votes : ~votes;
            }
            const int rank = __popcll(same & ((1ull << lane) - 1ull));
            const int at = __hip_atomic_load(&mine[d], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
            buf[at + rank] = item[r];
            if (rank == 0) __hip_atomic_store(&mine[d], at + __popcll(same), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; ++r) item[r] = buf[first + r * 64];
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = first + r * 64, key = (int)(item[r] >> ONE_BITS);
        if (i < a.n) {
            a.out[i] = make_int2(key, (int)(item[r] & (ONE_MAX - 1)));
            if (a.present && key < a.vocab) a.present[key] = 1;
        }
    }
}

// ------------------------------------------------------------------ sums over runs of equal keys
struct SumArgs {
    const int2* sorted; int n; int vocab; int chunk, chunks, slabs;        // (key, row of dy), by key, then row
    const void* dy; int64_t ld; int cols; float scale; int accumulate;
    float* grad; float* part; int2* owners; int* owner_count;              // owners: (chunk, key) of each cut run
    const uint8_t* present; unsigned sum_blocks;                 // present: NULL, or the other rows' zeros are written too
};
template <int V, int A>
__device__ __forceinline__ void grad_write(const SumArgs& a, int key, int c, const float (&acc)[V]) {
    float* g = a.grad + (size_t)key * a.cols + c;
    float o[V];
    if (a.accumulate) vec_load_n<float, V, A>(g, a.cols - c, o);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = a.accumulate ? o[j] + acc[j] * a.scale : acc[j] * a.scale;
    vec_store_n<float, V, A>(g, a.cols - c, o);
}
// One wave takes `chunk` (at most 64) consecutive sorted tokens and 64 V columns, eight rows in flight.  A run of equal keys
// belongs to the chunk it begins in, which follows it into the next chunk.  Only a run that covers a whole further chunk is
// cut: its sum over the chunk it begins in goes to part[chunk][1] (that chunk owns the run and notes it for
// embed_join_kernel), its sums over the chunks it reaches into go to part[.][0].
// The wave's number is taken as a scalar, so what follows from it (addresses, branches) is scalar; all loads of a batch have
// arrived before its sums begin: with a wait per row, stores of finished runs between them were waited for too.
// 131 072 x 1 024 bf16, vocabulary 65 536, 61 000 rows alive: 80 us for some 400 MB, 5.0 TB/s; 8 192 x 768 fp16, 32 000:
// 19 us for 111 MB, 5.8 TB/s.  ONCE: dy past the caches (the whole gradient of the first, dy behind other writes:
// 149 us, with ordinary loads 175; dy just written: 138 either way).
template <typename T, int V, int A, bool ONCE>
__global__ __launch_bounds__(256) void embed_sum_kernel(const SumArgs a) {
    const int lane = threadIdx.x & 63;
    if (blockIdx.x >= a.sum_blocks) {           // a wave per eight rows of the table
        const size_t group = (size_t)(blockIdx.x - a.sum_blocks) * 4 + wave_id(), row0 = group * 8;
        if (row0 >= (size_t)a.vocab) return;
        const int rows = (int)min((size_t)8, a.vocab - row0);
        const unsigned long long there = __ballot(lane >= rows || a.present[row0 + (lane & 7)] != 0);
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
        for (int r = 0; r < rows; ++r) {
            if ((there >> r) & 1) continue;
            float* g = a.grad + (row0 + r) * a.cols;
            for (int c = lane * 4; c < a.cols; c += 256) vec_store_n<float, 4, A>(g + c, a.cols - c, zero);
        }
        return;
    }
    const unsigned w = blockIdx.x * 4u + (unsigned)wave_id();
    const int chunk = (int)(w / (unsigned)a.slabs), slab = (int)(w - (unsigned)chunk * (unsigned)a.slabs);
    if (chunk >= a.chunks) return;
    const int s = chunk * a.chunk, here = min(a.chunk, a.n - s);
    const int there = max(0, min(a.chunk, a.n - s - a.chunk));            // tokens of the next chunk
    const int2 mine = lane < here ? a.sorted[s + lane] : make_int2(a.vocab, 0);
    const int2 ahead = lane < there ? a.sorted[s + a.chunk + lane] : make_int2(-1, 0);
    const int kl = mine.x, il = mine.y, kn = ahead.x, in = ahead.y;
    // uniform addresses: scalar loads
    const int prev = s > 0 ? a.sorted[s - 1].x : -1, prev2 = s > a.chunk ? a.sorted[s - a.chunk - 1].x : -1;
    const int next2 = s + 2 * a.chunk < a.n ? a.sorted[s + 2 * a.chunk].x : -1;
    const int live = __popcll(__ballot(lane < here && kl < a.vocab));      // sorted: the live ones come first
    if (live == 0) return;
    const int c = (slab * 64 + lane) * V, nc = a.cols - c;
    float* part = a.part + (size_t)chunk * 2 * a.cols + c;
    const int k_first = __builtin_amdgcn_readlane(kl, 0), k_last = __builtin_amdgcn_readlane(kl, live - 1);
    const int next = there > 0 ? __builtin_amdgcn_readfirstlane(kn) : -1;
    // the run this chunk begins inside of: the chunk before has it if it began there and ends here
    bool head = k_first == prev;
    int i = 0;
    if (head && prev2 != k_first && next != k_first) {
        i = __popcll(__ballot(lane < here && kl == k_first));
        head = false;
    }
    // the run this chunk ends inside of: followed to its end if that lies in the next chunk
    const bool open = live == here && next == k_last, cut = open && next2 == k_last;
    const bool whole = head && k_first == k_last;                          // began before and fills the chunk
    int stop = live;
    if (open && !cut && !whole) stop += __popcll(__ballot(lane < there && kn == k_last));
    float acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.f;
    while (i < stop) {
        Chunk<T, V, A> f[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int at = min(i + u, stop - 1);
            const int row = at < here ? __builtin_amdgcn_readlane(il, at) : __builtin_amdgcn_readlane(in, at - here);
            f[u].template load<ONCE>(a.dy, (size_t)row * a.ld + c, nc);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) f[u].arrived();
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (i + u < stop) {
                const int at = i + u;
                float v[V];
                f[u].take(v, nc);
#pragma unroll
                for (int j = 0; j < V; ++j) acc[j] += v[j];
                const int key = at < here ? __builtin_amdgcn_readlane(kl, at) : k_last;
                // the key behind this token; a cut run ends with the chunk
                const int after = at + 1 == stop ? -1 : at + 1 < here ? __builtin_amdgcn_readlane(kl, at + 1) : k_last;
                if (after != key) {
                    if (head) {
                        vec_store_n<float, V, A>(part, nc, acc);
                    } else if (cut && at + 1 == stop) {
                        vec_store_n<float, V, A>(part + a.cols, nc, acc);
                        if (slab == 0 && lane == 0) a.owners[atomicAdd(a.owner_count, 1)] = make_int2(chunk, key);
                    } else {
                        grad_write<V, A>(a, key, c, acc);
                    }
                    head = false;
#pragma unroll
                    for (int j = 0; j < V; ++j) acc[j] = 0.f;
                }
            }
        }
        i += 8;
    }
}
// One workgroup per cut run (their order in the list does not matter: each has a gradient row of its own) and 256 columns:
// finds the last chunk that starts with the run's key, sums the partial rows in order, sixteen waves a share each.
template <int A>
__global__ __launch_bounds__(1024) void embed_join_kernel(const SumArgs a) {
    __shared__ float4 red[16][64];
    __shared__ int found[16];
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int slabs = (a.cols + 255) / 256;
    const int total = *a.owner_count * slabs;
    for (int wk = blockIdx.x; wk < total; wk += gridDim.x) {
        const int2 owner = a.owners[wk / slabs];
        const int chunk = owner.x, key = owner.y, c = (wk % slabs) * 256 + lane * 4, nc = a.cols - c;
        int lo = chunk + 1, hi = a.chunks;      // chunk lo starts with the key; hi does not (or is behind the last)
        while (hi - lo > 1) {                   // 1 024 places at a time
            const int step = (hi - lo + 1023) >> 10, at = lo + ((int)threadIdx.x + 1) * step;
            const bool in = at < hi && a.sorted[(size_t)at * a.chunk].x == key;
            const int votes = __popcll(__ballot(in));
            if (lane == 0) found[wave] = votes;
            __syncthreads();
            int sum = 0;
#pragma unroll
            for (int k = 0; k < 16; ++k) sum += found[k];
            lo += step * sum;
            hi = min(hi, lo + step);
            __syncthreads();
        }
        const int many = lo - chunk + 1, share = (many + 15) >> 4;          // partial rows: part[chunk][1], part[chunk + 1 ..][0]
        const int from = wave * share, to = min(many, from + share);
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int t = from; t < to; t += 8) {
            Chunk<float, 4, A> f[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int at = min(t + u, to - 1);
                f[u].load(a.part, ((size_t)(chunk + at) * 2 + (at == 0)) * a.cols + c, nc);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                float v[4];
                f[u].take(v, nc);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] += t + u < to ? v[j] : 0.f;
            }
        }
        red[wave][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int k = 1; k < 16; ++k) {
                const float4 f = red[k][lane];
                acc[0] += f.x; acc[1] += f.y; acc[2] += f.z; acc[3] += f.w;
            }
            grad_write<4, A>(a, key, c, acc);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------ few tokens: one launch, no sort
// A workgroup per token: the first token of its id gathers the others' places in order and sums their rows, each wave 64 V
// columns and a share of the rows.  Behind them, workgroups that write zeros into `zero_rows` rows each of a dense gradient,
// where none of the tokens is.
// Up to 512 tokens (x 1 024 fp32 columns, added into a gradient): 7 us with few repeats, 17 with half of them one token, 29
// with all; the sort's launches take 22 from there on.  One workgroup draws some 80 GB/s, which is why not more.
#define FEW 512
template <typename T, int V, int A>
__global__ __launch_bounds__(FEW) void embed_few_kernel(const int32_t* __restrict__ ids, int pad, int* __restrict__ err_flag,
                                                                int zero_rows, const SumArgs a) {
    constexpr int WAVES = FEW / 64;
    __shared__ unsigned long long words[WAVES];
    __shared__ unsigned short list[FEW];
    __shared__ float red[WAVES][64 * V];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), me = blockIdx.x;
    if (me >= a.n) {
        const size_t row0 = (size_t)(me - a.n) * zero_rows;
        const int rows = (int)min((size_t)zero_rows, a.vocab - row0);
        list[tid] = 0;
        __syncthreads();
        if (tid < a.n) {
            const int id = ids[tid];
            const unsigned at = (unsigned)id - (unsigned)row0;
            if (id >= 0 && id != pad && at < (unsigned)rows) list[at] = 1;
        }
        __syncthreads();
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
        for (int r = wave; r < rows; r += WAVES) {
            if (list[r]) continue;
            float* g = a.grad + (row0 + r) * a.cols;
            for (int c = lane * 4; c < a.cols; c += 256) vec_store_n<float, 4, A>(g + c, a.cols - c, zero);
        }
        return;
    }
    const int key = ids[me];
    if (key < 0 || key >= a.vocab) {
        if (tid == 0 && err_flag) atomicExch(err_flag, 1);
        return;
    }
    if (key == pad) return;
    const bool same = tid < a.n && ids[tid] == key;
    const unsigned long long votes = __ballot(same);
    if (lane == 0) words[wave] = votes;
    __syncthreads();
    int many = 0;
    bool earlier = false;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const unsigned long long v = words[w];
        const int below = me - w * 64;          // tokens of this word in front of this one
        earlier |= below >= 64 ? v != 0 : below > 0 ? (v & ((1ull << below) - 1ull)) != 0 : false;
        if (w == wave && same) list[many + __popcll(v & ((1ull << lane) - 1ull))] = (unsigned short)tid;
        many += __popcll(v);
    }
    if (earlier) return;                        // uniform: the first token of this id does the work
    __syncthreads();
    const int shares = a.slabs >= WAVES ? 1 : WAVES / a.slabs;
    for (int slab0 = 0; slab0 < a.slabs; slab0 += WAVES) {
        const int at = wave / shares, slab = slab0 + at, sh = wave - at * shares;
        const bool in = slab < a.slabs && at < WAVES / shares;
        const int per = (many + shares - 1) / shares, from = sh * per, to = in ? min(many, from + per) : 0;
        const int c = (slab * 64 + lane) * V, nc = a.cols - c;
        float acc[V];
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = 0.f;
        for (int t = from; t < to; t += 8) {
            Chunk<T, V, A> f[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) f[u].load(a.dy, (size_t)list[min(t + u, to - 1)] * a.ld + c, nc);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                float v[V];
                f[u].take(v, nc);
#pragma unroll
                for (int j = 0; j < V; ++j) acc[j] += t + u < to ? v[j] : 0.f;
            }
        }
        if (shares > 1) {
#pragma unroll
            for (int j = 0; j < V; ++j) red[wave][j * 64 + lane] = acc[j];
            __syncthreads();
            if (sh == 0 && in) {
                for (int k = 1; k < shares; ++k)
#pragma unroll
                    for (int j = 0; j < V; ++j) acc[j] += red[wave + k][j * 64 + lane];
            }
            __syncthreads();
        }
        if (sh == 0 && in) grad_write<V, A>(a, key, c, acc);
    }
}

// ------------------------------------------------------------------ plan of a call
struct EmbedPlan {
    bool one, self;                             // sorted by one workgroup; without count launches
    int passes, dbits, rounds, tiles, chunk, chunks;
    size_t pairs, hist, owners, present, part, bytes;            // offsets into the workspace
};
EmbedPlan embed_plan(int n, int cols, int vocab) {
    EmbedPlan p;
    int bits = 0;
    while (bits < 31 && (vocab >> bits) != 0) ++bits;            // the key `vocab` itself is used
    p.one = n <= ONE_MAX && vocab < (1 << 18);
    p.passes = p.one ? (bits + 7) / 8 : (bits + 8) / 9;          // digits of up to 8 or 9 bits
    p.dbits = (bits + p.passes - 1) / p.passes;
    p.self = !p.one && p.passes > 1 && n <= SORT_SELF;           // the first pass clears the table of bytes, later ones mark
    const long span = (long)SORT_THREADS * SORT_MAX_TILES;
    p.rounds = (int)((n + span - 1) / span);
    p.tiles = (n + SORT_THREADS * p.rounds - 1) / (SORT_THREADS * p.rounds);
    // tokens per wave: enough waves for the chip first, then few partial rows (131 072 tokens x 1 024: sum + join 108.9 us with
    // 64, 102.6 with 32; 8 192 x 768: 25.2 us with 16, 26.8 with 8)
    p.chunk = n >= 16384 ? 32 : 16;
    p.chunks = (n + p.chunk - 1) / p.chunk;
    auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
    p.pairs = 0;
    p.hist = up((size_t)n * 16);
    p.owners = p.hist + up((size_t)p.tiles * SORT_MAX_BINS * 4);
    p.present = p.owners + up((size_t)(p.chunks + 1) * 8);
    p.part = p.present + up((size_t)vocab + 8);
    p.bytes = p.part + up((size_t)p.chunks * 2 * cols * 4);
    return p;
}

template <typename T, int V, int A>
void embed_sum_launch(SumArgs a, hipStream_t s) {
    a.sum_blocks = (unsigned)(((size_t)a.chunks * a.slabs + 3) / 4);
    const unsigned zeros = a.present ? (unsigned)(((size_t)a.vocab + 31) / 32) : 0u;
    const dim3 grid(a.sum_blocks + zeros);
    // a dy larger than the L2 caches is read past them (12 MB read again and again: 22 us so, 19 through the caches)
    if (A == ROWS_ALIGNED && (size_t)a.n * a.cols * sizeof(T) >= (size_t)32 << 20)
        hipLaunchKernelGGL((embed_sum_kernel<T, V, A, A == ROWS_ALIGNED>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((embed_sum_kernel<T, V, A, false>), grid, dim3(256), 0, s, a);
}
template <typename T, int V>
void embed_bwd_type(bool few, int mode, const int32_t* ids, int pad, int* err_flag, const SumArgs& a, hipStream_t s) {
    if (few) {
        // some 64 KB a workgroup
        const int zero_rows = a.cols >= 16384 ? 1 : 16384 / a.cols < FEW ? 16384 / a.cols : FEW;
        const dim3 grid((unsigned)a.n + (a.accumulate ? 0u : (unsigned)(((size_t)a.vocab + zero_rows - 1) / zero_rows)));
        if (mode == ROWS_ALIGNED)
            hipLaunchKernelGGL((embed_few_kernel<T, V, ROWS_ALIGNED>), grid, dim3(FEW), 0, s, ids, pad, err_flag, zero_rows, a);
        else if (mode == ROWS_ANY)
            hipLaunchKernelGGL((embed_few_kernel<T, V, ROWS_ANY>), grid, dim3(FEW), 0, s, ids, pad, err_flag, zero_rows, a);
        else
            hipLaunchKernelGGL((embed_few_kernel<T, V, ROWS_TINY>), grid, dim3(FEW), 0, s, ids, pad, err_flag, zero_rows, a);
    } else if (mode == ROWS_ALIGNED) {
        embed_sum_launch<T, V, ROWS_ALIGNED>(a, s);
    } else if (mode == ROWS_ANY) {
        embed_sum_launch<T, V, ROWS_ANY>(a, s);
    } else {
        embed_sum_launch<T, V, ROWS_TINY>(a, s);
    }
}
int rows_mode(bool al, int cols) { return al ? ROWS_ALIGNED : cols >= 8 ? ROWS_ANY : ROWS_TINY; }
bool float_type(int dt) { return dt == BF_F32 || bf_is_half(dt); }

}  // namespace

extern "C" int bf_embed_scaled_fwd(const int32_t* tokens, const void* table, int table_dtype, void* out, int out_dtype, float scale,
                                   int n, int cols, int vocab, int* err_flag, bf_stream_t stream) {
    const char* name = "bf_embed_scaled_fwd";
    BF_REQUIRE(float_type(table_dtype) && float_type(out_dtype), BF_EINVAL, "%s: bad table_dtype %d or out_dtype %d", name,
               table_dtype, out_dtype);
    BF_REQUIRE(n >= 0 && cols > 0 && cols <= (1 << 30) && vocab > 0, BF_EINVAL, "%s: bad shape (n=%d cols=%d vocab=%d)", name, n, cols, vocab);
    if (n == 0) return BF_OK;
    BF_REQUIRE(tokens && table && out, BF_EINVAL, "%s: null pointer", name);
    const size_t ts = bf_dtype_size(table_dtype), os = bf_dtype_size(out_dtype);
    BF_REQUIRE((uintptr_t)tokens % 4 == 0 && (uintptr_t)table % ts == 0 && (uintptr_t)out % os == 0, BF_EALIGN,
               "%s: a tensor is not aligned to its element", name);
    const int V = table_dtype == BF_F32 ? 4 : 8;
    const unsigned vpr = (unsigned)((cols + V - 1) / V);
    const unsigned long long nvec = (unsigned long long)n * vpr;
    BF_REQUIRE(nvec <= 0x7FFFF000ull, BF_EINVAL, "%s: n=%d x cols=%d is too large", name, n, cols);
    const int mode = rows_mode(cols % V == 0 && bf_aligned16(table) && bf_aligned16(out), cols);
    hipStream_t s = (hipStream_t)stream;
    // vectors a lane: many for a long batch (131 072 x 1 024 bf16: 75.9 us with four, 91.8 with one), one where the launch's
    // latency counts (8 192 x 768: 5.9 us, with four 6.3; 77 x 512: 3.0 and 3.8)
    const int U = nvec >= (1u << 21) && mode != ROWS_TINY ? 4 : 1;
    const dim3 grid((unsigned)((nvec + 256 * U - 1) / (256 * U))), block(256);
#define EMBED_FWD2(T, A, N)                                                                                                      \
    hipLaunchKernelGGL((embed_scaled_kernel<T, A, N>), grid, block, 0, s, tokens, (const T*)table, out, out_dtype, scale,        \
                       (unsigned)nvec, vpr, cols, vocab, err_flag)
#define EMBED_FWD(T)                                                                                                             \
    do {                                                                                                                         \
        if (mode == ROWS_ALIGNED) { if (U == 4) EMBED_FWD2(T, ROWS_ALIGNED, 4); else EMBED_FWD2(T, ROWS_ALIGNED, 1); }           \
        else if (mode == ROWS_ANY) { if (U == 4) EMBED_FWD2(T, ROWS_ANY, 4); else EMBED_FWD2(T, ROWS_ANY, 1); }                  \
        else EMBED_FWD2(T, ROWS_TINY, 1);                                                                                        \
    } while (0)
    if (table_dtype == BF_F32) EMBED_FWD(float);
    else if (table_dtype == BF_BF16) EMBED_FWD(bf16_t);
    else EMBED_FWD(f16_t);
#undef EMBED_FWD
#undef EMBED_FWD2
    BF_CHECK_LAUNCH(name);
    return BF_OK;
}

extern "C" size_t bf_embed_scaled_bwd_workspace_bytes(int n, int cols, int vocab) {
    if (n <= FEW || cols <= 0 || vocab <= 0) return 0;
    return embed_plan(n, cols, vocab).bytes;
}

extern "C" int bf_embed_scaled_bwd(const void* dy, int64_t ld_dy, int dy_dtype, const int32_t* tokens, float* grad, float scale,
                                   int accumulate, int padding_idx, int n, int cols, int vocab, int* err_flag, void* workspace,
                                   size_t workspace_bytes, bf_stream_t stream) {
    const char* name = "bf_embed_scaled_bwd";
    BF_REQUIRE(float_type(dy_dtype), BF_EINVAL, "%s: bad dy_dtype %d", name, dy_dtype);
    BF_REQUIRE(n >= 0 && cols > 0 && cols <= (1 << 30) && vocab > 0 && vocab < 0x7FFFFFFF, BF_EINVAL, "%s: bad shape (n=%d cols=%d vocab=%d)", name, n,
               cols, vocab);
    BF_REQUIRE(n <= (1 << 30), BF_EINVAL, "%s: over 2^30 tokens (n=%d)", name, n);
    BF_REQUIRE(grad && (uintptr_t)grad % 4 == 0, BF_EALIGN, "%s: grad is null or not aligned to its element", name);
    hipStream_t s = (hipStream_t)stream;
    if (n == 0) {
        if (!accumulate) {
            const hipError_t e = bf_zero_f32_async(grad, (size_t)vocab * cols, s);
            BF_REQUIRE(e == hipSuccess, BF_ELAUNCH, "%s: launch failed", name);
        }
        return BF_OK;
    }
    BF_REQUIRE(dy && tokens, BF_EINVAL, "%s: null pointer", name);
    BF_REQUIRE(ld_dy >= cols, BF_EINVAL, "%s: ld_dy=%lld is under cols=%d", name, (long long)ld_dy, cols);
    const size_t esz = bf_dtype_size(dy_dtype);
    BF_REQUIRE((uintptr_t)dy % esz == 0 && (uintptr_t)tokens % 4 == 0, BF_EALIGN, "%s: a tensor is not aligned to its element", name);
    const int V = dy_dtype == BF_F32 ? 4 : 8;
    const int mode = rows_mode(cols % V == 0 && bf_aligned16(dy) && ((size_t)ld_dy * esz) % 16 == 0 && bf_aligned16(grad), cols);
    SumArgs a = {};
    a.n = n; a.vocab = vocab; a.dy = dy; a.ld = ld_dy; a.cols = cols; a.scale = scale; a.accumulate = accumulate; a.grad = grad;
    a.slabs = (cols + 64 * V - 1) / (64 * V);
    const bool few = n <= FEW;
    // a grid counts threads in 32 bits: 2^24 workgroups of 256
    BF_REQUIRE((unsigned long long)(n / 16 + 1) * a.slabs / 4 + (unsigned)vocab / 32 < (1u << 24) - 2, BF_EINVAL,
               "%s: n=%d x cols=%d, vocab=%d is too large", name, n, cols, vocab);
    if (!few) {
        const EmbedPlan p = embed_plan(n, cols, vocab);
        BF_REQUIRE(workspace && workspace_bytes >= p.bytes, BF_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed", name,
                   workspace_bytes, p.bytes);
        BF_REQUIRE(bf_aligned16(workspace), BF_EALIGN, "%s: unaligned workspace", name);
        char* ws = (char*)workspace;
        int2* const pairs[2] = {(int2*)(ws + p.pairs), (int2*)(ws + p.pairs) + n};
        int2* owners = (int2*)(ws + p.owners);
        SortArgs q = {};
        q.ids = tokens; q.n = n; q.vocab = vocab; q.pad = padding_idx; q.hist = (int*)(ws + p.hist);
        q.owner_count = (int*)(owners + p.chunks); q.err_flag = err_flag; q.rounds = p.rounds; q.tiles = p.tiles; q.dbits = p.dbits;
        q.present = accumulate ? nullptr : (uint8_t*)(ws + p.present);
        if (p.one) {
            q.out = pairs[0];
            const dim3 block(ONE_THREADS);
            if (n <= 1024) hipLaunchKernelGGL(embed_sort_one_kernel<1>, dim3(1), block, 0, s, q, p.passes);
            else hipLaunchKernelGGL(embed_sort_one_kernel<2>, dim3(1), block, 0, s, q, p.passes);
            BF_CHECK_LAUNCH(name);
        }
        const dim3 grid((unsigned)p.tiles), block(SORT_THREADS);
        for (int pass = 0; pass < p.passes && !p.one; ++pass) {
            q.shift = pass * p.dbits;
            q.in = pairs[(pass + 1) & 1];
            q.out = pairs[pass & 1];
            if (p.self) {
                if (pass == 0) hipLaunchKernelGGL((embed_scatter_kernel<true, true>), grid, block, 0, s, q);
                else hipLaunchKernelGGL((embed_scatter_kernel<false, true>), grid, block, 0, s, q);
            } else if (pass == 0) {
                hipLaunchKernelGGL((embed_hist_kernel<true>), grid, block, 0, s, q);
                hipLaunchKernelGGL((embed_scatter_kernel<true, false>), grid, block, 0, s, q);
            } else {
                hipLaunchKernelGGL((embed_hist_kernel<false>), grid, block, 0, s, q);
                hipLaunchKernelGGL((embed_scatter_kernel<false, false>), grid, block, 0, s, q);
            }
            BF_CHECK_LAUNCH(name);
        }
        a.present = q.present;
        a.sorted = q.out; a.chunk = p.chunk; a.chunks = p.chunks; a.owners = owners; a.owner_count = q.owner_count;
        a.part = (float*)(ws + p.part);
    }
    if (dy_dtype == BF_F32) embed_bwd_type<float, 4>(few, mode, tokens, padding_idx, err_flag, a, s);
    else if (dy_dtype == BF_BF16) embed_bwd_type<bf16_t, 8>(few, mode, tokens, padding_idx, err_flag, a, s);
    else embed_bwd_type<f16_t, 8>(few, mode, tokens, padding_idx, err_flag, a, s);
    BF_CHECK_LAUNCH(name);
    if (!few) {
        const size_t most = (size_t)a.chunks * ((cols + 255) / 256);
        const dim3 grid((unsigned)(most < 512 ? most : 512)), block(1024);
        if (mode == ROWS_ALIGNED) hipLaunchKernelGGL(embed_join_kernel<ROWS_ALIGNED>, grid, block, 0, s, a);
        else if (mode == ROWS_ANY) hipLaunchKernelGGL(embed_join_kernel<ROWS_ANY>, grid, block, 0, s, a);
        else hipLaunchKernelGGL(embed_join_kernel<ROWS_TINY>, grid, block, 0, s, a);
        BF_CHECK_LAUNCH(name);
    }
    return BF_OK;
}
