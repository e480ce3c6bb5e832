// Rows of a table picked by index, scaled, plus a bias, and the gradient of that:
//   y[t][f]      = table[index[t]][f] * w_gain + bias[f] * b_gain
//   dtable[v][f] = w_gain * sum over the tokens t with index[t] == v of dy[t][f]      dbias[f] = b_gain * sum over t of dy[t][f]
// Every operand is moved once; all of it is bound by HBM (few tokens: by launches).  The forward pass is a gather.  The table's
// gradient sums, in float32 and in the order of the tokens, the rows of dy that share an index; no atomics, so that the same
// inputs give the same bits:
//   * few tokens (plan_grad): one launch.  A workgroup owns 64 classes x 64 features of the table, each wave a quarter of
//     the classes; it lists the tokens that fall on its classes, sums them and writes the tile, zeros included.
//   * beyond: the tokens are sorted by index (stable radix sort, 8 bits a pass; one launch while one workgroup can hold
//     them, two launches a pass otherwise: 4096 tokens of 1000 x 512 24.6 us the first way, 28.7 the second) and a wave
//     walks a fixed number of sorted positions with the running sum in registers.  A run of equal indices inside one wave's
//     positions is written straight to its row.  A run that crosses into other waves' positions leaves one partial sum per
//     wave, and a second kernel adds those in order: the most frequent index costs no more than any other.  Rows without
//     tokens are zeroed by the sort's first launch.
// An index outside [0, v) reads as a row of NaN and adds to no row of the table's gradient (the bias's sums every token).
// 65536 tokens of 32000 x 1024 in bfloat16, natural frequencies: lookup 40 us (268 MB moved, repeated rows from the caches), gradient
// 84: sort and clearing 27, sums 46 (200 MB, 4.3 TB/s), runs that cross spans 8; a bias 6 more.  64 labels of 1000 x 512 in float32: 3.7
// and 4.9 us.  A transposed table is read and, beyond few tokens, written a row apart by neighbouring lanes: 4096 tokens of 4096 x 2048
// in bfloat16 35 us for the lookup (7 the other way), 93 with the gradient (51).
#include "sg_common.h"
#include "sg_column_sums.h"

namespace sg {
namespace {

constexpr int kOwnerTokens = 256;
constexpr int kBlockSortTokens = 4096;
constexpr int kSortBlocks = 128;         // bounds the table of digit counts that every block of a pass reads

struct IndexView {
    const void* p;
    int is64;
    __device__ __forceinline__ int64_t at(int64_t i) const { return is64 ? ((const int64_t*)p)[i] : (int64_t)((const int*)p)[i]; }
};

// ---- forward --------------------------------------------------------------------------------------------------------

struct EmbedParams {
    IndexView index;
    const void* table;
    const void* bias;
    void* y;
    int64_t tokens, v, f, stride_v, stride_f;
    float w_gain, b_gain;
};

constexpr int kFwdUnroll = 4;

// PACKED: rows of whole aligned 16-byte packets (a lane moves packets); otherwise a lane moves single elements.  kFwdUnroll
// independent rows per lane: their index and table loads overlap.
template <class T, bool PACKED>
__global__ void __launch_bounds__(256) embedding_kernel(const EmbedParams p) {
    constexpr int N = PACKED ? Pack<T>::N : 1;
    const int64_t per_row = p.f / N, total = p.tokens * per_row;
    const int64_t stride = (int64_t)gridDim.x * 256;
    const T* __restrict__ table = (const T*)p.table;
    const T* __restrict__ bias = (const T*)p.bias;
    T* __restrict__ y = (T*)p.y;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += stride * kFwdUnroll) {
        int64_t row[kFwdUnroll], col[kFwdUnroll];
#pragma unroll
        for (int u = 0; u < kFwdUnroll; u++) {
            const int64_t k = i + u * stride < total ? i + u * stride : i;
            // (32-bit division where the count allows: a 64-bit one is a long sequence)
            const int64_t t = total <= UINT32_MAX ? (int64_t)((uint32_t)k / (uint32_t)per_row) : k / per_row;
            row[u] = p.index.at(t);
            col[u] = (k - t * per_row) * N;
        }
        T v[kFwdUnroll][N];
#pragma unroll
        for (int u = 0; u < kFwdUnroll; u++) {
            const bool ok = (uint64_t)row[u] < (uint64_t)p.v;
            const T* src = table + (ok ? row[u] : 0) * p.stride_v + col[u] * p.stride_f;
            if constexpr (PACKED) {
                const Pack<T> q = load_pack(src);
#pragma unroll
                for (int j = 0; j < N; j++) v[u][j] = q.v[j];
            } else {
                v[u][0] = *src;
            }
        }
#pragma unroll
        for (int u = 0; u < kFwdUnroll; u++) {
            if (i + u * stride >= total) break;
            const bool ok = (uint64_t)row[u] < (uint64_t)p.v;
            Pack<T> out;
#pragma unroll
            for (int j = 0; j < N; j++) {
                float r = __fmul_rn(Elem<T>::load(v[u][j]), p.w_gain);
                if (bias) r = __fadd_rn(r, __fmul_rn(Elem<T>::load(bias[col[u] + j]), p.b_gain));
                out.v[j] = Elem<T>::store(ok ? r : NAN);
            }
            const int64_t at = (i + u * stride) * N;
            if constexpr (PACKED) store_pack(y + at, out);
            else y[at] = out.v[0];
        }
    }
}

// ---- gradient, few tokens ---------------------------------------------------------------------------------------------

struct GradParams {
    IndexView index;
    const void* dy;                      // [tokens][f]
    void* dtable;
    void* dbias;                         // or NULL
    int64_t tokens, v, f, stride_v, stride_f;
    float w_gain, b_gain;
    int f_inner;                         // dtable is written along f (stride_f == 1) rather than along v
};

constexpr int kOwnTile = 64, kOwnBatch = 16;

// Tiles [v / 64][f / 64], then f / 64 more workgroups for the bias gradient.
template <class T>
__global__ void __launch_bounds__(256) embedding_grad_owner_kernel(const GradParams p, int tiles_v, int tiles_f) {
    __shared__ float acc[kOwnTile][kOwnTile + 1];
    __shared__ unsigned list[4][kOwnerTokens];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T* __restrict__ dy = (const T*)p.dy;
    const int tokens = (int)p.tokens;
    const int block = blockIdx.x;
    if (block >= tiles_v * tiles_f) {                 // bias: the waves take every fourth run of kOwnBatch tokens, added in wave order
        const int64_t f = (int64_t)(block - tiles_v * tiles_f) * kOwnTile + lane;
        float sum = 0;
        for (int t0 = wave * kOwnBatch; t0 < tokens; t0 += 4 * kOwnBatch) {
            float g[kOwnBatch];
#pragma unroll
            for (int u = 0; u < kOwnBatch; u++) g[u] = (t0 + u < tokens && f < p.f) ? Elem<T>::load(dy[(int64_t)(t0 + u) * p.f + f]) : 0.f;
#pragma unroll
            for (int u = 0; u < kOwnBatch; u++) sum += g[u];
        }
        acc[wave][lane] = sum;
        __syncthreads();
        if (wave == 0 && f < p.f)
            ((T*)p.dbias)[f] = Elem<T>::store(((acc[0][lane] + acc[1][lane]) + (acc[2][lane] + acc[3][lane])) * p.b_gain);
        return;
    }
    const int64_t v0 = (int64_t)(block / tiles_f) * kOwnTile, f0 = (int64_t)(block % tiles_f) * kOwnTile;
    // the wave's own classes: v0 + 4 * i + wave
    for (int i = 0; i < kOwnTile / 4; i++) acc[4 * i + wave][lane] = 0.f;
    int count = 0;
    for (int t0 = 0; t0 < tokens; t0 += 64) {
        const int t = t0 + lane;
        const int64_t v = t < tokens ? p.index.at(t) - v0 : -1;
        const bool mine = v >= 0 && v < kOwnTile && v0 + v < p.v && (v & 3) == wave;
        const uint64_t mask = __ballot(mine);
        if (mine) list[wave][count + __popcll(mask & ((1ull << lane) - 1))] = (unsigned)t << 8 | (unsigned)v;
        count += __popcll(mask);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const bool inside = f0 + lane < p.f;
    for (int e0 = 0; e0 < count; e0 += kOwnBatch) {
        unsigned e[kOwnBatch];
        float g[kOwnBatch];
#pragma unroll
        for (int u = 0; u < kOwnBatch; u++) e[u] = list[wave][e0 + u < count ? e0 + u : e0];
#pragma unroll
        for (int u = 0; u < kOwnBatch; u++) g[u] = inside ? Elem<T>::load(dy[(int64_t)(e[u] >> 8) * p.f + f0 + lane]) : 0.f;
#pragma unroll
        for (int u = 0; u < kOwnBatch; u++)
            if (e0 + u < count) acc[e[u] & 255][lane] += g[u];
    }
    T* __restrict__ dt = (T*)p.dtable;
    if (p.f_inner) {
        for (int i = 0; i < kOwnTile / 4; i++) {
            const int64_t v = v0 + 4 * i + wave;
            if (inside && v < p.v) dt[v * p.stride_v + (f0 + lane) * p.stride_f] = Elem<T>::store(acc[4 * i + wave][lane] * p.w_gain);
        }
    } else {                                          // classes along the lanes: a transposed table's rows are contiguous in v
        __syncthreads();
        for (int i = 0; i < kOwnTile / 4; i++) {
            const int fl = 4 * i + wave;
            if (f0 + fl < p.f && v0 + lane < p.v)
                dt[(v0 + lane) * p.stride_v + (f0 + fl) * p.stride_f] = Elem<T>::store(acc[lane][fl] * p.w_gain);
        }
    }
}

// ---- sorting tokens by index ----------------------------------------------------------------------------------------------

// Stable ranks of ITEMS x 64 digits of one wave among equal digits of the same wave: rank[i] for item i of this lane (items
// are ordered by i, then lane); count[d] ends as the wave's number of digit d (it starts as zero).
template <int ITEMS> __device__ __forceinline__ void wave_ranks(const unsigned (&digit)[ITEMS], const bool (&valid)[ITEMS], volatile int* count, int (&rank)[ITEMS]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        uint64_t same = __ballot(valid[i]);
#pragma unroll
        for (int b = 0; b < 8; b++) {
            const uint64_t set = __ballot((digit[i] >> b) & 1);
            same &= (digit[i] >> b) & 1 ? set : ~set;
        }
        // (one wave's LDS accesses are executed in program order; volatile keeps the compiler's order the same)
        const int before = count[digit[i]];
        __builtin_amdgcn_wave_barrier();
        const int below = __popcll(same & ((1ull << lane) - 1));
        rank[i] = before + below;
        if (valid[i] && below == 0) count[digit[i]] = before + __popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
}

__device__ __forceinline__ unsigned key_of(int64_t index, int64_t v) { return (uint64_t)index < (uint64_t)v ? (unsigned)index : (unsigned)v; }

// Exclusive prefix sum of 256 values, one per thread of the first four waves (every thread of the block calls it).
__device__ __forceinline__ int scan256(int x, int* scratch) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(s, d, 64);
        if (lane >= d) s += o;
    }
    if (wave < 4 && lane == 63) scratch[wave] = s;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < 4; w++) before += w < wave ? scratch[w] : 0;
    __syncthreads();
    return before + s - x;
}

__device__ void zero_fill(void* base, int64_t bytes, int block, int blocks, int threads) {
    const uint4 zero = make_uint4(0, 0, 0, 0);
    uint4* p = (uint4*)base;
    const int64_t packets = bytes / 16;
    for (int64_t i = (int64_t)block * threads + threadIdx.x; i < packets; i += (int64_t)blocks * threads) p[i] = zero;
    if (block == 0 && threadIdx.x < (unsigned)(bytes % 16) / 2) ((unsigned short*)base)[packets * 8 + threadIdx.x] = 0;
}

// Up to kBlockSortTokens tokens: block 0 sorts, the others clear the table's gradient.
__global__ void __launch_bounds__(1024) sort_block_kernel(IndexView index, int tokens, int64_t v, int passes, unsigned* keys, unsigned* perm,
                                                          void* zero, int64_t zero_bytes) {
    constexpr int ITEMS = kBlockSortTokens / 1024, WAVES = 16;
    if (blockIdx.x > 0) {
        zero_fill(zero, zero_bytes, blockIdx.x - 1, gridDim.x - 1, 1024);
        return;
    }
    __shared__ unsigned key[2][kBlockSortTokens], id[2][kBlockSortTokens];
    __shared__ int count[WAVES][256];
    __shared__ int scratch[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < tokens; i += 1024) {
        key[0][i] = key_of(index.at(i), v);
        id[0][i] = i;
    }
    int from = 0;
    for (int pass = 0; pass < passes; pass++) {
        for (int i = threadIdx.x; i < WAVES * 256; i += 1024) (&count[0][0])[i] = 0;
        __syncthreads();
        unsigned digit[ITEMS];
        bool valid[ITEMS];
        int rank[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            const int at = (wave * ITEMS + i) * 64 + lane;
            valid[i] = at < tokens;
            digit[i] = valid[i] ? (key[from][at] >> (8 * pass)) & 255 : 0;
        }
        wave_ranks<ITEMS>(digit, valid, count[wave], rank);
        __syncthreads();
        int sum = 0;
        if (threadIdx.x < 256)
            for (int w = 0; w < WAVES; w++) {
                const int c = count[w][threadIdx.x];
                count[w][threadIdx.x] = sum;
                sum += c;
            }
        const int base = scan256(threadIdx.x < 256 ? sum : 0, scratch);
        if (threadIdx.x < 256)
            for (int w = 0; w < WAVES; w++) count[w][threadIdx.x] += base;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ITEMS; i++)
            if (valid[i]) {
                const int at = (wave * ITEMS + i) * 64 + lane, to = count[wave][digit[i]] + rank[i];
                key[from ^ 1][to] = key[from][at];
                id[from ^ 1][to] = id[from][at];
            }
        __syncthreads();
        from ^= 1;
    }
    for (int i = threadIdx.x; i < tokens; i += 1024) {
        keys[i] = key[from][i];
        perm[i] = id[from][i];
    }
}

// One pass over many blocks, first half: digit counts of every block's share of the tokens.  In the first pass the blocks
// behind the sort's clear the table's gradient.
__global__ void __launch_bounds__(256) sort_count_kernel(IndexView index, const unsigned* __restrict__ keys, int64_t tokens, int64_t v, int shift,
                                                         int64_t share, int blocks, int* __restrict__ counts, void* zero, int64_t zero_bytes) {
    if ((int)blockIdx.x >= blocks) {
        zero_fill(zero, zero_bytes, blockIdx.x - blocks, gridDim.x - blocks, 256);
        return;
    }
    __shared__ int hist[256];
    hist[threadIdx.x] = 0;
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * share, last = first + share < tokens ? first + share : tokens;
    for (int64_t i = first + threadIdx.x; i < last; i += 256) {
        const unsigned key = keys ? keys[i] : key_of(index.at(i), v);
        atomicAdd(&hist[(key >> shift) & 255], 1);        // (whole numbers: the order of the additions does not matter)
    }
    __syncthreads();
    counts[blockIdx.x * 256 + threadIdx.x] = hist[threadIdx.x];
}

// Second half: every token to its place.  A place is (tokens of smaller digits) + (equal digits of earlier blocks, of earlier
// rounds and waves of this block, of earlier lanes).  Sixteen waves: the table of counts is read by four threads a digit.
__global__ void __launch_bounds__(1024) sort_place_kernel(IndexView index, const unsigned* __restrict__ keys, const unsigned* __restrict__ ids,
                                                          int64_t tokens, int64_t v, int shift, int64_t share, const int* __restrict__ counts,
                                                          unsigned* __restrict__ keys_out, unsigned* __restrict__ ids_out) {
    constexpr int WAVES = 16, ROUND = 1024;
    __shared__ int count[WAVES][256];
    __shared__ int scratch[4];
    const int wave = threadIdx.x >> 6, digit_of_thread = threadIdx.x & 255, quarter = threadIdx.x >> 8;
    const int blocks = gridDim.x;
    int earlier = 0, total = 0;
#pragma unroll 8
    for (int b = quarter; b < blocks; b += 4) {
        const int c = counts[b * 256 + digit_of_thread];
        earlier += b < (int)blockIdx.x ? c : 0;
        total += c;
    }
    count[quarter][digit_of_thread] = total;
    count[4 + quarter][digit_of_thread] = earlier;
    __syncthreads();
    if (threadIdx.x < 256) {
        total = count[0][threadIdx.x] + count[1][threadIdx.x] + count[2][threadIdx.x] + count[3][threadIdx.x];
        earlier = count[4][threadIdx.x] + count[5][threadIdx.x] + count[6][threadIdx.x] + count[7][threadIdx.x];
    }
    int next = scan256(threadIdx.x < 256 ? total : 0, scratch) + earlier;     // threads 0 .. 255: place of the block's next token with that digit
    const int64_t first = (int64_t)blockIdx.x * share, last = first + share < tokens ? first + share : tokens;
    for (int64_t at0 = first; at0 < last; at0 += ROUND) {
        for (int i = threadIdx.x; i < WAVES * 256; i += 1024) (&count[0][0])[i] = 0;
        __syncthreads();
        const int64_t at = at0 + threadIdx.x;
        const bool valid[1] = {at < last};
        const unsigned key = valid[0] ? (keys ? keys[at] : key_of(index.at(at), v)) : 0;
        const unsigned id = valid[0] ? (ids ? ids[at] : (unsigned)at) : 0;
        const unsigned digit[1] = {(key >> shift) & 255};
        int rank[1];
        wave_ranks<1>(digit, valid, count[wave], rank);
        __syncthreads();
        if (threadIdx.x < 256)
            for (int w = 0; w < WAVES; w++) {
                const int c = count[w][threadIdx.x];
                count[w][threadIdx.x] = next;
                next += c;
            }
        __syncthreads();
        if (valid[0]) {
            const int to = count[wave][digit[0]] + rank[0];
            keys_out[to] = key;
            ids_out[to] = id;
        }
        __syncthreads();
    }
}

// ---- sums over runs of equal indices --------------------------------------------------------------------------------------

struct RunParams {
    const unsigned* keys;
    const unsigned* perm;
    const void* dy;
    void* dtable;
    float* partial;                      // [spans][2][f]: slot 0 the run that began in an earlier span, slot 1 the one that goes on
    float* columns;                      // [spans][f] or NULL: sums over all of the span's tokens, for the bias
    int64_t tokens, v, f, stride_v, stride_f;
    float w_gain;
    int span;                            // sorted positions per wave, at most 64
    int spans, tiles;
};

constexpr int kRunBatch = 8;

// One wave per (span, feature tile of 64 x N).  N > 1: rows of whole aligned packets.
template <class T, int N>
__global__ void __launch_bounds__(256) embedding_grad_runs_kernel(const RunParams p) {
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= (int64_t)p.spans * p.tiles) return;
    const int span = (int)(item / p.tiles), tile = (int)(item % p.tiles);
    const int64_t p0 = (int64_t)span * p.span;
    const int here = (int)(p.tokens - p0 < p.span ? p.tokens - p0 : p.span);
    const int64_t f = ((int64_t)tile * 64 + lane) * N;
    const bool inside = f < p.f;
    const unsigned my_key = lane < here ? p.keys[p0 + lane] : 0xffffffffu;
    const unsigned my_id = lane < here ? p.perm[p0 + lane] : 0;
    const unsigned none = 0xffffffffu;
    const unsigned key_before = p0 > 0 ? p.keys[p0 - 1] : none;
    const unsigned key_after = p0 + here < p.tokens ? p.keys[p0 + here] : none;
    const T* __restrict__ dy = (const T*)p.dy;
    float acc[N], all[N];
#pragma unroll
    for (int j = 0; j < N; j++) acc[j] = all[j] = 0.f;
    unsigned key = __builtin_amdgcn_readfirstlane(my_key);
    bool from_before = key == key_before;
    auto flush = [&](bool goes_on) {
        if (inside && key < (unsigned)p.v) {
            if (from_before || goes_on) {
                float* out = p.partial + ((int64_t)span * 2 + (from_before ? 0 : 1)) * p.f + f;
#pragma unroll
                for (int j = 0; j < N; j++) out[j] = acc[j];
            } else {
                T* out = (T*)p.dtable + (int64_t)key * p.stride_v + f * p.stride_f;
                if constexpr (N > 1) {
                    Pack<T> q;
#pragma unroll
                    for (int j = 0; j < N; j++) q.v[j] = Elem<T>::store(acc[j] * p.w_gain);
                    store_pack(out, q);
                } else {
                    *out = Elem<T>::store(acc[0] * p.w_gain);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < N; j++) acc[j] = 0.f;
    };
    for (int t0 = 0; t0 < here; t0 += kRunBatch) {
        T g[kRunBatch][N];
#pragma unroll
        for (int u = 0; u < kRunBatch; u++) {
            const unsigned id = __builtin_amdgcn_readlane(my_id, t0 + u < here ? t0 + u : t0);
            const T* src = dy + (int64_t)id * p.f + (inside ? f : 0);
            if constexpr (N > 1) {
                const Pack<T> q = load_pack(src);
#pragma unroll
                for (int j = 0; j < N; j++) g[u][j] = q.v[j];
            } else {
                g[u][0] = *src;
            }
        }
#pragma unroll
        for (int u = 0; u < kRunBatch; u++) {
            if (t0 + u >= here) break;
            const unsigned k = __builtin_amdgcn_readlane(my_key, t0 + u);
            if (k != key) {
                flush(false);
                key = k;
                from_before = false;
            }
#pragma unroll
            for (int j = 0; j < N; j++) {
                acc[j] += Elem<T>::load(g[u][j]);
                all[j] += Elem<T>::load(g[u][j]);
            }
        }
    }
    flush(key == key_after);
    if (p.columns && inside)
#pragma unroll
        for (int j = 0; j < N; j++) p.columns[(int64_t)span * p.f + f + j] = all[j];
}

// Runs that cross spans: the workgroup of the span a run begins in adds the later spans' partial sums to its own.  A wave takes 64 * N
// features; where that leaves waves over, 2, 4 or 8 of them take consecutive shares of the spans, which are added in their order.
template <class T, int N>
__global__ void __launch_bounds__(512) embedding_grad_join_kernel(const RunParams p, const ColumnJoin columns) {
    constexpr int WAVES = 8;
    __shared__ float part[WAVES][64 * (N > 2 ? N : 2)];
    if ((int)blockIdx.x >= p.spans) {                                  // the workgroups behind the spans': the bias
        join_columns<T, WAVES>(columns, blockIdx.x - p.spans, &part[0][0]);
        return;
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int span = blockIdx.x;
    const int64_t p0 = (int64_t)span * p.span, end = p0 + p.span;
    if (end >= p.tokens) return;                                       // the last span: nothing goes on
    const unsigned key = p.keys[end - 1];
    if (key >= (unsigned)p.v || p.keys[end] != key) return;            // the run ends here
    if (p.keys[p0] == key && p0 > 0 && p.keys[p0 - 1] == key) return;  // it began earlier
    // the last span the run reaches: the largest j for which position (span + j) * p.span still holds the key (sorted, so
    // 64 probes at a time find it in three rounds up to 2^18 spans; most runs end within the first 64)
    int reach = 1;
    auto probe = [&](int step) {
        for (;;) {
            const int64_t at = (int64_t)(span + reach + (int64_t)step * (lane + 1)) * p.span;
            const uint64_t in = __ballot(at < p.tokens && p.keys[at < p.tokens ? at : 0] == key);
            const int more = in == ~0ull ? 64 : __ffsll((unsigned long long)~in) - 1;
            reach += step * more;
            if (more < 64) return more;
        }
    };
    const int64_t far = (int64_t)(span + reach + 64) * p.span;
    if (far < p.tokens && p.keys[far] == key) {
        probe(4096);
        probe(64);
    }
    probe(1);
    const int tiles = (int)((p.f + 64 * N - 1) / (64 * N));
    const int shares = tiles >= 8 ? 1 : tiles >= 4 ? 2 : tiles >= 2 ? 4 : 8;
    const int mine = wave % shares, each = (reach + shares - 1) / shares;
    const int a = mine * each, b = a + each < reach ? a + each : reach;
    for (int tile0 = 0; tile0 < tiles; tile0 += WAVES / shares) {       // (the same number of turns for every wave)
        const int64_t f = ((int64_t)(tile0 + wave / shares) * 64 + lane) * N;
        const bool inside = f < p.f;
        const float* src = p.partial + (int64_t)(span + 1) * 2 * p.f + (inside ? f : 0);
        const float* own = p.partial + ((int64_t)span * 2 + 1) * p.f + (inside ? f : 0);
        float sum[N];
#pragma unroll
        for (int j = 0; j < N; j++) sum[j] = mine == 0 ? own[j] : 0.f;
        for (int i = a; i < b; i += 4) {
            float g[4][N];
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int j = 0; j < N; j++) g[u][j] = src[(int64_t)(i + u < b ? i + u : a) * 2 * p.f + j];
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int j = 0; j < N; j++) sum[j] += i + u < b ? g[u][j] : 0.f;
        }
        if (shares > 1) {
#pragma unroll
            for (int j = 0; j < N; j++) part[wave][j * 64 + lane] = sum[j];
            __syncthreads();
            if (mine == 0)
                for (int w = 1; w < shares; w++)
#pragma unroll
                    for (int j = 0; j < N; j++) sum[j] += part[wave + w][j * 64 + lane];
            __syncthreads();
        }
        if (mine == 0 && inside) {
            T* out = (T*)p.dtable + (int64_t)key * p.stride_v + f * p.stride_f;
            if constexpr (N > 1) {
                Pack<T> q;
#pragma unroll
                for (int j = 0; j < N; j++) q.v[j] = Elem<T>::store(sum[j] * p.w_gain);
                store_pack(out, q);
            } else {
                *out = Elem<T>::store(sum[0] * p.w_gain);
            }
        }
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------

int check(const sg_embedding_params* p, const char* what) {
    SG_REQUIRE(p != nullptr, SG_ERR_NULL_POINTER, "params is NULL");
    SG_REQUIRE(p->dtype == SG_F32 || p->dtype == SG_F16 || p->dtype == SG_BF16, SG_ERR_UNSUPPORTED, "%s: dtype %d (float32, float16 or bfloat16)", what, p->dtype);
    SG_REQUIRE(p->tokens >= 0 && p->tokens <= INT32_MAX, SG_ERR_INVALID_ARGUMENT, "%s: %lld tokens", what, (long long)p->tokens);
    SG_REQUIRE(p->v >= 1 && p->v <= INT32_MAX && p->f >= 0 && p->f <= INT32_MAX, SG_ERR_INVALID_ARGUMENT, "%s: table of %lld x %lld", what, (long long)p->v, (long long)p->f);
    SG_REQUIRE(p->index_bytes == 4 || p->index_bytes == 8, SG_ERR_INVALID_ARGUMENT, "%s: indices of %d bytes", what, p->index_bytes);
    SG_REQUIRE(p->tokens == 0 || p->f == 0 || (p->index && p->table), SG_ERR_NULL_POINTER, "%s: index or table is NULL", what);
    SG_REQUIRE(p->stride_v >= 0 && p->stride_f >= 0, SG_ERR_INVALID_ARGUMENT, "%s: negative stride", what);
    return SG_OK;
}

struct GradPlan {
    int passes = 0, span = 0, spans = 0, sort_blocks = 0;
    int64_t share = 0;
    size_t keys = 0, counts = 0, partial = 0, sums = 0, total = 0;      // offsets into the workspace
    bool owner = false;
};

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

GradPlan plan_grad(const sg_embedding_params& p, int packet) {
    GradPlan g;
    // Owner or sort, us, float32: 64 tokens of 1000 x 512 4 / 17, 256 tokens 5 / 19.5 (all on ten classes 11 / 18, on one class 26 / 18), 512
    // tokens 7 / 19.5 (20 / 18, 50 / 19).  Every tile looks at every token: 64 of 60000 x 512 18 / 26, 256 of them 28 / 26, 256 of 20000 x
    // 1024 in bfloat16 33 / 21.
    g.owner = p.tokens <= kOwnerTokens && p.tokens * ((p.v + kOwnTile - 1) / kOwnTile) * ((p.f + kOwnTile - 1) / kOwnTile) <= 1 << 20;
    if (g.owner) return g;
    while (((uint64_t)p.v >> (8 * g.passes)) != 0) g.passes++;
    // sorted positions per wave: 64, halved (down to 16) while the launch would not reach eight waves on every CU
    const int64_t tiles = (p.f + 64 * packet - 1) / (64 * packet);
    g.span = 64;
    while (g.span > 16 && (p.tokens + g.span - 1) / g.span * tiles < 2048) g.span /= 2;
    g.spans = (int)((p.tokens + g.span - 1) / g.span);
    size_t at = 0;
    g.keys = at;
    at += up256((size_t)p.tokens * 4) * (p.tokens <= kBlockSortTokens ? 2 : 4);
    if (p.tokens > kBlockSortTokens) {
        g.share = (p.tokens + kSortBlocks - 1) / kSortBlocks;
        g.share = (g.share + 1023) / 1024 * 1024;
        g.sort_blocks = (int)((p.tokens + g.share - 1) / g.share);
        g.counts = at;
        at += up256((size_t)g.sort_blocks * 256 * 4);
    }
    g.partial = at;
    at += up256((size_t)g.spans * 2 * p.f * 4);
    g.sums = at;
    at += up256((size_t)g.spans * p.f * 4);
    g.total = at;
    return g;
}

bool packed_rows(const sg_embedding_params& p, const void* dy) {
    const int64_t n = p.dtype == SG_F32 ? 4 : 8;
    return p.stride_f == 1 && p.f % n == 0 && p.stride_v % n == 0 && aligned16(p.table) && aligned16(dy);
}

}  // namespace
}  // namespace sg

extern "C" int sg_embedding(const sg_embedding_params* p, void* y, sg_stream_t stream) {
    using namespace sg;
    const int rc = check(p, "embedding");
    if (rc != SG_OK) return rc;
    if (p->tokens == 0 || p->f == 0) return SG_OK;
    SG_REQUIRE(y != nullptr, SG_ERR_NULL_POINTER, "embedding: y is NULL");
    EmbedParams e{{p->index, p->index_bytes == 8}, p->table, p->bias, y, p->tokens, p->v, p->f, p->stride_v, p->stride_f, p->w_gain, p->b_gain};
    const bool packed = packed_rows(*p, y);
    const int64_t items = p->tokens * (packed ? p->f / (p->dtype == SG_F32 ? 4 : 8) : p->f);
    int64_t blocks = (items + 256 * kFwdUnroll - 1) / (256 * kFwdUnroll);
    if (items <= 256 * 256 * kFwdUnroll) blocks = (items + 255) / 256;                // few items: one per lane, on as many CUs as there are
    if (blocks > 1 << 20) blocks = 1 << 20;
    SG_DISPATCH_16_32(p->dtype, {
        if (packed) hipLaunchKernelGGL((embedding_kernel<T, true>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, e);
        else hipLaunchKernelGGL((embedding_kernel<T, false>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, e);
    });
    return check_launch("sg_embedding");
}

extern "C" size_t sg_embedding_backward_workspace_bytes(const sg_embedding_params* p) {
    using namespace sg;
    if (check(p, "embedding_backward") != SG_OK || p->tokens == 0 || p->f == 0) return 0;
    const size_t a = plan_grad(*p, 1).total, b = plan_grad(*p, p->dtype == SG_F32 ? 4 : 8).total;
    return a > b ? a : b;                                  // (whether rows are packed is known with dy)
}

extern "C" int sg_embedding_backward(const sg_embedding_params* p, const void* dy, void* dbias, void* workspace, size_t workspace_bytes,
                                     sg_stream_t stream_) {
    using namespace sg;
    const int rc = check(p, "embedding_backward");
    if (rc != SG_OK) return rc;
    if (p->f == 0) return SG_OK;
    hipStream_t stream = (hipStream_t)stream_;
    void* dtable = const_cast<void*>(p->table);
    SG_REQUIRE(dtable != nullptr, SG_ERR_NULL_POINTER, "embedding_backward: dtable is NULL");
    SG_REQUIRE(p->tokens == 0 || dy != nullptr, SG_ERR_NULL_POINTER, "embedding_backward: dy is NULL");
    // dense in either order: the launch that clears it writes v * f elements from its first one on
    const bool rows = p->stride_f == 1 && p->stride_v == p->f, cols = p->stride_v == 1 && p->stride_f == p->v;
    SG_REQUIRE(rows || cols, SG_ERR_INVALID_ARGUMENT, "embedding_backward: dtable must be dense");
    SG_REQUIRE(aligned16(dtable), SG_ERR_INVALID_ARGUMENT, "embedding_backward: dtable must be 16-byte aligned");
    const bool packed = packed_rows(*p, dy);
    const int packet = p->dtype == SG_F32 ? 4 : 8, n = packed ? packet : 1;
    const GradPlan g = plan_grad(*p, n);
    SG_REQUIRE(g.total == 0 || (workspace && workspace_bytes >= g.total && aligned16(workspace)), SG_ERR_INVALID_ARGUMENT,
               "embedding_backward: needs %zu bytes of aligned workspace", g.total);
    const IndexView index{p->index, p->index_bytes == 8};
    if (g.owner) {
        const int64_t tiles_v = (p->v + kOwnTile - 1) / kOwnTile, tiles_f = (p->f + kOwnTile - 1) / kOwnTile;
        SG_REQUIRE((tiles_v + 1) * tiles_f <= INT32_MAX, SG_ERR_INVALID_ARGUMENT, "embedding_backward: table too large");
        const GradParams q{index, dy, dtable, dbias, p->tokens, p->v, p->f, p->stride_v, p->stride_f, p->w_gain, p->b_gain, rows ? 1 : 0};
        SG_DISPATCH_16_32(p->dtype,
            hipLaunchKernelGGL((embedding_grad_owner_kernel<T>), dim3((unsigned)((tiles_v + (dbias ? 1 : 0)) * tiles_f)), dim3(256), 0, stream, q,
                               (int)tiles_v, (int)tiles_f));
        return check_launch("sg_embedding_backward");
    }
    char* ws = (char*)workspace;
    const int64_t zero_bytes = p->v * p->f * (p->dtype == SG_F32 ? 4 : 2);
    int64_t zero_blocks = (zero_bytes + 65535) / 65536;
    if (zero_blocks > 2048) zero_blocks = 2048;
    const size_t row = up256((size_t)p->tokens * 4);
    unsigned* a[2] = {(unsigned*)(ws + g.keys), (unsigned*)(ws + g.keys + row)};
    const unsigned *keys = a[0], *perm = a[1];
    if (p->tokens <= kBlockSortTokens) {
        hipLaunchKernelGGL(sort_block_kernel, dim3(1 + (unsigned)zero_blocks), dim3(1024), 0, stream, index, (int)p->tokens, p->v, g.passes, a[0], a[1],
                           dtable, zero_bytes);
        const int done = check_launch("sg_embedding_backward");
        if (done != SG_OK) return done;
    } else {
        unsigned* b[2] = {(unsigned*)(ws + g.keys + 2 * row), (unsigned*)(ws + g.keys + 3 * row)};
        int* counts = (int*)(ws + g.counts);
        const unsigned *k_in = nullptr, *i_in = nullptr;
        for (int pass = 0; pass < g.passes; pass++) {
            unsigned** out = pass & 1 ? b : a;
            hipLaunchKernelGGL(sort_count_kernel, dim3(g.sort_blocks + (pass == 0 ? (unsigned)zero_blocks : 0)), dim3(256), 0, stream, index, k_in,
                               p->tokens, p->v, 8 * pass, g.share, g.sort_blocks, counts, dtable, zero_bytes);
            hipLaunchKernelGGL(sort_place_kernel, dim3(g.sort_blocks), dim3(1024), 0, stream, index, k_in, i_in, p->tokens, p->v, 8 * pass, g.share,
                               counts, out[0], out[1]);
            const int done = check_launch("sg_embedding_backward");
            if (done != SG_OK) return done;
            k_in = out[0];
            i_in = out[1];
        }
        keys = k_in;
        perm = i_in;
    }
    const int tiles = (int)((p->f + 64 * n - 1) / (64 * n));
    const RunParams r{keys, perm, dy, dtable, (float*)(ws + g.partial), dbias ? (float*)(ws + g.sums) : nullptr,
                      p->tokens, p->v, p->f, p->stride_v, p->stride_f, p->w_gain, g.span, g.spans, tiles};
    const int64_t items = (int64_t)g.spans * tiles;
    const ColumnJoin columns{r.columns, dbias, p->f, g.spans, p->b_gain};
    const unsigned joins = (unsigned)(g.spans + (dbias ? (p->f + 63) / 64 : 0));
    SG_REQUIRE((items + 3) / 4 <= INT32_MAX, SG_ERR_INVALID_ARGUMENT, "embedding_backward: too many elements");
    SG_DISPATCH_16_32(p->dtype, {
        if (packed) {
            hipLaunchKernelGGL((embedding_grad_runs_kernel<T, Pack<T>::N>), dim3((unsigned)((items + 3) / 4)), dim3(256), 0, stream, r);
            hipLaunchKernelGGL((embedding_grad_join_kernel<T, Pack<T>::N>), dim3(joins), dim3(512), 0, stream, r, columns);
        } else {
            hipLaunchKernelGGL((embedding_grad_runs_kernel<T, 1>), dim3((unsigned)((items + 3) / 4)), dim3(256), 0, stream, r);
            hipLaunchKernelGGL((embedding_grad_join_kernel<T, 1>), dim3(joins), dim3(512), 0, stream, r, columns);
        }
    });
    return check_launch("sg_embedding_backward");
}
