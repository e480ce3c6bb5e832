// Fully connected layer with its epilogue, and its gradients:
//   z = x w^T * w_gain + b * b_gain        y = act(z) * gain + residual           x [m, k], w [n, k], y [m, n]
//   s = dy * act'(z)      dx = s w * (gain w_gain)    dw = s^T x * (gain w_gain)    db = sum over rows of s * (gain b_gain)
// Three matrix products that differ in which index of each operand is contiguous; one kernel template covers them:
//   C[i, j] = sum over p of A(i, p) B(j, p),   each operand stored with p contiguous ("rows") or with i / j contiguous ("columns").
// An operand is never transposed in memory.  Tiles of 128 bytes along p travel to LDS as they lie (16 bytes per lane, straight
// into LDS where rows are 16-byte aligned), and a fragment of a "columns" operand is read by the transposing LDS read (16-bit)
// or two rows at a time (float32).  16-bit operands multiply on v_mfma_f32_16x16x32, float32 ones on v_mfma_f32_16x16x4_f32,
// whose products and sums are plain float32.  All sums are float32; every output is rounded once.
// Large products are bound by the matrix unit at the clock that power leaves: bfloat16 8192 x 4096 -> 4096 with bias, activation and
// residual 199 to 217 us (1270 to 1380 TFLOP/s), its gradients 200 to 207 each; float32 4096^3 915 to 975 (141 to 150).  Small ones
// are bound by launches: one row of 512 -> 512 3.8 us, a training step of 32 rows 18 in four launches.  float16 gradients have a launch
// more, which finds the largest |dy|: 3 us at 1000 x 1025.
//
// The gradient of the activation is s above without the gains: for the piecewise linear activations with slope 1 on one side
// its 16-bit rounding is exact there, so that folding sqrt(2) into the products' scale keeps it that way.  float16, whose range a
// slope above one leaves at the upper end and one far below at the lower, holds s times the power of two that brings
// max |dy| * (largest slope) to 2^14 .. 2^15; the sums are multiplied by its inverse (exact both ways).
#include "sg_absmax.h"
#include "sg_common.h"
#include "sg_column_sums.h"

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

namespace sg {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));

constexpr int kStepBytes = 128;                    // of p per step: two halves of 32 16-bit elements (one product) or 16 float32 ones (four)
constexpr unsigned kOutside = 0x80000000u;         // a buffer offset beyond every descriptor: the load yields zeros

enum { kActLinear = 1, kActRelu, kActLrelu, kActTanh, kActSigmoid, kActElu, kActSelu, kActSoftplus, kActSwish };
constexpr float kSeluScale = 1.0507009873554804934193349852946f, kSeluAlpha = 1.6732632423543772848170429916717f;

// exp and friends: the library's for float32 outputs; for 16-bit ones the hardware's exp2, log2 and reciprocal (1 ulp each, the
// argument's rounding adds |z| * 2^-24), which a 16-bit result does not see, with a series where a difference would cancel.
// An epilogue of ~35 instructions per element (expf, a division) takes 17 us of a 256 x 256 tile's 60 otherwise.
template <bool FAST> struct Math {
    static __device__ __forceinline__ float exp(float z) { return FAST ? __builtin_amdgcn_exp2f(z * 1.44269504088896341f) : expf(z); }
    static __device__ __forceinline__ float sigmoid(float z) { return FAST ? __builtin_amdgcn_rcpf(1.f + exp(-z)) : 1.f / (1.f + expf(-z)); }
    static __device__ __forceinline__ float tanh(float z) {
        if (!FAST) return tanhf(z);
        const float t = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + exp(2.f * z));
        return fabsf(z) < 0.02f ? z - z * z * z * (1.f / 3.f) : t;
    }
    static __device__ __forceinline__ float expm1(float z) {
        if (!FAST) return expm1f(z);
        return fabsf(z) < 0.01f ? z + z * z * (0.5f + z * (1.f / 6.f)) : exp(z) - 1.f;
    }
    static __device__ __forceinline__ float softplus(float z) {
        if (!FAST) return fmaxf(z, 0.f) + log1pf(expf(-fabsf(z)));
        const float t = exp(-fabsf(z));
        return fmaxf(z, 0.f) + (t < 0.001f ? t - 0.5f * t * t : __builtin_amdgcn_logf(1.f + t) * 0.693147180559945309f);
    }
};

template <int ACT, bool FAST> __device__ __forceinline__ float activation(float alpha, float z) {
    using M = Math<FAST>;
    if constexpr (ACT == kActRelu) return z > 0.f ? z : (z != z ? z : 0.f);
    if constexpr (ACT == kActLrelu) return z > 0.f ? z : z * alpha;
    if constexpr (ACT == kActTanh) return M::tanh(z);
    if constexpr (ACT == kActSigmoid) return M::sigmoid(z);
    if constexpr (ACT == kActElu) return z > 0.f ? z : M::expm1(z);
    if constexpr (ACT == kActSelu) return kSeluScale * (z > 0.f ? z : kSeluAlpha * M::expm1(z));
    if constexpr (ACT == kActSoftplus) return M::softplus(z);
    if constexpr (ACT == kActSwish) return z * M::sigmoid(z);
    return z;
}

// v = act(v) * gain for N values (one switch for all of them; the elements are a loop, not N copies of nine functions)
template <bool FAST, int N> __device__ __forceinline__ void activate(int act, float alpha, float gain, float (&v)[N]) {
#define SG_ACT(A) case A: _Pragma("unroll") for (int e = 0; e < N; e++) v[e] = activation<A, FAST>(alpha, v[e]) * gain; break;
    switch (act) {
        SG_ACT(kActRelu) SG_ACT(kActLrelu) SG_ACT(kActTanh) SG_ACT(kActSigmoid) SG_ACT(kActElu) SG_ACT(kActSelu) SG_ACT(kActSoftplus) SG_ACT(kActSwish)
        SG_ACT(kActLinear)
    }
#undef SG_ACT
}

// act'(z) of the activations that are not piecewise linear with corner at zero alone
template <bool FAST> __device__ __forceinline__ float slope_at(int act, float z) {
    using M = Math<FAST>;
    switch (act) {
        case kActTanh: { const float t = M::tanh(z); return 1.f - t * t; }
        case kActSigmoid: { const float t = M::sigmoid(z); return t * (1.f - t); }
        case kActElu: return z > 0.f ? 1.f : M::exp(z);
        case kActSelu: return kSeluScale * (z > 0.f ? 1.f : kSeluAlpha * M::exp(z));
        case kActSoftplus: return M::sigmoid(z);
        case kActSwish: { const float t = M::sigmoid(z); return t * (1.f + z * (1.f - t)); }
        default: return 1.f;
    }
}

// Rounding to T, to nearest even (bfloat16: the hardware's conversion).
template <class T> __device__ __forceinline__ T rounded(float v) { return Elem<T>::store(v); }
template <> __device__ __forceinline__ __hip_bfloat16 rounded<__hip_bfloat16>(float v) { return __builtin_bit_cast(__hip_bfloat16, (__bf16)v); }

// ---- the matrix product -----------------------------------------------------------------------------------------------------

struct Gemm {
    const void* a;                       // operand of the rows i
    const void* b;                       // operand of the columns j
    int64_t lda, ldb;                    // elements between rows as stored
    int64_t ni, nj, np;
    int tiles_i, tiles_j, slices, slice_steps;           // slice_steps: steps of 128 bytes along p
    int a_padded, b_padded;              // its rows go on with zeros to whole 16-byte packets
    float* partial;                      // [slices][ni][nj] when slices > 1
    void* out;                           // [ni][nj]
    float scale;
    const float* rescale;                // device value the scale is multiplied with (float16 gradients: a power of two), or NULL
    // epilogue of the forward pass
    const void* bias;                    // [nj]
    const void* residual;                // [ni][ldr]
    int64_t ldr;
    float* z;                            // [ni][nj] or NULL: pre-activation values for the backward pass
    uint8_t* positive;                   // [ni][nj] or NULL: z > 0
    int act;
    float alpha, gain, b_gain;
    int whole;                           // rows of everything the epilogue touches are whole aligned 16-byte packets
};

// Factor of the sums.  (The forward pass has none but the host's, and only float16 has one on the device.)
template <class T, bool FORWARD> __device__ __forceinline__ float scale_of(const Gemm& g) {
    if constexpr (!FORWARD && std::is_same_v<T, __half>) return g.rescale ? g.scale * *g.rescale : g.scale;
    else return g.scale;
}

// (of up to 16 bytes' alignment: longer runs are moved as packets)
template <class T, int N> struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Run { T v[N]; };

template <class T, int N> __device__ __forceinline__ Run<T, N> bias_run(const Gemm& g, int64_t j) {
    return g.bias ? *reinterpret_cast<const Run<T, N>*>((const T*)g.bias + j) : Run<T, N>{};
}

// N consecutive results (i, j .. j + N - 1), all inside; runs of N are aligned wherever they are read and written.
template <class T, int N, bool FORWARD>
__device__ __forceinline__ void finish(const Gemm& g, int64_t i, int64_t j, float (&v)[N]) {
    Run<T, N> bias{}, res{};
    if constexpr (FORWARD) {
        bias = bias_run<T, N>(g, j);
        if (g.residual) res = *reinterpret_cast<const Run<T, N>*>((const T*)g.residual + i * g.ldr + j);
    }
    const int64_t at = i * g.nj + j;
    Run<T, N> out;
    const float scale = scale_of<T, FORWARD>(g);
#pragma unroll
    for (int e = 0; e < N; e++) v[e] *= scale;
    if constexpr (FORWARD) {
        if (g.bias)
#pragma unroll
            for (int e = 0; e < N; e++) v[e] += Elem<T>::load(bias.v[e]) * g.b_gain;
        if (g.z) {
            Run<float, N> z;
#pragma unroll
            for (int e = 0; e < N; e++) z.v[e] = v[e];
            *reinterpret_cast<Run<float, N>*>(g.z + at) = z;
        }
        if (g.positive) {
            Run<uint8_t, N> pos;
#pragma unroll
            for (int e = 0; e < N; e++) pos.v[e] = v[e] > 0.f;
            *reinterpret_cast<Run<uint8_t, N>*>(g.positive + at) = pos;
        }
        activate<sizeof(T) == 2>(g.act, g.alpha, g.gain, v);
        if (g.residual)
#pragma unroll
            for (int e = 0; e < N; e++) v[e] += Elem<T>::load(res.v[e]);
    }
#pragma unroll
    for (int e = 0; e < N; e++) out.v[e] = rounded<T>(v[e]);
    *reinterpret_cast<Run<T, N>*>((T*)g.out + at) = out;
}

// Whether runs of N elements at multiples of N may be moved as one access: everything finish() touches keeps them aligned.
template <class T> bool runs_aligned(const Gemm& g) {
    const int n = 16 / (int)sizeof(T);
    auto ok = [&](const void* p, size_t bytes) { return p == nullptr || reinterpret_cast<uintptr_t>(p) % bytes == 0; };
    return g.nj % n == 0 && ok(g.out, n * sizeof(T)) && ok(g.bias, n * sizeof(T)) && ok(g.residual, n * sizeof(T)) &&
           (g.residual == nullptr || g.ldr % n == 0) && ok(g.z, 16) && ok(g.positive, n);
}

// Buffer descriptor of what follows p (offsets below kOutside).  p is the same in every lane of the wave.
__device__ __forceinline__ i32x4_t descriptor(const void* p) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return i32x4_t{__builtin_amdgcn_readfirstlane((int)a), __builtin_amdgcn_readfirstlane((int)(a >> 32) & 0xffff), (int)kOutside, 0x00020000};
}

// 16 bytes per lane from `offset` behind the descriptor's address to LDS at lds + PLACE + 16 * lane; zeros for kOutside.  Written as
// assembly because of its wait: the compiler holds every LDS read behind all copies into LDS that came before it, those into the
// other tiles included.  The kernel places the waits.  (One instruction sets the LDS address: a wave that has a SIMD to itself
// issues one in four cycles, 32 in the time of 8 products, and a step is built to stay below that.)
// (m0 is said to be overwritten, which is what is meant: the compiler warns, at every copy, that nobody saves it.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int PLACE> __device__ __forceinline__ void copy_to_lds(i32x4_t from, unsigned offset, unsigned lds) {
    asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds" ::"s"(lds), "n"(PLACE), "v"(offset), "s"(from) : "m0", "scc");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void copies_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ unsigned lds_address(const void* p) { return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const void*)p; }

// 16 bytes from the address of any element of T.  (A plain vector: a class type would keep its own alignment within the packed struct,
// and the load would claim an address that is a multiple of 16.)
template <class T> struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    sg_u32x4_t v;
    static __device__ __forceinline__ uint4 load(const T* p) {
        static_assert(alignof(Loose) == sizeof(T) && sizeof(Loose) == 16, "no more aligned than an element");
        const sg_u32x4_t q = reinterpret_cast<const Loose*>(p)->v;
        return make_uint4(q.x, q.y, q.z, q.w);
    }
};

// One operand's tile of SIDE rows i (or j) by 128 bytes of p in LDS: slots of 16 bytes, slot k * THREADS + t filled by thread t.
//   ROWS:  slot (row, c) holds the 16 bytes c ^ turn(row) of the row: the lanes that read at one time - 16 rows at one c, or 8 rows
//          each at two - hit 16 different 16-byte banks.
//   !ROWS: lines of SIDE elements at one p.  16-bit: the 32-byte block c of line q holds block c ^ swizzle(q), so that the
//          transposing read of 16 lines hits each 32-byte bank twice, once per half wave; float32: as it lies.  Line q holds
//          p = p_of(q): where a thread fills every 8th line (256 columns), bits 2 and 3 trade places, so that a thread's slots
//          share one swizzle.
// Either way a thread's slots are one address and constant distances apart.
template <class T, int SIDE, bool ROWS, int THREADS> struct Tile {
    static constexpr int ES = sizeof(T), E = 16 / ES, PITCH = kStepBytes, BK = PITCH / ES;
    static constexpr int BYTES = SIDE * PITCH;
    static constexpr int LOADS = BYTES / 16 / THREADS;             // 16-byte slots per thread
    static constexpr int LINE = ROWS ? PITCH / 16 : SIDE / E;      // slots per row or line
    static constexpr int APART = THREADS / LINE;                   // rows or lines from one slot of a thread to its next
    static constexpr bool SWAP = !ROWS && ES == 2 && APART == 8;
    static_assert(LOADS >= 1 && LOADS * THREADS * 16 == BYTES, "slots divide among the threads");
    static_assert(ROWS ? APART % 16 == 0 : ES == 4 || APART % 16 == 0 || SWAP, "a thread's slots share one swizzle");

    static __device__ __forceinline__ constexpr int turn(int row) { return (row >> 1) & 7; }
    static __device__ __forceinline__ constexpr int p_of(int q) { return SWAP ? (q & ~12) | (q & 4) << 1 | (q & 8) >> 1 : q; }
    static __device__ __forceinline__ int swizzle(int q) {
        if (ES == 4) return 0;
        if (SWAP) return q & 7;
        return SIDE >= 128 ? (q & 3) | ((q >> 3) & 1) << 2 : ((q >> 1) & 1) | ((q >> 3) & 1) << 1;
    }
    // distance of slot k from the first, along side (ROWS) or p (!ROWS)
    static __device__ __forceinline__ constexpr int apart(int k) { return ROWS ? k * APART : p_of(k * APART); }
    // the slots of a thread: its first one as (side, p) within the tile; byte offsets of all, kOutside beyond the matrix's side
    struct Slots { int side, p; unsigned off[LOADS]; };
    static __device__ __forceinline__ Slots plan(int64_t ld, int left_side) {
        Slots s;
        const int line = threadIdx.x / LINE, c = threadIdx.x % LINE;
        if (ROWS) {
            s.side = line;
            s.p = (c ^ turn(line)) * E;
        } else {
            s.p = p_of(line);
            s.side = (c ^ (swizzle(line) << 1)) * E;
        }
#pragma unroll
        for (int k = 0; k < LOADS; k++)
            s.off[k] = (ROWS ? s.side < left_side - apart(k) : s.side < left_side)
                           ? (unsigned)((ROWS ? s.side + apart(k) : s.p + apart(k)) * (unsigned)ld + (ROWS ? s.p : s.side)) * ES : kOutside;
        return s;
    }
    // slot k straight to LDS, at `lds` (the wave's share of the tile) + FIRST.  FULL: the step lies whole within p, else left_p of it
    template <int FIRST, int K, bool FULL> static __device__ __forceinline__ void copy(const Slots& s, i32x4_t from, unsigned lds, int left_p) {
        const bool in = FULL || s.p < left_p - (ROWS ? 0 : apart(K));
        copy_to_lds<FIRST + K * THREADS * 16>(from, in ? s.off[K] : kOutside, lds);
    }
    // by way of registers: any alignment, any extent
    // A slot that the end of its row cuts is read from the row's last 16 bytes and shifted into place when it is written to LDS, so
    // that every slot is one load without a branch around it and nothing waits for a load before then.  (extent_c: elements from
    // the tile's first one to the end of its rows, along the contiguous index.)  Rows shorter than 16 bytes are read element by
    // element (SHORT).
    struct Regs { uint4 v[LOADS]; };
    static __device__ __forceinline__ bool line_inside(const Slots& s, int k, int left_side, int left_p) {
        return ROWS ? s.side < left_side - apart(k) : s.p < left_p - apart(k);
    }
    // elements of the slot beyond the end of its row
    static __device__ __forceinline__ int cut_of(const Slots& s, int64_t extent_c) {
        const int c = ROWS ? s.p : s.side;
        return c + E > extent_c ? (int)min(c + E - extent_c, (int64_t)E) : 0;
    }
    template <bool SHORT>
    static __device__ __forceinline__ void fetch(Regs& r, const Slots& s, const T* base, int64_t ld, int left_side, int left_p, int64_t extent_c) {
        const int c = ROWS ? s.p : s.side, cut = cut_of(s, extent_c);
        const int64_t back = SHORT ? 0 : cut == E ? extent_c - E : c - cut;        // (a slot wholly outside reads what is inside)
#pragma unroll
        for (int k = 0; k < LOADS; k++) {
            const T* line = base + (line_inside(s, k, left_side, left_p) ? (ROWS ? s.side : s.p) + apart(k) : 0) * ld;
            if constexpr (SHORT) {
                Pack<T> q;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const T v = line[c + e < extent_c ? c + e : 0];
                    q.v[e] = c + e < extent_c ? v : Elem<T>::store(0.f);
                }
                __builtin_memcpy(&r.v[k], &q, 16);
            } else {
                r.v[k] = Loose<T>::load(line + back);
            }
        }
    }
    template <bool SHORT>
    static __device__ __forceinline__ void commit(unsigned char* lds, const Regs& r, const Slots& s, int left_side, int left_p, int64_t extent_c) {
        const int cut = cut_of(s, extent_c);
#pragma unroll
        for (int k = 0; k < LOADS; k++) {
            uint4 q = r.v[k];
            if (!SHORT) {                                              // up by `cut` elements, zeros behind them
                if (ES == 2 && (cut & 1)) q = make_uint4(q.x >> 16 | q.y << 16, q.y >> 16 | q.z << 16, q.z >> 16 | q.w << 16, q.w >> 16);
                if (cut & (4 / ES)) q = make_uint4(q.y, q.z, q.w, 0);
                if (cut & (8 / ES)) q = make_uint4(q.z, q.w, 0, 0);
            }
            const bool zero = cut == E || left_side <= 0 || !line_inside(s, k, left_side, left_p);
            *reinterpret_cast<uint4*>(lds + (k * THREADS + threadIdx.x) * 16) = zero ? make_uint4(0, 0, 0, 0) : q;
        }
    }
};

// Fragments of COUNT 16-row tiles from row `first` of an LDS tile, for half kk of a step.
template <class T, int SIDE, bool ROWS, int THREADS, int COUNT> struct Frags {
    using Here = Tile<T, SIDE, ROWS, THREADS>;
    static constexpr int V = sizeof(T) == 4 && !ROWS ? 2 : 1;                          // tiles whose rows interleave
    static_assert(COUNT % V == 0, "interleaved tiles come in pairs");
    uint4 q[COUNT];                                                                   // 8 16-bit values, or 4 float32 (ROWS)
    float f[sizeof(T) == 4 && !ROWS ? COUNT : 1][4];

    // row within the wave's share of element `r16` (0 .. 15) of tile t
    static __device__ __forceinline__ int row(int t, int r16) { return (t / V) * 16 * V + r16 * V + t % V; }

    // tile t (with V == 2: tiles t and t + 1, for an even t)
    __device__ __forceinline__ void read(const unsigned char* lds, int first, int kk, int t) {
        const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
        if constexpr (ROWS) {
            const int at = (first + l16) * Here::PITCH + (((kk * 4 + g) ^ Here::turn(l16)) << 4);
            q[t] = *reinterpret_cast<const uint4*>(lds + at + t * 16 * Here::PITCH);
        } else if constexpr (sizeof(T) == 2) {
            constexpr int LINE = SIDE * 2;
            const int q0 = Here::p_of(kk * 32 + g * 8 + (l16 >> 2));        // (its own inverse)
            const unsigned char* at = lds + q0 * LINE + (l16 & 3) * 8 + (((first >> 4) + t) ^ Here::swizzle(q0)) * 32;
            typedef __attribute__((address_space(3))) s16x4_t* Lds;
            const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)at);
            const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(at + Here::p_of(4) * LINE));
            const uint2 a = __builtin_bit_cast(uint2, lo), b = __builtin_bit_cast(uint2, hi);
            q[t] = make_uint4(a.x, a.y, b.x, b.y);
        } else {
            constexpr int LINE = SIDE * 4;
            if (t % V == 0)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const unsigned char* at = lds + (kk * 16 + g * 4 + e) * LINE + (first + t * 16 + l16 * V) * 4;
                    const f32x2_t v = *reinterpret_cast<const f32x2_t*>(at);
                    f[t][e] = v.x; f[t + 1][e] = v.y;
                }
        }
    }
    __device__ __forceinline__ void read(const unsigned char* lds, int first, int kk) {
#pragma unroll
        for (int t = 0; t < COUNT; t++) read(lds, first, kk, t);
    }
    __device__ __forceinline__ float value(int t, int e) const {
        if constexpr (ROWS) return __builtin_bit_cast(f32x4_t, q[t])[e];
        else return f[t][e];
    }
};

__device__ __forceinline__ f32x4_t mfma(const uint4& a, const uint4& b, f32x4_t c, __hip_bfloat16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mfma(const uint4& a, const uint4& b, f32x4_t c, __half) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// c += a b, written as assembly for the one thing the builtin does not say: c is read and written in place, in accumulation
// registers.  (With 256 of them a lane the register allocator otherwise moves accumulators about, up to 448 moves in a step of 128
// products and two thirds more time.)  Products of one accumulator are four or more products apart, and settle() is the wait
// before anything else reads them.
__device__ __forceinline__ void mfma_in_place(f32x4_t& c, const uint4& a, const uint4& b, __hip_bfloat16) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(__builtin_bit_cast(bf16x8_t, a)), "v"(__builtin_bit_cast(bf16x8_t, b)));
}
__device__ __forceinline__ void mfma_in_place(f32x4_t& c, const uint4& a, const uint4& b, __half) {
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(__builtin_bit_cast(f16x8_t, a)), "v"(__builtin_bit_cast(f16x8_t, b)));
}
template <int M, int N> __device__ __forceinline__ void settle(f32x4_t (&acc)[M][N]) {
    asm volatile("s_nop 15\n\ts_nop 15");               // more than the passes of a 16 x 16 x 32 product
#pragma unroll
    for (int t = 0; t < M; t++)
#pragma unroll
        for (int s = 0; s < N; s++) asm volatile("" : "+a"(acc[t][s]));
}

// f(integral_constant 0), f(integral_constant 1), ...
template <class F, int... K> __device__ __forceinline__ void for_each(F f, std::integer_sequence<int, K...>) { (f(std::integral_constant<int, K>{}), ...); }

// How operands travel: kDirect, rows of both are whole aligned 16-byte packets; kLoose, rows start anywhere and end anywhere;
// kShort, rows of one of them are shorter than 16 bytes.
enum { kDirect, kLoose, kShort };

// Steps of A and B in LDS: RING of both, and one more of A in tiles that have a CU to themselves or share it with one other.
template <int BI, int RING> constexpr int kRingA = BI >= 128 ? RING + 1 : RING;
template <int BI, int BJ, int RING> constexpr int kTileBytes = (kRingA<BI, RING> * BI + RING * BJ) * kStepBytes;

// One tile BI x BJ by a workgroup of WI x WJ waves.  Products of two "rows" operands are the forward pass and carry its epilogue.
template <class T, int BI, int BJ, int WI, int WJ, bool ROWS_A, bool ROWS_B, int MODE, int RING>
__device__ __forceinline__ void gemm_tile(const Gemm& g, unsigned id, unsigned char* smem) {
    constexpr bool FORWARD = ROWS_A && ROWS_B;
    constexpr int THREADS = WI * WJ * 64, TI = BI / WI / 16, TJ = BJ / WJ / 16, BK = kStepBytes / (int)sizeof(T);
    constexpr int RING_A = kRingA<BI, RING>;
    using TileA = Tile<T, BI, ROWS_A, THREADS>;
    using TileB = Tile<T, BJ, ROWS_B, THREADS>;
    using FragA = Frags<T, BI, ROWS_A, THREADS, TI>;
    using FragB = Frags<T, BJ, ROWS_B, THREADS, TJ>;
    constexpr int BUF = TileA::BYTES + TileB::BYTES;

    // Workgroups go round robin over the 8 XCDs: each XCD gets a contiguous share of the tiles, in groups of 8 tile rows so that
    // the tiles it works on at one time share rows of A and columns of B in its L2.
    const unsigned tiles = (unsigned)g.tiles_i * g.tiles_j, total = tiles * g.slices;
    {
        const unsigned per = total / 8, extra = total % 8, xcd = id % 8, k = id / 8;
        id = xcd * per + (xcd < extra ? xcd : extra) + k;
    }
    const unsigned slice = id / tiles, tile = id % tiles;
    const unsigned group = 8u * g.tiles_j, g0 = tile / group * 8u;
    const unsigned rows = min((unsigned)g.tiles_i - g0, 8u);
    const int64_t i0 = (int64_t)(g0 + tile % group % rows) * BI, j0 = (int64_t)(tile % group / rows) * BJ;

    const T* a = (const T*)g.a + (ROWS_A ? i0 * g.lda : i0);
    const T* b = (const T*)g.b + (ROWS_B ? j0 * g.ldb : j0);
    const int left_i = (int)min(g.ni - i0, (int64_t)BI), left_j = (int)min(g.nj - j0, (int64_t)BJ);
    const int steps_all = (int)((g.np + BK - 1) / BK);
    const int first = (int)slice * g.slice_steps, steps = min(g.slice_steps, steps_all - first);

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = (wave / WJ) * (BI / WI), wj = (wave % WJ) * (BJ / WJ);
    f32x4_t acc[TJ][TI];
#pragma unroll
    for (int t = 0; t < TJ; t++)
#pragma unroll
        for (int s = 0; s < TI; s++) acc[t][s] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    auto left_p = [&](int step) { return (int)min(g.np - (int64_t)step * BK, (int64_t)BK); };
    const typename TileA::Slots sa = TileA::plan(g.lda, left_i);
    const typename TileB::Slots sb = TileB::plan(g.ldb, left_j);
    auto at_a = [&](int step) { return a + (ROWS_A ? (int64_t)step * BK : (int64_t)step * BK * g.lda); };
    auto at_b = [&](int step) { return b + (ROWS_B ? (int64_t)step * BK : (int64_t)step * BK * g.ldb); };
    auto multiply = [&](const FragA& fa, const FragB& fb, int t, int s) {
        if constexpr (sizeof(T) == 2) {
            mfma_in_place(acc[t][s], fb.q[t], fa.q[s], T());
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) acc[t][s] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb.value(t, e), fa.value(s, e), acc[t][s], 0, 0, 0);
        }
    };
    // column tile t of the wave's part
    auto multiply_tile = [&](const FragA& fa, const FragB& fb, int t) {
#pragma unroll
        for (int s = 0; s < TI; s++) multiply(fa, fb, t, s);
    };
    if constexpr (MODE == kDirect) {
        // Two sets of fragments, one for each half of a step: one is multiplied while the other is read, so that the matrix unit has
        // its operands in registers at the barrier between the halves: every wave has read the step's tiles for the last time, and
        // the next step's have landed.  Behind it the copies of step n + RING start into the tiles just read.  With a tile
        // more of A, those of A start in the first half of the step after: reads and copies then lie evenly between the
        // products.  (As a batch they hold up the wave's products behind them.)
        const unsigned lds = __builtin_amdgcn_readfirstlane(lds_address(smem) + wave * 1024);
        constexpr int PARTS = TI > TJ ? TI : TJ, BASE_B = RING_A * TileA::BYTES, COPIES = TileA::LOADS + TileB::LOADS;
        constexpr bool EARLY_A = RING_A > RING;
        FragA fa[2];
        FragB fb[2];
        // where the next step to be copied starts, and goes
        const T *from_a = at_a(first), *from_b = at_b(first);
        const int64_t step_a = ROWS_A ? BK : BK * g.lda, step_b = ROWS_B ? BK : BK * g.ldb;
        i32x4_t a4 = descriptor(from_a), b4 = descriptor(from_b);
        unsigned to_a = lds, to_b = lds + BASE_B;
        // share `part` of PARTS of a step's copies.  full: it lies whole within p, else `left` of it (none of a step behind the
        // last: zeros, which count for nothing)
        auto copy_a = [&](int part, auto full, int left) {
            for_each([&](auto k) {
                constexpr int K = decltype(k)::value;
                if (K * PARTS / TileA::LOADS == part) TileA::template copy<0, K, decltype(full)::value>(sa, a4, to_a, left);
            }, std::make_integer_sequence<int, TileA::LOADS>{});
        };
        auto copy_b = [&](int part, auto full, int left) {
            for_each([&](auto k) {
                constexpr int K = decltype(k)::value;
                if (K * PARTS / TileB::LOADS == part) TileB::template copy<0, K, decltype(full)::value>(sb, b4, to_b, left);
            }, std::make_integer_sequence<int, TileB::LOADS>{});
        };
        auto next_a = [&] {
            from_a += step_a;
            a4 = descriptor(from_a);
            to_a = to_a == lds + (RING_A - 1) * TileA::BYTES ? lds : to_a + TileA::BYTES;
        };
        auto next_b = [&] {
            from_b += step_b;
            b4 = descriptor(from_b);
            to_b = to_b == lds + BASE_B + (RING - 1) * TileB::BYTES ? lds + BASE_B : to_b + TileB::BYTES;
        };
        auto left_of = [&](int n) { return n < steps ? left_p(first + n) : 0; };
        auto copy_all = [&](int n) {
            const int left = left_of(n);
#pragma unroll
            for (int part = 0; part < PARTS; part++) {
                copy_a(part, std::false_type{}, left);
                copy_b(part, std::false_type{}, left);
            }
            next_a();
            next_b();
        };
        // share `part` of the reads: spread over the first three quarters, so that the last of them are back in time
        constexpr int READ_PARTS = PARTS >= 4 ? PARTS * 3 / 4 : PARTS;
        auto read_a = [&](int set, const unsigned char* from, int part) {
#pragma unroll
            for (int t = 0; t < TI; t++)
                if (t * READ_PARTS / TI == part) fa[set].read(from, wi, set, t);
        };
        auto read_b = [&](int set, const unsigned char* from, int part) {
#pragma unroll
            for (int t = 0; t < TJ; t++)
                if (t * READ_PARTS / TJ == part) fb[set].read(from, wj, set, t);
        };
        const unsigned char *now_a = smem, *now_b = smem + BASE_B;
        // half a step: multiplies set, reads the other one, copies between the products
        auto half = [&](auto set, auto copies, auto next) {
            constexpr int SET = decltype(set)::value;
#pragma unroll
            for (int t = 0; t < PARTS; t++) {
#pragma unroll
                for (int s = 0; s < TI; s++) {
                    if (s == 0) copies(t);
                    if (s == TI / 4) read_a(SET ^ 1, now_a, t);
                    if (s == TI / 2) read_b(SET ^ 1, now_b, t);
                    if (t == PARTS - 1 && s == TI / 4) next();
                    if (t < TJ) multiply(fa[SET], fb[SET], t, s);
                    if (TI == 8 || s == TI - 1) __builtin_amdgcn_sched_barrier(0);      // (or the reads gather behind the products)
                }
            }
        };
        using First = std::integral_constant<int, 0>;
        using Second = std::integral_constant<int, 1>;
        auto step = [&](int n, auto full) {                              // full: step n + RING is
            const int left = full ? BK : left_of(n + RING);
            half(First{}, [&](int t) { if (EARLY_A) copy_a(t, full, left); }, [&] { if (EARLY_A) next_a(); });
            now_a = now_a == smem + (RING_A - 1) * TileA::BYTES ? smem : now_a + TileA::BYTES;
            now_b = now_b == smem + BASE_B + (RING - 1) * TileB::BYTES ? smem + BASE_B : now_b + TileB::BYTES;
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((RING - 2) * COPIES + (EARLY_A ? TileA::LOADS : 0)) : "memory");
            half(Second{}, [&](int t) { if (!EARLY_A) copy_a(t, full, left); copy_b(t, full, left); }, [&] { if (!EARLY_A) next_a(); next_b(); });
        };
        if (steps > 0) {
#pragma unroll
            for (int k = 0; k < RING; k++) copy_all(k);
            asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((RING - 1) * COPIES) : "memory");
            fa[0].read(smem, wi, 0);
            fb[0].read(smem + BASE_B, wj, 0);
        }
        int n = 0;
        const int full_steps = min(steps, (int)(g.np / BK) - first);      // of this slice
#pragma unroll 1
        for (; n + RING < full_steps; n++) step(n, std::true_type{});
#pragma unroll 1
        for (; n < steps; n++) step(n, std::false_type{});
        copies_landed();                                                 // (the epilogue writes where they go)
    } else {
        // Two LDS buffers and two sets of registers: a step's loads have the two steps before it to arrive; one barrier a step.
        // Steps go in pairs and every step loads, the last ones their own data again (behind a branch the compiler would wait
        // for the newest loads where it needs those of the step before); what lies behind the last step is written as zeros.
        typename TileA::Regs ra[2];
        typename TileB::Regs rb[2];
        auto rest = [&](int n) { return g.np - (int64_t)(first + n) * BK; };
        auto fetch = [&](int n, int set) {
            n = min(n, steps - 1);
            const int left = left_p(first + n);
            TileA::template fetch<MODE == kShort>(ra[set], sa, at_a(first + n), g.lda, left_i, left, ROWS_A ? rest(n) : g.ni - i0);
            TileB::template fetch<MODE == kShort>(rb[set], sb, at_b(first + n), g.ldb, left_j, left, ROWS_B ? rest(n) : g.nj - j0);
        };
        auto commit = [&](int n, int set) {
            const int li = n < steps ? left_i : 0, lj = n < steps ? left_j : 0;
            n = min(n, steps - 1);
            const int left = left_p(first + n);
            TileA::template commit<MODE == kShort>(smem + set * BUF, ra[set], sa, li, left, ROWS_A ? rest(n) : g.ni - i0);
            TileB::template commit<MODE == kShort>(smem + set * BUF + TileA::BYTES, rb[set], sb, lj, left, ROWS_B ? rest(n) : g.nj - j0);
        };
        auto step = [&](int n, int set) {                          // set = n & 1
            __syncthreads();
            fetch(n + 2, set);
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                FragA fa;
                FragB fb;
                fa.read(smem + set * BUF, wi, kk);
                fb.read(smem + set * BUF + TileA::BYTES, wj, kk);
#pragma unroll
                for (int t = 0; t < TJ; t++) multiply_tile(fa, fb, t);
            }
            commit(n + 1, set ^ 1);
        };
        if (steps > 0) {
            fetch(0, 0);
            fetch(1, 1);
            commit(0, 0);
            for (int n = 0; n < steps; n += 2) {
                step(n, 0);
                step(n + 1, 1);
            }
        }
    }

    if constexpr (sizeof(T) == 2) settle(acc);

    // acc[t][s][r]: row i = tile s of A at lane % 16, column j = tile t of B at 4 * (lane / 16) + r.  Each wave lays its part
    // down in LDS as rows of four-column chunks (chunk c of row r at c ^ r: the 16 rows a store touches lie in 16 different
    // 16-byte banks) and takes it up again in runs of consecutive columns: stores of 16 bytes, and one copy of the
    // epilogue's code.
    constexpr int COLS = BJ / WJ, CHUNKS = COLS / 4, ROWS_MAX = BUF * 2 / (WI * WJ) / (COLS * 4);
    constexpr int S_PASS = ROWS_MAX / 16 < TI ? ROWS_MAX / 16 : TI;      // A tiles per pass
    constexpr int N = 16 / (int)sizeof(T), RUNS = COLS / N;
    static_assert(S_PASS >= 1 && TI % S_PASS == 0, "the epilogue's passes");
    const int lane = threadIdx.x & 63, l16 = lane & 15, quad = lane >> 4;
    float* mine = reinterpret_cast<float*>(smem) + wave * (S_PASS * 16 * COLS);
    auto chunk_at = [&](int row, int chunk) -> f32x4_t& { return *reinterpret_cast<f32x4_t*>(mine + row * COLS + (chunk ^ (row & (CHUNKS - 1))) * 4); };
    const float scale = scale_of<T, FORWARD>(g);
    __syncthreads();                                                     // every wave is done with the tiles
    auto lay_down = [&](int s, int row) {                                 // A tile s, constant, as the region's rows from `row` on
#pragma unroll
        for (int t = 0; t < TJ; t++) {
            if constexpr (FragB::V == 1) {
                chunk_at(row, t * 4 + quad) = acc[t][s];
            } else {                                                     // tiles t and t + 1 hold alternate columns
                if (t % 2 == 0)
#pragma unroll
                    for (int r = 0; r < 4; r += 2)
                        chunk_at(row, t / 2 * 8 + quad * 2 + r / 2) = f32x4_t{acc[t][s][r], acc[t + 1][s][r], acc[t][s][r + 1], acc[t + 1][s][r + 1]};
            }
        }
    };
    // (one copy of the code behind lay_down for all passes; accumulators are picked by constants, or they would move to memory)
#pragma unroll 1
    for (int s0 = 0; s0 < TI; s0 += S_PASS) {
#pragma unroll
        for (int pass = 0; pass < TI / S_PASS; pass++)
            if (s0 == pass * S_PASS)
#pragma unroll
                for (int s = 0; s < S_PASS; s++) lay_down(pass * S_PASS + s, s * 16 + l16);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        // 64 / RUNS rows at a time; a lane keeps its columns.
        constexpr int ROUND = 64 / RUNS, ROUNDS = S_PASS * 16 / ROUND;
        static_assert(ROUND * RUNS == 64 && ROUNDS * ROUND == S_PASS * 16, "whole rounds");
        const int run = lane % RUNS, row0 = lane / RUNS;
        const int64_t j = j0 + wj + run * N;
        auto row_of = [&](int round) { const int row = round * ROUND + row0; return i0 + wi + FragA::row(s0 + row / 16, row % 16); };
        auto take = [&](int round, float* v) {
#pragma unroll
            for (int q = 0; q < N / 4; q++) {
                const f32x4_t c = chunk_at(round * ROUND + row0, run * (N / 4) + q);
                v[4 * q] = c.x; v[4 * q + 1] = c.y; v[4 * q + 2] = c.z; v[4 * q + 3] = c.w;
            }
        };
        // Rows of whole packets.  Inside the matrix there is no branch around a load or a store: both count in vmcnt, behind a branch
        // the compiler cannot count, and a wait for the prefetched residual becomes one for every store as well (28 us a 256 x 256
        // tile instead of 8).
        if (g.slices == 1 && g.whole) {
            constexpr int U = ROUNDS % 2 == 0 ? 2 : 1;
            auto rounds = [&](auto has_residual, auto edge) {
                if (edge && j >= g.nj) return;
                auto there = [&](int64_t i) { return edge ? i < g.ni : true; };
                auto clamped = [&](int64_t i) { return edge ? min(i, g.ni - 1) : i; };
                float bias[N] = {};
                Run<T, N> next[U];
                if constexpr (FORWARD) {
                    const Run<T, N> raw = bias_run<T, N>(g, j);
#pragma unroll
                    for (int e = 0; e < N; e++) bias[e] = Elem<T>::load(raw.v[e]) * g.b_gain;
                    if constexpr (has_residual)
#pragma unroll
                        for (int u = 0; u < U; u++) next[u] = *reinterpret_cast<const Run<T, N>*>((const T*)g.residual + clamped(row_of(u)) * g.ldr + j);
                }
#pragma unroll 1
                for (int round = 0; round < ROUNDS; round += U) {
                    Run<T, N> now[U];
                    if constexpr (has_residual) {
                        const int ahead = min(round + U, ROUNDS - U);
#pragma unroll
                        for (int u = 0; u < U; u++) {
                            now[u] = next[u];
                            next[u] = *reinterpret_cast<const Run<T, N>*>((const T*)g.residual + clamped(row_of(ahead + u)) * g.ldr + j);
                        }
                    }
                    float v[U * N];
#pragma unroll
                    for (int u = 0; u < U; u++) take(round + u, v + u * N);
#pragma unroll
                    for (int e = 0; e < U * N; e++) v[e] = v[e] * scale + bias[e % N];
                    if constexpr (FORWARD) {
                        if (g.z)
#pragma unroll
                            for (int u = 0; u < U; u++)
#pragma unroll
                                for (int q = 0; q < N; q += 4)
                                    if (there(row_of(round + u))) *reinterpret_cast<f32x4_t*>(g.z + row_of(round + u) * g.nj + j + q) =
                                        f32x4_t{v[u * N + q], v[u * N + q + 1], v[u * N + q + 2], v[u * N + q + 3]};
                        if (g.positive)
#pragma unroll
                            for (int u = 0; u < U; u++) {
                                Run<uint8_t, N> pos;
#pragma unroll
                                for (int e = 0; e < N; e++) pos.v[e] = v[u * N + e] > 0.f;
                                if (there(row_of(round + u))) *reinterpret_cast<Run<uint8_t, N>*>(g.positive + row_of(round + u) * g.nj + j) = pos;
                            }
                        activate<sizeof(T) == 2>(g.act, g.alpha, g.gain, v);
                        if constexpr (has_residual)
#pragma unroll
                            for (int e = 0; e < U * N; e++) v[e] += Elem<T>::load(now[e / N].v[e % N]);
                    }
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        Run<T, N> out;
#pragma unroll
                        for (int e = 0; e < N; e++) out.v[e] = rounded<T>(v[u * N + e]);
                        if (there(row_of(round + u))) *reinterpret_cast<Run<T, N>*>((T*)g.out + row_of(round + u) * g.nj + j) = out;
                    }
                }
            };
            using Yes = std::true_type;
            using No = std::false_type;
            const bool edge = left_i < BI || left_j < BJ;
            if (FORWARD && g.residual) edge ? rounds(Yes{}, Yes{}) : rounds(Yes{}, No{});
            else edge ? rounds(No{}, Yes{}) : rounds(No{}, No{});
        } else if (g.slices == 1) {
            // Rows that start anywhere: a lane takes single elements, neighbouring lanes neighbouring columns.
            constexpr int SETS = COLS > 64 ? COLS / 64 : 1, STRIDE = COLS > 64 ? 1 : 64 / COLS, U = sizeof(T) == 2 ? 8 : 4;     // columns per lane; rows per round
            static_assert(S_PASS * 16 % (STRIDE * U) == 0, "whole rounds");
#pragma unroll 1
            for (int set = 0; set < SETS; set++) {
                const int col = set * 64 + (COLS > 64 ? lane : lane % COLS);
                const int64_t jj = j0 + wj + col;
                if (jj >= g.nj) continue;
                const float bias = FORWARD && g.bias ? Elem<T>::load(((const T*)g.bias)[jj]) * g.b_gain : 0.f;
#pragma unroll 1
                for (int r0 = COLS > 64 ? 0 : lane / COLS; r0 < S_PASS * 16; r0 += STRIDE * U) {
                    float v[U], res[U];
                    int64_t at[U];
                    bool there[U];
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const int row = r0 + u * STRIDE;
                        const int64_t i = i0 + wi + FragA::row(s0 + row / 16, row % 16);
                        there[u] = i < g.ni;
                        at[u] = i * g.nj + jj;
                        v[u] = chunk_at(row, col / 4)[col % 4] * scale + bias;
                        if (FORWARD && g.residual) res[u] = Elem<T>::load(((const T*)g.residual)[(there[u] ? i : 0) * g.ldr + jj]);
                    }
                    if constexpr (FORWARD) {
                        if (g.z)
#pragma unroll
                            for (int u = 0; u < U; u++)
                                if (there[u]) g.z[at[u]] = v[u];
                        if (g.positive)
#pragma unroll
                            for (int u = 0; u < U; u++)
                                if (there[u]) g.positive[at[u]] = v[u] > 0.f;
                        activate<sizeof(T) == 2>(g.act, g.alpha, g.gain, v);
                        if (g.residual)
#pragma unroll
                            for (int u = 0; u < U; u++) v[u] += res[u];
                    }
#pragma unroll
                    for (int u = 0; u < U; u++)
                        if (there[u]) ((T*)g.out)[at[u]] = rounded<T>(v[u]);
                }
            }
        } else {
#pragma unroll 1
            for (int round = 0; round < ROUNDS; round++) {
                const int64_t i = row_of(round);
                if (i >= g.ni || j >= g.nj) continue;
                float v[N];
                take(round, v);
                float* out = g.partial + ((int64_t)slice * g.ni + i) * g.nj + j;
                if (g.whole) {
#pragma unroll
                    for (int q = 0; q < N; q += 4) *reinterpret_cast<f32x4_t*>(out + q) = f32x4_t{v[q], v[q + 1], v[q + 2], v[q + 3]};
                } else {
#pragma unroll
                    for (int e = 0; e < N; e++)
                        if (j + e < g.nj) out[e] = v[e];
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// (64 x 64: five workgroups on a CU, as many as its LDS holds.  float32 10000 x 512 -> 512, 1256 of them: 55 us with four and 49 with
// five when they were compared, 44 with the steps of today)
template <class T, int BI, int BJ, int WI, int WJ, bool ROWS_A, bool ROWS_B, int MODE, int RING>
__global__ void __launch_bounds__(WI * WJ * 64, BI == 64 && MODE == kDirect && RING == 2 ? 5 : 1) linear_gemm_kernel(const Gemm g) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[kTileBytes<BI, BJ, RING>];
    gemm_tile<T, BI, BJ, WI, WJ, ROWS_A, ROWS_B, MODE, RING>(g, blockIdx.x, smem);
}

// Few rows (at most 32) and a short sum: the tile kernel would spend most of its products on rows that are not there, and need
// slices and a second launch to use more than a few CUs.  Here eight waves share the sum of 16 (ROWS_B) or 32 columns: operands go
// from global memory to fragments, 64 bytes of p per wave and turn (the eight waves' turns lie side by side), the waves' sums are
// added in wave order.  Rows of both operands are whole aligned packets.  TI: row tiles.  One row of 512 -> 512 in float32: 3.8 us, and
// 7.5 as one 64 x 64 tile in eight slices.
template <class T, int TI, bool ROWS_B>
__global__ void __launch_bounds__(512) linear_thin_kernel(const Gemm g) {
    constexpr int WAVES = 8, TJ = ROWS_B ? 1 : 2, COLS = 16 * TJ, E = 16 / (int)sizeof(T), UNIT = 4 * E, UNROLL = 4;
    static_assert(ROWS_B || sizeof(T) == 4, "16-bit columns need the transposing read");
    __shared__ __attribute__((aligned(16))) float part[WAVES][TI * 16][COLS + 4];
    const int lane = threadIdx.x & 63, l16 = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t j0 = (int64_t)blockIdx.x * COLS;
    const T* a = (const T*)g.a;
    const T* b = (const T*)g.b;
    const int64_t units = (g.np + UNIT - 1) / UNIT;
    f32x4_t acc[TJ][TI];
#pragma unroll
    for (int t = 0; t < TJ; t++)
#pragma unroll
        for (int s = 0; s < TI; s++) acc[t][s] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int64_t u0 = wave; u0 < units; u0 += WAVES * UNROLL) {
        uint4 fa[UNROLL][TI], fb[UNROLL];
        float fc[UNROLL][TJ][4];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const int64_t p = (u0 + u * WAVES) * UNIT + quad * E;
            const bool in = p < g.np;
#pragma unroll
            for (int s = 0; s < TI; s++) fa[u][s] = load16_or_zero(in && s * 16 + l16 < g.ni, a + (s * 16 + l16) * g.lda + p);
            if constexpr (ROWS_B) {
                fb[u] = load16_or_zero(in && j0 + l16 < g.nj, b + (j0 + l16) * g.ldb + p);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {              // two columns a lane
                    const uint2 v = load8_or_zero(p + e < g.np && j0 + 2 * l16 < g.nj, b + (p + e) * g.ldb + j0 + 2 * l16);
                    fc[u][0][e] = __uint_as_float(v.x);
                    fc[u][1][e] = __uint_as_float(v.y);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; u++)
#pragma unroll
            for (int t = 0; t < TJ; t++)
#pragma unroll
                for (int s = 0; s < TI; s++) {
                    if constexpr (sizeof(T) == 2) {
                        acc[t][s] = mfma(fb[u], fa[u][s], acc[t][s], T());
                    } else {
                        const f32x4_t va = __builtin_bit_cast(f32x4_t, fa[u][s]);
                        const f32x4_t vb = ROWS_B ? __builtin_bit_cast(f32x4_t, fb[u]) : f32x4_t{fc[u][t][0], fc[u][t][1], fc[u][t][2], fc[u][t][3]};
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[t][s] = __builtin_amdgcn_mfma_f32_16x16x4f32(vb[e], va[e], acc[t][s], 0, 0, 0);
                    }
                }
    }
    // row s * 16 + l16, columns quad * 4 + r (two tiles: interleaved)
#pragma unroll
    for (int s = 0; s < TI; s++)
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int t = 0; t < TJ; t++) part[wave][s * 16 + l16][(quad * 4 + r) * TJ + t] = acc[t][s][r];
    __syncthreads();
    for (int k = threadIdx.x; k < TI * 16 * COLS; k += 512) {
        const int i = k / COLS, c = k % COLS;
        if (i >= g.ni || j0 + c >= g.nj) continue;
        float v[1] = {0.f};
#pragma unroll
        for (int w = 0; w < WAVES; w++) v[0] += part[w][i][c];
        finish<T, 1, ROWS_B>(g, i, j0 + c, v);
    }
}

// The slices' partial sums, added in slice order, and the epilogue.
template <class T, int RUN, bool FORWARD> __device__ __forceinline__ void join_slices(const Gemm& g, unsigned block) {
    const int64_t k = ((int64_t)block * 256 + threadIdx.x) * RUN;
    const int64_t plane = g.ni * g.nj;
    if (k >= plane) return;
    float v[RUN];
#pragma unroll
    for (int e = 0; e < RUN; e++) v[e] = 0.f;
    constexpr int AHEAD = 8;              // loads under way (slices behind the last read it again and count as nothing)
    for (int s = 0; s < g.slices; s += AHEAD) {
        Run<float, RUN> q[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; u++) q[u] = *reinterpret_cast<const Run<float, RUN>*>(g.partial + (int64_t)min(s + u, g.slices - 1) * plane + k);
#pragma unroll
        for (int u = 0; u < AHEAD; u++)
#pragma unroll
            for (int e = 0; e < RUN; e++) v[e] += s + u < g.slices ? q[u].v[e] : 0.f;
    }
    finish<T, RUN, FORWARD>(g, k / g.nj, k % g.nj, v);
}

template <class T, int RUN, bool FORWARD> __global__ void __launch_bounds__(256) linear_join_kernel(const Gemm g) { join_slices<T, RUN, FORWARD>(g, blockIdx.x); }

// ---- the activation's gradient and column sums ----------------------------------------------------------------------------------

struct SlopeParams {
    const void* dy;                      // [rows][ld]
    const void* y;                       // the layer's output, or NULL   (slope by its sign)
    const uint8_t* positive;             // or NULL
    const float* z;                      // or NULL
    void* s;                             // [rows][lds], or NULL: column sums only; columns behind cols become zeros
    float* partial;                      // [row blocks][cols]
    void* sums;                          // [cols], written directly when there is one row block
    int64_t rows, cols, ld, lds;
    int rows_per_block;
    int act;
    float alpha, sign;                   // sign: of the layer's gain
    float scale;
    // float16: the largest finite |dy| of each of range_blocks shares, and where the inverse of s's factor goes; or NULL
    const float* range;
    float* rescale;
    int range_blocks;
    float largest_slope;
};

// The largest finite |dy| of each workgroup's share, packets or (dy starting anywhere) elements.  One read of dy, which the slope
// kernel then finds in the last-level cache.
constexpr int kRangeBlocks = 256;

__global__ void __launch_bounds__(256) linear_range_kernel(const __half* __restrict__ dy, int64_t n, float* __restrict__ range) {
    __shared__ unsigned part[4];
    const unsigned short* bits = reinterpret_cast<const unsigned short*>(dy);
    const int64_t packets = aligned16(dy) ? n / 8 : 0, first = (int64_t)blockIdx.x * 256 + threadIdx.x, stride = (int64_t)gridDim.x * 256;
    unsigned largest = 0;                                               // magnitudes of halves are ordered as their bits are
    auto take = [&](unsigned v) { v &= 0x7fff; largest = max(largest, v < 0x7c00 ? v : 0u); };
    for (int64_t i = first; i < packets; i += stride) {
        const uint4 q = reinterpret_cast<const uint4*>(dy)[i];
        take(q.x); take(q.x >> 16); take(q.y); take(q.y >> 16); take(q.z); take(q.z >> 16); take(q.w); take(q.w >> 16);
    }
    for (int64_t i = packets * 8 + first; i < n; i += stride) take(bits[i]);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) largest = max(largest, (unsigned)__shfl_xor((int)largest, d, 64));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = largest;
    __syncthreads();
    if (threadIdx.x == 0) {
        const unsigned short all = (unsigned short)max(max(part[0], part[1]), max(part[2], part[3]));
        range[blockIdx.x] = __half2float(__builtin_bit_cast(__half, all));
    }
}

// The factor of s from all shares, the same in every workgroup (256 threads); the first one leaves its inverse for the products.
__device__ __forceinline__ float range_factor(const SlopeParams& p, float (&part)[4]) {
    float largest = (int)threadIdx.x < p.range_blocks ? p.range[threadIdx.x] : 0.f;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) largest = fmaxf(largest, __shfl_xor(largest, d, 64));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = largest;
    __syncthreads();
    float factor, inverse;
    half_range_scale(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])) * p.largest_slope, factor, inverse);
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *p.rescale = inverse;
    return factor;
}

// A workgroup: 64 * N columns (N: elements per lane, one 16-byte packet or a single one), rows_per_block rows, the waves taking
// every fourth row, UNROLL of them requested at a time (rows behind the last read it again and count as nothing).  BY: where the
// slope comes from.  Bound by HBM: 8192 x 2048 in bfloat16 by a byte an element 15 us (84 MB, 5.6 TB/s).
enum { kByNothing, kByY, kByPositive, kByZ };

template <class T, int N, int BY>
__global__ void __launch_bounds__(256) linear_slope_kernel(const SlopeParams p) {
    constexpr int UNROLL = BY == kByZ && N == 8 ? 4 : 8;
    __shared__ float part[4][64 * N];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = ((int64_t)blockIdx.x * 64 + lane) * N;
    float factor = 1.f;
    if constexpr (std::is_same_v<T, __half>) {
        __shared__ float range_part[4];
        if (p.range) factor = range_factor(p, range_part);
    }
    const int64_t r0 = (int64_t)blockIdx.y * p.rows_per_block, r1 = min(r0 + p.rows_per_block, p.rows);
    float sum[N];
#pragma unroll
    for (int e = 0; e < N; e++) sum[e] = 0.f;
    if (c >= p.cols && c < p.lds && p.s)                  // (N = 1: otherwise rows are whole packets)
        for (int64_t r = r0 + wave; r < r1; r += 4) ((T*)p.s)[r * p.lds + c] = rounded<T>(0.f);
    if (c < p.cols) {
        for (int64_t r = r0 + wave; r < r1; r += 4 * UNROLL) {
            Run<T, N> dy[UNROLL], y[UNROLL];
            Run<uint8_t, N> pos[UNROLL];
            Run<float, N> z[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; u++) {
                const int64_t row = min(r + 4 * u, r1 - 1), at = row * p.cols + c;
                dy[u] = *reinterpret_cast<const Run<T, N>*>((const T*)p.dy + row * p.ld + c);
                if constexpr (BY == kByY) y[u] = *reinterpret_cast<const Run<T, N>*>((const T*)p.y + at);
                if constexpr (BY == kByPositive) pos[u] = *reinterpret_cast<const Run<uint8_t, N>*>(p.positive + at);
                if constexpr (BY == kByZ) z[u] = *reinterpret_cast<const Run<float, N>*>(p.z + at);
            }
#pragma unroll
            for (int u = 0; u < UNROLL; u++) {
                const int64_t row = r + 4 * u;
                const bool there = row < r1;
                Run<T, N> out;
#pragma unroll
                for (int e = 0; e < N; e++) {
                    float s = Elem<T>::load(dy[u].v[e]);
                    // (relu selects its zero: a dy that is not finite stays out of the gradient of a unit that is off)
                    const float off = p.act == kActRelu ? 0.f : s * p.alpha;
                    if constexpr (BY == kByY) s = Elem<T>::load(y[u].v[e]) * p.sign > 0.f ? s : off;
                    if constexpr (BY == kByPositive) s = pos[u].v[e] ? s : off;
                    if constexpr (BY == kByZ) s *= slope_at<sizeof(T) == 2>(p.act, z[u].v[e]);
                    sum[e] += there ? s : 0.f;
                    out.v[e] = rounded<T>(s * factor);
                }
                if (p.s && there) *reinterpret_cast<Run<T, N>*>((T*)p.s + row * p.lds + c) = out;
            }
        }
    }
    if (p.sums == nullptr) return;
#pragma unroll
    for (int e = 0; e < N; e++) part[wave][lane * N + e] = sum[e];
    __syncthreads();
    for (int k = threadIdx.x; k < 64 * N; k += 256) {
        const int64_t col = (int64_t)blockIdx.x * 64 * N + k;
        if (col >= p.cols) break;
        const float total = (part[0][k] + part[1][k]) + (part[2][k] + part[3][k]);
        if (gridDim.y == 1) ((T*)p.sums)[col] = rounded<T>(total * p.scale);
        else p.partial[(int64_t)blockIdx.y * p.cols + col] = total;
    }
}

template <class T> __global__ void __launch_bounds__(1024) column_join_kernel(const ColumnJoin p) {
    __shared__ float part[16 * 64];
    join_columns<T, 16>(p, blockIdx.x, part);
}

// ---- both gradients in one launch ---------------------------------------------------------------------------------------------------
// The gradients of x and w read the same s and do not wait for each other: where both are made of 64 x 64 tiles, one launch holds
// the tiles of both and the last sums of the bias gradient, and one more joins the slices of both.  All three gradients, us with a
// launch each (few rows: linear_thin_kernel for x) and so: float32 512 -> 512 with 32 rows 13.7 and 10.7, 256 rows 21 and 14.7, 10000
// rows 107 and 100; 8192 -> 512 with 64 rows 27 and 22; bfloat16 1024 -> 1024 with 1024 rows 27 and 16.5.
struct Pair {
    Gemm x, w;
    ColumnJoin columns;
    unsigned blocks_x, blocks_w;         // then the columns' workgroups
    int x_first;                         // the longer sums start first, or they would end last and alone
};

template <class T, int MODE, int RING> __global__ void __launch_bounds__(256) linear_pair_kernel(const Pair p) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[kTileBytes<64, 64, RING>];
    const unsigned first_x = p.x_first ? 0 : p.blocks_w, first_w = p.x_first ? p.blocks_x : 0;
    if (blockIdx.x - first_x < p.blocks_x) gemm_tile<T, 64, 64, 2, 2, true, false, MODE, RING>(p.x, blockIdx.x - first_x, smem);
    else if (blockIdx.x - first_w < p.blocks_w) gemm_tile<T, 64, 64, 2, 2, false, false, MODE, RING>(p.w, blockIdx.x - first_w, smem);
    else join_columns<T, 4>(p.columns, blockIdx.x - p.blocks_x - p.blocks_w, reinterpret_cast<float*>(smem));
}

template <class T> __device__ __forceinline__ void join_slices_either(const Gemm& g, unsigned block) {
    if (g.whole) join_slices<T, 4, false>(g, block);
    else join_slices<T, 1, false>(g, block);
}

template <class T> __global__ void __launch_bounds__(256) linear_pair_join_kernel(const Pair p) {       // blocks_x, blocks_w: of this launch
    if (blockIdx.x < p.blocks_x) join_slices_either<T>(p.x, blockIdx.x);
    else join_slices_either<T>(p.w, blockIdx.x - p.blocks_x);
}

// ---- operands whose rows are not whole packets ------------------------------------------------------------------------------------
// Copies with rows of whole aligned packets, zeros behind the last element: two passes over an operand, and from there on the tiles
// travel to LDS directly and not by way of registers, and may be large ones.  Forward / gradients of x / of w in us, without and with:
//   float16  1000 x 771 -> 1025    17.2 / 17.8 / 16.8      16.6 / 14.8 / 15.6 (the last two together share one launch for the copies)
//   float32  1000 x 771 -> 1025    42.8 / 39.8 / 36.6      40.5 / 31.6 / 31.9
//   float16  2047 x 2049 -> 2051   74 / 75 / 68            59 / 52 / 49
//   bfloat16 8192 x 4095 -> 4097   741 / 680 / 775         322 / 272 / 357
//   float32  64 x 8191 -> 511      19.0 / 19.4 / 13.0      23.1 / 19.8 / 14.9
// so products from 2^29 terms on are laid out so, smaller ones are not.
struct PackParams {
    struct { const void* src; void* dst; int64_t ld, rows, cols, packets; } m[3];      // packets: per row
    int64_t first[4];                    // number of packets of the matrices before
};

template <class T> __global__ void __launch_bounds__(256) linear_pack_kernel(const PackParams p) {
    constexpr int E = 16 / (int)sizeof(T);
    const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (k >= p.first[3]) return;
    const int which = k >= p.first[2] ? 2 : k >= p.first[1] ? 1 : 0;
    const auto& m = p.m[which];
    const int64_t at = k - p.first[which];
    const int64_t row = (uint64_t)at >> 32 ? at / m.packets : (uint32_t)at / (uint32_t)m.packets, c = (at - row * m.packets) * E;
    const T* src = (const T*)m.src + row * m.ld + c;
    Pack<T> q;
    if (c + E <= m.cols) {
        const uint4 raw = Loose<T>::load(src);
        __builtin_memcpy(&q, &raw, 16);
    } else {
#pragma unroll
        for (int e = 0; e < E; e++) q.v[e] = c + e < m.cols ? src[e] : rounded<T>(0.f);
    }
    store_pack((T*)m.dst + (row * m.packets) * E + c, q);
}

// ---- host -------------------------------------------------------------------------------------------------------------------------

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// Rows per workgroup of the slope kernel: 32, doubled up to 256 while more than 2048 workgroups remain (fewer partial sums), or
// all rows up to 64.
int slope_rows(int64_t rows, int64_t cols) {
    if (rows <= 64) return 64;
    int per = 32;
    while (per < 256 && (rows + per - 1) / per * ((cols + 255) / 256) > 2048) per *= 2;
    while ((rows + per - 1) / per > 65535) per *= 2;
    return per;
}

int64_t slope_blocks(int64_t rows, int64_t cols) { return rows == 0 ? 0 : (rows + slope_rows(rows, cols) - 1) / slope_rows(rows, cols); }

// columns: where given, receives the last sums over the row blocks instead of their launch (no blocks: there are none to make).
template <class T> int run_slope(SlopeParams p, hipStream_t stream, const char* what, ColumnJoin* columns = nullptr) {
    if (columns) columns->blocks = 0;
    if (p.cols == 0) return SG_OK;
    p.rows_per_block = slope_rows(p.rows, p.cols);
    constexpr int N = Pack<T>::N;
    const bool packed = p.cols % N == 0 && p.ld % N == 0 && aligned16(p.dy) && aligned16(p.y) && aligned16(p.s) && aligned16(p.z) &&
                        reinterpret_cast<uintptr_t>(p.positive) % N == 0;
    const int n = packed ? N : 1;
    if (p.s == nullptr || p.lds < p.cols) p.lds = p.cols;
    const int64_t bx = (p.lds + 64 * n - 1) / (64 * n), by = p.rows == 0 ? 1 : slope_blocks(p.rows, p.cols);
    SG_REQUIRE(bx <= INT32_MAX && by <= 65535, SG_ERR_INVALID_ARGUMENT, "%s: too many elements", what);
    const dim3 grid((unsigned)bx, (unsigned)by);
#define SG_SLOPE(BY)                                                                                                    \
    do {                                                                                                                \
        if (packed) hipLaunchKernelGGL((linear_slope_kernel<T, N, BY>), grid, dim3(256), 0, stream, p);                 \
        else hipLaunchKernelGGL((linear_slope_kernel<T, 1, BY>), grid, dim3(256), 0, stream, p);                        \
    } while (0)
    if (p.y) SG_SLOPE(kByY);
    else if (p.positive) SG_SLOPE(kByPositive);
    else if (p.z) SG_SLOPE(kByZ);
    else SG_SLOPE(kByNothing);
#undef SG_SLOPE
    if (p.sums && by > 1) {
        const ColumnJoin join{p.partial, p.sums, p.cols, (int)by, p.scale};
        if (columns) *columns = join;
        else hipLaunchKernelGGL((column_join_kernel<T>), dim3((unsigned)((p.cols + 63) / 64)), dim3(1024), 0, stream, join);
    }
    return check_launch(what);
}

struct Shape {                            // workgroup tile and slices of one product
    bool thin = false;
    int tile = 0;
    int tiles_i = 0, tiles_j = 0, slices = 1, slice_steps = 1;
    size_t partial_bytes = 0;
};

// Whether linear_thin_kernel covers a product: few rows, a sum of at most 16 turns of its eight waves, packets.
bool thin_fits(int dtype, bool rows_b, int64_t ni, int64_t nj, int64_t np) {
    const int e = dtype == SG_F32 ? 4 : 8;
    return ni <= 32 && np <= 16 * 8 * 4 * e && np % e == 0 && (rows_b || (dtype == SG_F32 && nj % 2 == 0));
}

// The tile and the number of slices with the least predicted time.  Measured on MI355X, us per step (128 bytes along p) of a
// workgroup that has a CU to itself / of each of several that share one, by the number of "columns" operands, and us for the ends
// of a tile (first copies, epilogue) that nothing overlaps:
//   16-bit  64 x 64: 0.22 / 0.19 (columns 0.20, 0.21), 0.4      128 x 128: 0.56 / 0.43 (two columns 0.46), 1      256 x 256: 1.35, 10
//   float32 64 x 64: 0.46 / 0.46, whichever, 0.4                 (a 128 x 128 tile takes four times that: not built)
// 3 us for a launch; slices cost a second launch and a round trip of their float32 sums at 6 TB/s.
// 1024^3 in bfloat16: 64 x 64 tiles 6.5 us, 128 x 128 10; 2048^3: 27, 21 and (256 x 256) 46; 4096^3: 190, 113 and 99 (1390 TFLOP/s); a
// weight gradient of 2048 x 2048 over 8192 rows: 256 x 256 in four slices 75, whole 160, 128 x 128 73.
Shape shape_of(int dtype, int columns, int64_t ni, int64_t nj, int64_t np) {
    struct Kind { int tile; double alone[3], shared[3], ends; };
    static const Kind kinds[] = {{64, {0.22, 0.22, 0.22}, {0.19, 0.20, 0.21}, 0.4}, {128, {0.56, 0.56, 0.56}, {0.43, 0.43, 0.46}, 1.0},
                                 {256, {1.35, 1.35, 1.35}, {1.35, 1.35, 1.35}, 10.0}};
    static const Kind kinds32[] = {{64, {0.46, 0.46, 0.46}, {0.46, 0.46, 0.46}, 0.4}};
    Shape best;
    best.thin = columns < 2 && thin_fits(dtype, columns == 0, ni, nj, np);
    const int bk = dtype == SG_F32 ? 32 : 64;
    const int64_t steps = np <= 0 ? 1 : (np + bk - 1) / bk;
    double best_us = 0;
    for (int k = 0; k < (dtype == SG_F32 ? 1 : 3); k++) {
        const Kind& kind = dtype == SG_F32 ? kinds32[k] : kinds[k];
        const int64_t ti = (ni + kind.tile - 1) / kind.tile, tj = (nj + kind.tile - 1) / kind.tile;
        for (int64_t slices = 1; slices <= 64 && (slices == 1 || 2 * slices <= steps); slices = slices < 4 ? slices + 1 : slices * 3 / 2) {
            const int64_t each = (steps + slices - 1) / slices, used = (steps + each - 1) / each;
            const int64_t per_cu = (ti * tj * used + 255) / 256;
            const double step = std::max(kind.alone[columns], kind.shared[columns] * (double)per_cu);
            const double us = 3 + (double)each * step + kind.ends * (double)per_cu + (used > 1 ? 4 + (double)used * ni * nj * 8 / 6e6 : 0);
            if (best.tile == 0 || us < best_us) {
                best_us = us;
                best.tile = kind.tile;
                best.tiles_i = (int)ti;
                best.tiles_j = (int)tj;
                best.slices = (int)used;
                best.slice_steps = (int)each;
            }
        }
    }
    if (best.slices > 1) best.partial_bytes = up256((size_t)best.slices * ni * nj * 4);
    return best;
}

// Steps in LDS for 64 x 64 tiles.  Three of them let a copy take two steps, but only three workgroups fit on a CU, two let five.
// 16-bit, us with two / three: 1024 x 1024 over 4096 rows (256 tiles of 64 steps) 29.3 / 17.6, 300 x 4096 -> 4096 (320 of 64) 30 / 23,
// 6000 x 768 -> 768 (1128 of 12) 16.9 / 15.7, 16384 x 256 -> 1024 (4096 of 4) 22.4 / 25.2: three for sums of eight steps or more.
// float32, whose steps take long enough: 10000 x 512 -> 512 44 / 46, two.
template <class T> bool three_steps(const Gemm& g) { return sizeof(T) == 2 && g.slice_steps >= 8; }

template <class T, int TILE, bool RA, bool RB, int MODE> void launch_gemm(const Gemm& g, hipStream_t stream) {
    const dim3 grid((unsigned)((int64_t)g.tiles_i * g.tiles_j * g.slices));
    if constexpr (TILE == 64 && MODE == kDirect && sizeof(T) == 2) {
        if (three_steps<T>(g)) {
            hipLaunchKernelGGL((linear_gemm_kernel<T, TILE, TILE, 2, 2, RA, RB, MODE, 3>), grid, dim3(256), 0, stream, g);
            return;
        }
    }
    hipLaunchKernelGGL((linear_gemm_kernel<T, TILE, TILE, 2, 2, RA, RB, MODE, 2>), grid, dim3(256), 0, stream, g);
}

// How a product's operands can travel, and the tiles that follow from it.
struct Route {
    bool thin = false, direct = false, is_short = false;
    int tile = 0;
};

template <class T, bool RA, bool RB> int route_gemm(Gemm& g, const Shape& s, Route& r, const char* what) {
    constexpr int ES = sizeof(T), E = 16 / ES;
    g.tiles_i = s.tiles_i; g.tiles_j = s.tiles_j; g.slices = s.slices; g.slice_steps = s.slice_steps;
    // offsets within a tile's lines are 32-bit
    SG_REQUIRE((g.lda + 1) * ES * 256 < (int64_t)kOutside && (g.ldb + 1) * ES * 256 < (int64_t)kOutside, SG_ERR_UNSUPPORTED,
               "%s: rows of %lld / %lld elements are too long", what, (long long)g.lda, (long long)g.ldb);
    r.direct = aligned16(g.a) && aligned16(g.b) && g.lda % E == 0 && g.ldb % E == 0 && ((RA ? g.np : g.ni) % E == 0 || g.a_padded) &&
               ((RB ? g.np : g.nj) % E == 0 || g.b_padded);
    g.whole = runs_aligned<T>(g);
    r.thin = RA && (RB || ES == 4) && s.thin && aligned16(g.a) && g.lda % E == 0 &&
             (RB ? aligned16(g.b) && g.ldb % E == 0 : reinterpret_cast<uintptr_t>(g.b) % 8 == 0 && g.ldb % 2 == 0);
    // (operands that travel by way of registers are those of small products: others are copied into packets first, but for a dy of a
    // linear layer that starts between packets)
    r.tile = r.direct ? s.tile : 64;
    if (r.tile != s.tile) {
        g.tiles_i = (int)((g.ni + 63) / 64);
        g.tiles_j = (int)((g.nj + 63) / 64);
    }
    SG_REQUIRE((int64_t)g.tiles_i * g.tiles_j * g.slices <= INT32_MAX, SG_ERR_INVALID_ARGUMENT, "%s: too many elements", what);
    r.is_short = (RA ? g.np : g.ni) < E || (RB ? g.np : g.nj) < E;
    return SG_OK;
}

int64_t join_blocks(const Gemm& g) { return g.slices > 1 ? (g.ni * g.nj / (g.whole ? 4 : 1) + 255) / 256 : 0; }

template <class T, bool RA, bool RB> int run_gemm(Gemm g, const Shape& s, hipStream_t stream, const char* what) {
    if (g.ni == 0 || g.nj == 0) return SG_OK;
    Route r;
    const int rc = route_gemm<T, RA, RB>(g, s, r, what);
    if (rc != SG_OK) return rc;
    if constexpr (RA && (RB || sizeof(T) == 4)) {
        if (r.thin) {
            const int cols = RB ? 16 : 32;
            const dim3 grid((unsigned)((g.nj + cols - 1) / cols));
            if (g.ni <= 16) hipLaunchKernelGGL((linear_thin_kernel<T, 1, RB>), grid, dim3(512), 0, stream, g);
            else hipLaunchKernelGGL((linear_thin_kernel<T, 2, RB>), grid, dim3(512), 0, stream, g);
            return check_launch(what);
        }
    }
    if constexpr (sizeof(T) == 2) {
        if (r.tile == 256) launch_gemm<T, 256, RA, RB, kDirect>(g, stream);
        if (r.tile == 128) launch_gemm<T, 128, RA, RB, kDirect>(g, stream);
    }
    if (r.tile == 64) {
        if (r.direct) launch_gemm<T, 64, RA, RB, kDirect>(g, stream);
        else if (r.is_short) launch_gemm<T, 64, RA, RB, kShort>(g, stream);
        else launch_gemm<T, 64, RA, RB, kLoose>(g, stream);
    }
    const int64_t blocks = join_blocks(g);
    SG_REQUIRE(blocks <= INT32_MAX, SG_ERR_INVALID_ARGUMENT, "%s: too many elements", what);
    if (blocks && g.whole) hipLaunchKernelGGL((linear_join_kernel<T, 4, RA && RB>), dim3((unsigned)blocks), dim3(256), 0, stream, g);
    else if (blocks) hipLaunchKernelGGL((linear_join_kernel<T, 1, RA && RB>), dim3((unsigned)blocks), dim3(256), 0, stream, g);
    return check_launch(what);
}

// The two products of the backward pass (w's partial sums lie behind x's) and the columns that run_slope left.
template <class T> int run_pair(Gemm x, const Shape& sx, Gemm w, const Shape& sw, const ColumnJoin& columns, hipStream_t stream, const char* what) {
    Route rx, rw;
    int rc = route_gemm<T, true, false>(x, sx, rx, what);
    if (rc == SG_OK) rc = route_gemm<T, false, false>(w, sw, rw, what);
    if (rc != SG_OK) return rc;
    Pair p{x, w, columns, (unsigned)(x.tiles_i * x.tiles_j * x.slices), (unsigned)(w.tiles_i * w.tiles_j * w.slices), x.slice_steps >= w.slice_steps};
    const bool direct = rx.direct && rw.direct, loose = !rx.is_short && !rw.is_short;
    if (rx.tile != 64 || rw.tile != 64 || !(direct || loose)) {
        if (columns.blocks)
            hipLaunchKernelGGL((column_join_kernel<T>), dim3((unsigned)((columns.cols + 63) / 64)), dim3(1024), 0, stream, columns);
        rc = run_gemm<T, true, false>(x, sx, stream, what);
        return rc != SG_OK ? rc : run_gemm<T, false, false>(w, sw, stream, what);
    }
    const int64_t blocks = (int64_t)p.blocks_x + p.blocks_w + (columns.blocks ? (columns.cols + 63) / 64 : 0);
    SG_REQUIRE(blocks <= INT32_MAX, SG_ERR_INVALID_ARGUMENT, "%s: too many elements", what);
    const dim3 grid((unsigned)blocks);
    const bool three = direct && three_steps<T>(x) && three_steps<T>(w);
    if constexpr (sizeof(T) == 2) {
        if (three) hipLaunchKernelGGL((linear_pair_kernel<T, kDirect, 3>), grid, dim3(256), 0, stream, p);
    }
    if (direct && !three) hipLaunchKernelGGL((linear_pair_kernel<T, kDirect, 2>), grid, dim3(256), 0, stream, p);
    if (!direct) hipLaunchKernelGGL((linear_pair_kernel<T, kLoose, 2>), grid, dim3(256), 0, stream, p);
    const int64_t jx = join_blocks(x), jw = join_blocks(w);
    SG_REQUIRE(jx + jw <= INT32_MAX, SG_ERR_INVALID_ARGUMENT, "%s: too many elements", what);
    p.blocks_x = (unsigned)jx;
    if (jx + jw) hipLaunchKernelGGL((linear_pair_join_kernel<T>), dim3((unsigned)(jx + jw)), dim3(256), 0, stream, p);
    return check_launch(what);
}

int check(const sg_linear_params* p, const char* what) {
    SG_REQUIRE(p != nullptr, SG_ERR_NULL_POINTER, "params is NULL");
    SG_REQUIRE(p->dtype == SG_F32 || p->dtype == SG_F16 || p->dtype == SG_BF16, SG_ERR_UNSUPPORTED, "%s: dtype %d (float32, float16 or bfloat16)", what, p->dtype);
    SG_REQUIRE(p->act >= kActLinear && p->act <= kActSwish, SG_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", what, p->act);
    SG_REQUIRE(p->m >= 0 && p->n >= 0 && p->k >= 0 && p->m <= INT32_MAX && p->n <= INT32_MAX && p->k <= INT32_MAX, SG_ERR_INVALID_ARGUMENT,
               "%s: sizes %lld, %lld, %lld", what, (long long)p->m, (long long)p->n, (long long)p->k);
    SG_REQUIRE(p->ldx >= p->k && p->ldw >= p->k && p->ldr >= 0, SG_ERR_INVALID_ARGUMENT, "%s: row strides are smaller than rows", what);
    SG_REQUIRE(p->m == 0 || p->n == 0 || p->k == 0 || (p->x && p->w), SG_ERR_NULL_POINTER, "%s: x or w is NULL", what);
    return SG_OK;
}

bool piecewise(int act) { return act == kActRelu || act == kActLrelu; }

// A bound of |act'|.
float largest_slope(int act, float alpha) {
    switch (act) {
        case kActLrelu: return std::max(1.f, std::fabs(alpha));
        case kActSelu: return kSeluScale * kSeluAlpha;
        case kActSwish: return 1.1f;
        default: return 1.f;
    }
}

constexpr double kCopiedFrom = (double)(1 << 29);        // terms of a product; measured above

// An operand as the products read it: where it lies, or its copy in the workspace.
struct Operand {
    const void* p = nullptr;
    int64_t ld = 0;
    int padded = 0;
    size_t at = 0, bytes = 0;            // of the copy; none: 0 bytes
};

int elements(int dtype) { return dtype == SG_F32 ? 4 : 8; }
int64_t whole_packets(int64_t cols, int dtype) { return (cols + elements(dtype) - 1) / elements(dtype) * elements(dtype); }

// x and w of a layer; `at`: where in the workspace copies may lie (moved on behind them).  Products from 2^29 terms on.
void place_operands(const sg_linear_params& p, size_t& at, Operand& x, Operand& w) {
    const int e = elements(p.dtype);
    const bool large = (double)p.m * p.n * p.k >= kCopiedFrom;
    auto place = [&](Operand& o, const void* src, int64_t ld, int64_t rows) {
        o.p = src;
        o.ld = ld;
        if (!large || (aligned16(src) && ld % e == 0 && p.k % e == 0)) return;
        o.ld = whole_packets(p.k, p.dtype);
        o.padded = 1;
        o.at = at;
        o.bytes = up256((size_t)rows * o.ld * (16 / e));
        at += o.bytes;
    };
    place(x, p.x, p.ldx, p.m);
    place(w, p.w, p.ldw, p.n);
}

template <class T> int run_pack(PackParams& q, int count, hipStream_t stream, const char* what) {
    for (int i = 0; i < 3; i++) q.first[i + 1] = q.first[i] + (i < count ? q.m[i].rows * q.m[i].packets : 0);
    if (q.first[3] == 0) return SG_OK;
    SG_REQUIRE((q.first[3] + 255) / 256 <= INT32_MAX, SG_ERR_INVALID_ARGUMENT, "%s: too many elements", what);
    hipLaunchKernelGGL((linear_pack_kernel<T>), dim3((unsigned)((q.first[3] + 255) / 256)), dim3(256), 0, stream, q);
    return check_launch(what);
}

// Adds an operand's copy to the launch; from then on it is read there.
void add_pack(PackParams& q, int& count, Operand& o, char* ws, int64_t rows, int64_t cols, int64_t ld, int dtype) {
    if (o.bytes == 0) return;
    q.m[count].src = o.p; q.m[count].dst = ws + o.at;
    q.m[count].ld = ld; q.m[count].rows = rows; q.m[count].cols = cols;
    q.m[count].packets = o.ld / elements(dtype);
    count++;
    o.p = ws + o.at;
}

struct ForwardPlan {
    Shape y;
    Operand x, w;
    size_t total = 0;                     // the slices' sums come first
};

ForwardPlan plan_forward(const sg_linear_params& p) {
    ForwardPlan f;
    f.y = shape_of(p.dtype, 0, p.m, p.n, p.k);
    f.total = f.y.partial_bytes;
    place_operands(p, f.total, f.x, f.w);
    return f;
}

struct BackwardPlan {
    Shape dx, dw;
    Operand x, w, s;                      // s: the activation's gradient, or dy (copied only for its own n)
    bool ranged = false;                  // s times a power of two (float16; relu's s is dy or zero)
    size_t sums = 0, range = 0, partial = 0, partial_w = 0, total = 0;
};

BackwardPlan plan_backward(const sg_linear_params& p) {
    BackwardPlan b;
    const int e = elements(p.dtype);
    size_t at = 0;
    b.s.ld = p.n;
    const bool large = (double)p.m * p.n * p.k >= kCopiedFrom;
    if (p.act != kActLinear || (large && p.n % e != 0)) {
        b.s.ld = large ? whole_packets(p.n, p.dtype) : p.n;
        b.s.padded = b.s.ld != p.n;
        b.s.bytes = up256((size_t)p.m * b.s.ld * (16 / e));
        at += b.s.bytes;
    }
    b.sums = at;
    at += up256((size_t)slope_blocks(p.m, p.n) * p.n * 4);
    b.ranged = p.dtype == SG_F16 && p.act != kActLinear && p.act != kActRelu;
    b.range = at;
    if (b.ranged) at += up256((kRangeBlocks + 1) * 4);                  // the shares' largest values, then the inverse factor
    b.dx = shape_of(p.dtype, 1, p.m, p.k, p.n);
    b.dw = shape_of(p.dtype, 2, p.n, p.k, p.m);
    b.partial = at;
    b.partial_w = at + b.dx.partial_bytes;
    at += b.dx.partial_bytes + b.dw.partial_bytes;
    place_operands(p, at, b.x, b.w);
    b.total = at;
    return b;
}

}  // namespace

}  // namespace sg

extern "C" size_t sg_linear_workspace_bytes(const sg_linear_params* p) {
    using namespace sg;
    if (check(p, "linear") != SG_OK) return 0;
    return plan_forward(*p).total;
}

extern "C" int sg_linear(const sg_linear_params* p, void* y, float* z, uint8_t* positive, void* workspace, size_t workspace_bytes, sg_stream_t stream) {
    using namespace sg;
    const int rc = check(p, "linear");
    if (rc != SG_OK) return rc;
    if (p->m == 0 || p->n == 0) return SG_OK;
    SG_REQUIRE(y != nullptr, SG_ERR_NULL_POINTER, "linear: y is NULL");
    SG_REQUIRE(p->residual == nullptr || p->ldr >= p->n, SG_ERR_INVALID_ARGUMENT, "linear: the residual's row stride is smaller than its rows");
    ForwardPlan f = plan_forward(*p);
    SG_REQUIRE(f.total == 0 || (workspace && workspace_bytes >= f.total && aligned16(workspace)), SG_ERR_INVALID_ARGUMENT,
               "linear: needs %zu bytes of aligned workspace", f.total);
    PackParams q{};
    int copies = 0;
    add_pack(q, copies, f.x, (char*)workspace, p->m, p->k, p->ldx, p->dtype);
    add_pack(q, copies, f.w, (char*)workspace, p->n, p->k, p->ldw, p->dtype);
    if (copies) {
        int done = SG_OK;
        SG_DISPATCH_16_32(p->dtype, done = run_pack<T>(q, copies, (hipStream_t)stream, "sg_linear"));
        if (done != SG_OK) return done;
    }
    Gemm g{};
    g.a = f.x.p; g.lda = f.x.ld; g.a_padded = f.x.padded;
    g.b = f.w.p; g.ldb = f.w.ld; g.b_padded = f.w.padded;
    g.ni = p->m; g.nj = p->n; g.np = p->k;
    g.partial = (float*)workspace;
    g.out = y; g.scale = p->w_gain;
    g.bias = p->b; g.b_gain = p->b_gain;
    g.residual = p->residual; g.ldr = p->ldr;
    g.z = z; g.positive = positive;
    g.act = p->act; g.alpha = p->alpha; g.gain = p->gain;
    SG_DISPATCH_16_32(p->dtype, return (run_gemm<T, true, true>(g, f.y, (hipStream_t)stream, "sg_linear")));
    return SG_OK;
}

extern "C" size_t sg_linear_backward_workspace_bytes(const sg_linear_params* p) {
    using namespace sg;
    if (check(p, "linear_backward") != SG_OK) return 0;
    return plan_backward(*p).total;
}

extern "C" int sg_linear_backward(const sg_linear_params* p, const void* dy, const void* y, const float* z, const uint8_t* positive, void* dx, void* dw,
                                  void* db, void* workspace, size_t workspace_bytes, sg_stream_t stream_) {
    using namespace sg;
    const int rc = check(p, "linear_backward");
    if (rc != SG_OK) return rc;
    hipStream_t stream = (hipStream_t)stream_;
    const bool any = p->m > 0 && p->n > 0;
    SG_REQUIRE(!any || dy != nullptr, SG_ERR_NULL_POINTER, "linear_backward: dy is NULL");
    const int given = (y != nullptr) + (z != nullptr) + (positive != nullptr);
    SG_REQUIRE(!any || given == (p->act == kActLinear ? 0 : 1), SG_ERR_INVALID_ARGUMENT, "linear_backward: activation %d takes %s of y, z, positive", p->act,
               p->act == kActLinear ? "none" : "one");
    SG_REQUIRE(!any || p->act == kActLinear || (z != nullptr) != piecewise(p->act), SG_ERR_INVALID_ARGUMENT,
               "linear_backward: activation %d takes %s", p->act, piecewise(p->act) ? "y or positive" : "z");
    BackwardPlan plan = plan_backward(*p);
    SG_REQUIRE(plan.total == 0 || (workspace && workspace_bytes >= plan.total && aligned16(workspace)), SG_ERR_INVALID_ARGUMENT,
               "linear_backward: needs %zu bytes of aligned workspace", plan.total);
    char* ws = (char*)workspace;
    const bool own_s = p->act != kActLinear, products = any && (dx || dw);
    PackParams q{};
    int copies = 0;
    if (products) {
        if (own_s) plan.s.p = ws + plan.s.at;
        else plan.s.p = dy;
        if (!own_s) add_pack(q, copies, plan.s, ws, p->m, p->n, p->n, p->dtype);
        if (dw) add_pack(q, copies, plan.x, ws, p->m, p->k, p->ldx, p->dtype);
        if (dx) add_pack(q, copies, plan.w, ws, p->n, p->k, p->ldw, p->dtype);
    }
    if (copies) {
        int done = SG_OK;
        SG_DISPATCH_16_32(p->dtype, done = run_pack<T>(q, copies, stream, "sg_linear_backward"));
        if (done != SG_OK) return done;
    }
    ColumnJoin columns{};
    const bool pair = products && dx && dw && p->k > 0;
    if ((own_s && products) || db) {
        SlopeParams r{};
        r.dy = dy; r.y = y; r.positive = positive; r.z = z;
        r.s = own_s && products ? ws + plan.s.at : nullptr;
        r.lds = plan.s.ld;
        r.partial = (float*)(ws + plan.sums);
        r.sums = db;
        r.rows = p->m; r.cols = p->n; r.ld = p->n;
        r.act = p->act;
        r.alpha = p->alpha;
        r.sign = p->gain < 0.f ? -1.f : 1.f;
        r.scale = p->gain * p->b_gain;
        if (plan.ranged && products) {
            float* range = (float*)(ws + plan.range);
            const int64_t count = p->m * p->n;
            r.range = range;
            r.rescale = range + kRangeBlocks;
            r.range_blocks = (int)std::min<int64_t>((count + 2047) / 2048, kRangeBlocks);       // (a packet a lane, or more)
            r.largest_slope = largest_slope(p->act, p->alpha);
            hipLaunchKernelGGL(linear_range_kernel, dim3((unsigned)r.range_blocks), dim3(256), 0, stream, (const __half*)dy, count, range);
        }
        int done = SG_OK;
        SG_DISPATCH_16_32(p->dtype, done = run_slope<T>(r, stream, "sg_linear_backward", pair ? &columns : nullptr));
        if (done != SG_OK) return done;
    }
    Gemm gx{}, gw{};
    gx.scale = gw.scale = p->gain * p->w_gain;
    gx.rescale = gw.rescale = plan.ranged && products ? (const float*)(ws + plan.range) + kRangeBlocks : nullptr;
    gx.a = gw.a = plan.s.p; gx.lda = gw.lda = plan.s.ld; gx.a_padded = gw.a_padded = plan.s.padded;
    gx.partial = (float*)(ws + plan.partial);                      // [m, k] = s [m, n] w [n, k]
    gx.b = plan.w.p; gx.ldb = plan.w.ld; gx.b_padded = plan.w.padded;
    gx.ni = p->m; gx.nj = p->k; gx.np = p->n;
    gx.out = dx;
    gw.partial = (float*)(ws + plan.partial_w);                    // [n, k] = s [m, n]^T x [m, k]
    gw.b = plan.x.p; gw.ldb = plan.x.ld; gw.b_padded = plan.x.padded;
    gw.ni = p->n; gw.nj = p->k; gw.np = p->m;
    gw.out = dw;
    if (pair) {
        SG_DISPATCH_16_32(p->dtype, return run_pair<T>(gx, plan.dx, gw, plan.dw, columns, stream, "sg_linear_backward"));
    }
    int done = SG_OK;
    if (dx) SG_DISPATCH_16_32(p->dtype, done = (run_gemm<T, true, false>(gx, plan.dx, stream, "sg_linear_backward")));
    if (dw && done == SG_OK) SG_DISPATCH_16_32(p->dtype, done = (run_gemm<T, false, false>(gw, plan.dw, stream, "sg_linear_backward")));
    return done;
}

extern "C" const char* sg_linear_kernel(const sg_linear_params* p, int32_t product) {
    using namespace sg;
    static thread_local char text[96];
    if (check(p, "linear_kernel") != SG_OK || product < 0 || product > 2) return "";
    // (copies in the workspace are whole packets wherever it lies)
    auto here = [](const Operand& o) { return o.bytes ? reinterpret_cast<const void*>((uintptr_t)o.at) : o.p; };
    Gemm g{};
    Shape s;
    if (product == 0) {
        const ForwardPlan f = plan_forward(*p);
        s = f.y;
        g.a = here(f.x); g.lda = f.x.ld; g.a_padded = f.x.padded;
        g.b = here(f.w); g.ldb = f.w.ld; g.b_padded = f.w.padded;
        g.ni = p->m; g.nj = p->n; g.np = p->k;
    } else {
        const BackwardPlan b = plan_backward(*p);
        const Operand& o = product == 1 ? b.w : b.x;
        s = product == 1 ? b.dx : b.dw;
        g.lda = b.s.ld; g.a_padded = b.s.padded;
        g.b = here(o); g.ldb = o.ld; g.b_padded = o.padded;
        g.ni = product == 1 ? p->m : p->n; g.nj = p->k; g.np = product == 1 ? p->n : p->m;
    }
    Route r;
    int rc = SG_OK;
    auto route = [&](auto element) {
        using T = decltype(element);
        rc = product == 0 ? route_gemm<T, true, true>(g, s, r, "linear_kernel") : product == 1 ? route_gemm<T, true, false>(g, s, r, "linear_kernel")
                                                                                              : route_gemm<T, false, false>(g, s, r, "linear_kernel");
    };
    if (p->dtype == SG_F32) route(float());
    else if (p->dtype == SG_F16) route(__half());
    else route(__hip_bfloat16());
    if (rc != SG_OK) return "";
    if (r.thin) return "linear_thin_kernel";
    snprintf(text, sizeof text, "linear_gemm_kernel<%d, %s> %d x %d", r.tile, r.direct ? "direct" : r.is_short ? "short" : "loose", g.slices, g.slice_steps);
    return text;
}
