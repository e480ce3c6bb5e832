// Optimizer step of the training loop over a list of tensors in one launch: gradient
// sanitising (NaN -> 0, +-Inf -> +-grad_limit; reference training_loop.py:509,
// misc.nan_to_num) followed by the Adam update the reference's optimizer applies
// (torch.optim.Adam, no weight decay, no amsgrad; constructed at training_loop.py:303-312),
// and the exponential moving average of the generator weights (training_loop.py:516-523)
// as a second list operation.  Streaming kernels: every element is read and written once.
//
// The tensor table travels by value in the kernel arguments (no device-side table to
// allocate or copy): up to kMaxTensors tensors per launch, cut into blocks of
// kBlockElems elements; block_start[i] is the first block of tensor i.
#include "sg_common.h"

namespace sg {
namespace {

constexpr int kMaxTensors = SG_OPTIM_MAX_TENSORS;
constexpr int kThreads = 256;
constexpr int kBlockElems = kThreads * 16;

struct AdamTable {
    float* param[kMaxTensors];
    float* grad[kMaxTensors];
    float* exp_avg[kMaxTensors];
    float* exp_avg_sq[kMaxTensors];
    float step_size[kMaxTensors];        // lr / (1 - beta1^t)
    float sqrt_bc2[kMaxTensors];         // sqrt(1 - beta2^t)
    int64_t numel[kMaxTensors];
    int block_start[kMaxTensors + 1];
    int count;
    float beta1, beta2, eps, grad_limit;
};

struct LerpTable {
    float* dst[kMaxTensors];
    const float* src[kMaxTensors];
    int64_t numel[kMaxTensors];
    int block_start[kMaxTensors + 1];
    int count;
    float weight;                        // dst = lerp(src, dst, weight)
};

// start + weight * (end - start), in the form that is exact at the end point the weight is nearer to (the
// library's lerp; with beta1 = 0 the first moment is then the gradient itself, bit for bit)
__device__ __forceinline__ float lerp(float start, float end, float weight) {
    return (weight < 0.5f) ? start + weight * (end - start) : end - (end - start) * (1.f - weight);
}

template <class Table>
__device__ __forceinline__ int find_tensor(const Table& t, int block) {
    int lo = 0, hi = t.count - 1;        // last i with block_start[i] <= block
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.block_start[mid] <= block) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// CLIP: the gradient is multiplied by *grad_scale (a device value: min(1, max_norm / norm)) as it enters the update.  24 million
// elements: 124 us (771 MB, 6.2 TB/s: part of the gradients comes from the last-level cache), 24 more for their norm; as a pass of its own
// over the gradients the scaling would take 40.
template <bool CLIP>
__global__ void __launch_bounds__(kThreads) adam_kernel(const AdamTable t, const float* __restrict__ grad_scale) {
    const int ti = find_tensor(t, blockIdx.x);
    const int64_t n = t.numel[ti];
    float* __restrict__ p = t.param[ti];
    float* __restrict__ g = t.grad[ti];
    float* __restrict__ m = t.exp_avg[ti];
    float* __restrict__ v = t.exp_avg_sq[ti];
    const float step_size = t.step_size[ti], sqrt_bc2 = t.sqrt_bc2[ti];
    const float scale = CLIP ? *grad_scale : 1.f;
    // 16-byte accesses where the four tensors start equally far from a 16-byte boundary: the elements in front of it
    // (tensors cut from flat buffers start anywhere) go to the first block's first lanes
    const uintptr_t ap = reinterpret_cast<uintptr_t>(p), ag = reinterpret_cast<uintptr_t>(g);
    const uintptr_t am = reinterpret_cast<uintptr_t>(m), av = reinterpret_cast<uintptr_t>(v);
    const bool vec = (((ap ^ ag) | (ap ^ am) | (ap ^ av)) & 15u) == 0;
    const int lead = vec ? (int)((16u - (ap & 15u)) & 15u) / 4 : 0;
    const int block = blockIdx.x - t.block_start[ti];
    const int64_t base = lead + (int64_t)block * kBlockElems;
    auto update = [&](float& pv, float& gv, float& mv, float& vv) {
        float gs = gv;
        if (gs != gs) gs = 0.f;
        else if (gs == INFINITY) gs = t.grad_limit;
        else if (gs == -INFINITY) gs = -t.grad_limit;
        gv = gs;                                            // the sanitised gradient is what stays in .grad
        if (CLIP) gs *= scale;
        mv = lerp(mv, gs, 1.f - t.beta1);
        vv = vv * t.beta2 + gs * gs * (1.f - t.beta2);
        const float denom = sqrtf(vv) / sqrt_bc2 + t.eps;
        pv = pv - step_size * (mv / denom);
    };
    if (block == 0 && (int)threadIdx.x < lead && threadIdx.x < n) update(p[threadIdx.x], g[threadIdx.x], m[threadIdx.x], v[threadIdx.x]);
#pragma unroll
    for (int k = 0; k < kBlockElems / (kThreads * 4); k++) {
        const int64_t i = base + ((int64_t)k * kThreads + threadIdx.x) * 4;
        if (i >= n) break;
        if (vec && i + 4 <= n) {
            float4 pv = *reinterpret_cast<float4*>(p + i), gv = *reinterpret_cast<float4*>(g + i);
            float4 mv = *reinterpret_cast<float4*>(m + i), vv = *reinterpret_cast<float4*>(v + i);
            update(pv.x, gv.x, mv.x, vv.x);
            update(pv.y, gv.y, mv.y, vv.y);
            update(pv.z, gv.z, mv.z, vv.z);
            update(pv.w, gv.w, mv.w, vv.w);
            *reinterpret_cast<float4*>(p + i) = pv;
            *reinterpret_cast<float4*>(g + i) = gv;
            *reinterpret_cast<float4*>(m + i) = mv;
            *reinterpret_cast<float4*>(v + i) = vv;
        } else {
            for (int64_t j = i; j < n && j < i + 4; j++) update(p[j], g[j], m[j], v[j]);
        }
    }
}

// ---- global gradient norm ---------------------------------------------------------------------------------------
//   norm = sqrt(sum over tensors and elements of g^2),   scale = min(1, max_norm / (norm + eps))
// One read of every gradient: bound by HBM.  Squares are formed and summed in double - a conversion and a multiply-add per
// element, a fifth of what the vector unit could do while the bytes arrive - so that neither a large element's square (1e20
// in float32) nor a sum over 10^8 elements loses anything.  A block sums one chunk of one tensor in a fixed order and writes
// one double; a single block adds those in a fixed order: the result does not depend on which block ran when, and needs no
// atomics.  Chunks are whole 16-byte packets from the tensor's first 16-byte boundary on; what lies in front of it and behind
// the last whole packet (at most 7 + 7 elements) goes to the tensor's first block.  134 million bfloat16 elements in 90 tensors: 43 us
// (6.2 TB/s) and 4.6 for the single block.
constexpr int kNormTensors = 128;
constexpr int kPacketsPerPass = kThreads * 4;          // four 16-byte loads per lane in flight
constexpr int64_t kNormBlocks = 4096;                  // two rounds of eight workgroups on every CU

struct NormTable {
    void* grad[kNormTensors];
    int64_t numel[kNormTensors];
    int block_start[kNormTensors + 1];
    uint8_t dtype[kNormTensors];
    int count;
    int passes;                                        // packets per block / kPacketsPerPass
    float grad_limit;                                  // > 0: NaN -> 0, +-Inf -> +-grad_limit, as adam_kernel does
};

struct Span {                                          // a tensor's elements as lead | packets | rest
    int lead;
    int64_t packets;
    __host__ __device__ Span(const void* p, int64_t n, int esize) {
        const int64_t to_boundary = (int64_t)((16u - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / esize;
        lead = (int)(to_boundary < n ? to_boundary : n);
        packets = (n - lead) / (16 / esize);
    }
};

__device__ __forceinline__ float sanitised(float g, float limit) {
    if (limit > 0.f) {
        if (g != g) g = 0.f;
        else if (g == INFINITY) g = limit;
        else if (g == -INFINITY) g = -limit;
    }
    return g;
}

// Sum of a double over the block's lanes in a fixed order; valid in thread 0.  WAVES waves.
template <int WAVES> __device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[WAVES];
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, kWave);
    if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    v = 0;
    if (threadIdx.x == 0)
        for (int i = 0; i < WAVES; i++) v += part[i];
    return v;
}

template <class T> __device__ __forceinline__ double squares(const T* __restrict__ g, int64_t n, int block, int passes, float limit) {
    constexpr int N = Pack<T>::N;
    const Span span(g, n, sizeof(T));
    const Pack<T>* __restrict__ body = reinterpret_cast<const Pack<T>*>(g + span.lead);
    const int64_t first = (int64_t)block * passes * kPacketsPerPass;
    double sum[4] = {0, 0, 0, 0};
    for (int pass = 0; pass < passes; pass++) {
        const int64_t at = first + (int64_t)pass * kPacketsPerPass + threadIdx.x;
        if (at - threadIdx.x >= span.packets) break;
        uint4 raw[4];
#pragma unroll
        for (int u = 0; u < 4; u++) raw[u] = load16_or_zero(at + u * kThreads < span.packets, body + at + u * kThreads);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            Pack<T> v;
            __builtin_memcpy(&v, &raw[u], 16);
#pragma unroll
            for (int j = 0; j < N; j++) {
                const double d = (double)sanitised(Elem<T>::load(v.v[j]), limit);
                sum[u] = fma(d, d, sum[u]);
            }
        }
    }
    if (block == 0) {
        const int64_t rest = span.lead + span.packets * N;
        int64_t i = -1;
        if ((int)threadIdx.x < span.lead) i = threadIdx.x;
        else if (threadIdx.x >= 64 && rest + threadIdx.x - 64 < n) i = rest + threadIdx.x - 64;
        if (i >= 0) {
            const double d = (double)sanitised(Elem<T>::load(g[i]), limit);
            sum[0] = fma(d, d, sum[0]);
        }
    }
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

__global__ void __launch_bounds__(kThreads) grad_norm_kernel(const NormTable t, double* __restrict__ partial) {
    const int ti = find_tensor(t, blockIdx.x);
    const int block = blockIdx.x - t.block_start[ti];
    double sum;
    switch (t.dtype[ti]) {
        case SG_F32: sum = squares((const float*)t.grad[ti], t.numel[ti], block, t.passes, t.grad_limit); break;
        case SG_F16: sum = squares((const __half*)t.grad[ti], t.numel[ti], block, t.passes, t.grad_limit); break;
        default: sum = squares((const __hip_bfloat16*)t.grad[ti], t.numel[ti], block, t.passes, t.grad_limit); break;
    }
    sum = block_sum<kThreads / kWave>(sum);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// out[0] = norm, out[1] = min(1, max_norm / (norm + eps)).  A NaN norm gives a NaN scale.
__global__ void __launch_bounds__(1024) norm_finish_kernel(const double* __restrict__ partial, int count, float max_norm, float eps,
                                                           float* __restrict__ out) {
    double sum = 0;
    for (int i = threadIdx.x; i < count; i += 1024) sum += partial[i];
    sum = block_sum<1024 / kWave>(sum);
    if (threadIdx.x == 0) {
        const float norm = (float)sqrt(sum);
        const float scale = max_norm / (norm + eps);
        out[0] = norm;
        out[1] = scale > 1.f ? 1.f : scale;
    }
}

template <class T> __device__ __forceinline__ void scale_chunk(T* __restrict__ g, int64_t n, int block, int passes, float scale) {
    constexpr int N = Pack<T>::N;
    const Span span(g, n, sizeof(T));
    Pack<T>* __restrict__ body = reinterpret_cast<Pack<T>*>(g + span.lead);
    const int64_t first = (int64_t)block * passes * kPacketsPerPass;
    for (int pass = 0; pass < passes; pass++) {
        const int64_t at = first + (int64_t)pass * kPacketsPerPass + threadIdx.x;
        if (at - threadIdx.x >= span.packets) break;
        uint4 raw[4];
#pragma unroll
        for (int u = 0; u < 4; u++) raw[u] = load16_or_zero(at + u * kThreads < span.packets, body + at + u * kThreads);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            Pack<T> v;
            __builtin_memcpy(&v, &raw[u], 16);
#pragma unroll
            for (int j = 0; j < N; j++) v.v[j] = Elem<T>::store(Elem<T>::load(v.v[j]) * scale);
            if (at + u * kThreads < span.packets) body[at + u * kThreads] = v;
        }
    }
    if (block == 0) {
        const int64_t rest = span.lead + span.packets * N;
        int64_t i = -1;
        if ((int)threadIdx.x < span.lead) i = threadIdx.x;
        else if (threadIdx.x >= 64 && rest + threadIdx.x - 64 < n) i = rest + threadIdx.x - 64;
        if (i >= 0) g[i] = Elem<T>::store(Elem<T>::load(g[i]) * scale);
    }
}

// A scale of exactly one leaves every element as it is (x * 1 = x, NaN included): nothing is read or written then.
__global__ void __launch_bounds__(kThreads) grad_scale_kernel(const NormTable t, const float* __restrict__ grad_scale) {
    const float scale = *grad_scale;
    if (scale == 1.f) return;
    const int ti = find_tensor(t, blockIdx.x);
    const int block = blockIdx.x - t.block_start[ti];
    switch (t.dtype[ti]) {
        case SG_F32: scale_chunk((float*)t.grad[ti], t.numel[ti], block, t.passes, scale); break;
        case SG_F16: scale_chunk((__half*)t.grad[ti], t.numel[ti], block, t.passes, scale); break;
        default: scale_chunk((__hip_bfloat16*)t.grad[ti], t.numel[ti], block, t.passes, scale); break;
    }
}

__global__ void __launch_bounds__(kThreads) lerp_kernel(const LerpTable t) {
    const int ti = find_tensor(t, blockIdx.x);
    const int64_t base = (int64_t)(blockIdx.x - t.block_start[ti]) * kBlockElems;
    const int64_t n = t.numel[ti];
    float* __restrict__ d = t.dst[ti];
    const float* __restrict__ s = t.src[ti];
    const bool vec = ((reinterpret_cast<uintptr_t>(d) | reinterpret_cast<uintptr_t>(s)) & 15u) == 0;
    const float w = t.weight;
#pragma unroll
    for (int k = 0; k < kBlockElems / (kThreads * 4); k++) {
        const int64_t i = base + ((int64_t)k * kThreads + threadIdx.x) * 4;
        if (i >= n) break;
        if (vec && i + 4 <= n) {
            float4 dv = *reinterpret_cast<float4*>(d + i);
            const float4 sv = *reinterpret_cast<const float4*>(s + i);
            dv.x = lerp(sv.x, dv.x, w); dv.y = lerp(sv.y, dv.y, w); dv.z = lerp(sv.z, dv.z, w); dv.w = lerp(sv.w, dv.w, w);
            *reinterpret_cast<float4*>(d + i) = dv;
        } else {
            for (int64_t j = i; j < n && j < i + 4; j++) d[j] = lerp(s[j], d[j], w);
        }
    }
}

}  // namespace
}  // namespace sg

extern "C" int sg_adam_step(const sg_adam_params* p, sg_stream_t stream) {
    using namespace sg;
    SG_REQUIRE(p != nullptr, SG_ERR_NULL_POINTER, "params is NULL");
    SG_REQUIRE(p->count >= 0 && p->count <= kMaxTensors, SG_ERR_INVALID_ARGUMENT, "adam_step: %d tensors (at most %d per call)",
               p->count, kMaxTensors);
    SG_REQUIRE(p->beta1 >= 0.f && p->beta1 < 1.f && p->beta2 >= 0.f && p->beta2 < 1.f && p->eps >= 0.f && p->grad_limit > 0.f,
               SG_ERR_INVALID_ARGUMENT, "adam_step: betas must lie in [0, 1), eps >= 0, grad_limit > 0");
    if (p->count == 0) return SG_OK;
    SG_REQUIRE(p->tensors != nullptr, SG_ERR_NULL_POINTER, "adam_step: tensors is NULL");
    AdamTable t;
    t.count = 0;
    t.beta1 = p->beta1; t.beta2 = p->beta2; t.eps = p->eps; t.grad_limit = p->grad_limit;
    int64_t blocks = 0;
    for (int i = 0; i < p->count; i++) {
        const sg_adam_tensor& e = p->tensors[i];
        SG_REQUIRE(e.numel >= 0 && e.step >= 1, SG_ERR_INVALID_ARGUMENT, "adam_step: tensor %d: numel %lld, step %d", i,
                   (long long)e.numel, e.step);
        if (e.numel == 0) continue;
        SG_REQUIRE(e.param && e.grad && e.exp_avg && e.exp_avg_sq, SG_ERR_NULL_POINTER, "adam_step: tensor %d has a NULL pointer", i);
        const int k = t.count++;
        t.param[k] = e.param; t.grad[k] = e.grad; t.exp_avg[k] = e.exp_avg; t.exp_avg_sq[k] = e.exp_avg_sq;
        // bias corrections in double, as the library computes them on the host
        const double bc1 = 1.0 - pow((double)p->beta1, (double)e.step), bc2 = 1.0 - pow((double)p->beta2, (double)e.step);
        t.step_size[k] = (float)((double)p->lr / bc1);
        t.sqrt_bc2[k] = (float)sqrt(bc2);
        t.numel[k] = e.numel;
        t.block_start[k] = (int)blocks;
        blocks += (e.numel + kBlockElems - 1) / kBlockElems;
        SG_REQUIRE(blocks <= INT32_MAX, SG_ERR_INVALID_ARGUMENT, "adam_step: too many elements");
    }
    if (t.count == 0) return SG_OK;
    t.block_start[t.count] = (int)blocks;
    hipLaunchKernelGGL(adam_kernel<false>, dim3((unsigned)blocks), dim3(kThreads), 0, (hipStream_t)stream, t, (const float*)nullptr);
    return check_launch("sg_adam_step");
}

namespace sg {
namespace {

int check_list(const sg_grad_list* p, const char* what) {
    SG_REQUIRE(p != nullptr, SG_ERR_NULL_POINTER, "params is NULL");
    SG_REQUIRE(p->count >= 0, SG_ERR_INVALID_ARGUMENT, "%s: %d tensors", what, p->count);
    if (p->count == 0) return SG_OK;
    SG_REQUIRE(p->grads && p->numel && p->dtype, SG_ERR_NULL_POINTER, "%s: grads, numel or dtype is NULL", what);
    for (int i = 0; i < p->count; i++) {
        SG_REQUIRE(p->numel[i] >= 0 && p->numel[i] <= (int64_t)1 << 40, SG_ERR_INVALID_ARGUMENT, "%s: tensor %d: numel %lld", what, i,
                   (long long)p->numel[i]);
        SG_REQUIRE(p->dtype[i] == SG_F32 || p->dtype[i] == SG_F16 || p->dtype[i] == SG_BF16, SG_ERR_UNSUPPORTED,
                   "%s: tensor %d: dtype %d (float32, float16 or bfloat16)", what, i, (int)p->dtype[i]);
        if (p->numel[i] == 0) continue;
        SG_REQUIRE(p->grads[i], SG_ERR_NULL_POINTER, "%s: tensor %d is NULL", what, i);
        const int esize = p->dtype[i] == SG_F32 ? 4 : 2;
        SG_REQUIRE(reinterpret_cast<uintptr_t>(p->grads[i]) % esize == 0, SG_ERR_INVALID_ARGUMENT, "%s: tensor %d is not aligned to its elements", what, i);
    }
    return SG_OK;
}

int64_t tensor_blocks(const sg_grad_list& p, int i, int passes) {
    if (p.numel[i] == 0) return 0;
    const int64_t per = (int64_t)passes * kPacketsPerPass;
    const int64_t blocks = (p.numel[i] * (p.dtype[i] == SG_F32 ? 4 : 2) / 16 + per - 1) / per;    // (at least the whole packets' share)
    return blocks < 1 ? 1 : blocks;
}

// Chunk size of a list: one pass per block, doubled until the list fits kNormBlocks blocks (or a block has 1024 passes).
int list_passes(const sg_grad_list& p, int64_t* total) {
    for (int passes = 1;; passes *= 2) {
        int64_t blocks = 0;
        for (int i = 0; i < p.count; i++) blocks += tensor_blocks(p, i, passes);
        *total = blocks;
        if (blocks <= kNormBlocks || passes >= 1024) return passes;
    }
}

template <class Launch> int for_tables(const sg_grad_list& p, int passes, float grad_limit, const char* what, Launch launch) {
    NormTable t;
    t.count = 0;
    t.passes = passes;
    t.grad_limit = grad_limit;
    int64_t blocks = 0, before = 0;
    for (int i = 0; i <= p.count; i++) {
        if (t.count == kNormTensors || (i == p.count && t.count > 0)) {
            SG_REQUIRE(blocks <= INT32_MAX, SG_ERR_INVALID_ARGUMENT, "%s: too many elements", what);
            t.block_start[t.count] = (int)blocks;
            launch(t, (unsigned)blocks, before);
            const int rc = check_launch(what);
            if (rc != SG_OK) return rc;
            before += blocks;
            t.count = 0;
            blocks = 0;
        }
        if (i == p.count || p.numel[i] == 0) continue;
        const int k = t.count++;
        t.grad[k] = p.grads[i];
        t.numel[k] = p.numel[i];
        t.dtype[k] = (uint8_t)p.dtype[i];
        t.block_start[k] = (int)blocks;
        blocks += tensor_blocks(p, i, passes);
        SG_REQUIRE(blocks <= INT32_MAX, SG_ERR_INVALID_ARGUMENT, "%s: too many elements", what);
    }
    return SG_OK;
}

}  // namespace
}  // namespace sg

extern "C" size_t sg_grad_norm_workspace_bytes(const sg_grad_list* p) {
    using namespace sg;
    if (check_list(p, "grad_norm") != SG_OK) return 0;
    int64_t total = 0;
    list_passes(*p, &total);
    return (size_t)total * sizeof(double);
}

extern "C" int sg_grad_norm(const sg_grad_list* p, float grad_limit, float max_norm, float eps, float* out, void* workspace,
                            size_t workspace_bytes, sg_stream_t stream) {
    using namespace sg;
    const int rc = check_list(p, "grad_norm");
    if (rc != SG_OK) return rc;
    SG_REQUIRE(out != nullptr, SG_ERR_NULL_POINTER, "grad_norm: out is NULL");
    SG_REQUIRE(max_norm >= 0.f && eps >= 0.f, SG_ERR_INVALID_ARGUMENT, "grad_norm: max_norm and eps must not be negative");
    int64_t total = 0;
    const int passes = list_passes(*p, &total);
    SG_REQUIRE(total <= INT32_MAX, SG_ERR_INVALID_ARGUMENT, "grad_norm: too many elements");
    SG_REQUIRE(total == 0 || (workspace != nullptr && workspace_bytes >= (size_t)total * sizeof(double) && reinterpret_cast<uintptr_t>(workspace) % 8 == 0),
               SG_ERR_INVALID_ARGUMENT, "grad_norm: needs %lld bytes of aligned workspace", (long long)total * 8);
    double* partial = (double*)workspace;
    const int done = for_tables(*p, passes, grad_limit, "sg_grad_norm", [&](const NormTable& t, unsigned blocks, int64_t before) {
        hipLaunchKernelGGL(grad_norm_kernel, dim3(blocks), dim3(kThreads), 0, (hipStream_t)stream, t, partial + before);
    });
    if (done != SG_OK) return done;
    hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, partial, (int)total, max_norm, eps, out);
    return check_launch("sg_grad_norm");
}

extern "C" int sg_scale_grads(const sg_grad_list* p, const float* scale, sg_stream_t stream) {
    using namespace sg;
    const int rc = check_list(p, "scale_grads");
    if (rc != SG_OK) return rc;
    SG_REQUIRE(scale != nullptr, SG_ERR_NULL_POINTER, "scale_grads: scale is NULL");
    int64_t total = 0;
    const int passes = list_passes(*p, &total);
    return for_tables(*p, passes, 0.f, "sg_scale_grads", [&](const NormTable& t, unsigned blocks, int64_t) {
        hipLaunchKernelGGL(grad_scale_kernel, dim3(blocks), dim3(kThreads), 0, (hipStream_t)stream, t, scale);
    });
}

extern "C" int sg_adam_step_list(const sg_adam_list* p, sg_stream_t stream) {
    using namespace sg;
    SG_REQUIRE(p != nullptr, SG_ERR_NULL_POINTER, "params is NULL");
    SG_REQUIRE(p->count >= 0, SG_ERR_INVALID_ARGUMENT, "adam_step_list: %d tensors", p->count);
    SG_REQUIRE(p->beta1 >= 0.f && p->beta1 < 1.f && p->beta2 >= 0.f && p->beta2 < 1.f && p->eps >= 0.f && p->grad_limit > 0.f,
               SG_ERR_INVALID_ARGUMENT, "adam_step_list: betas must lie in [0, 1), eps >= 0, grad_limit > 0");
    if (p->count == 0) return SG_OK;
    SG_REQUIRE(p->param && p->grad && p->exp_avg && p->exp_avg_sq && p->numel && p->step, SG_ERR_NULL_POINTER, "adam_step_list: an array is NULL");
    for (int i = 0; i < p->count; i++) {                    // nothing is launched for a list that is rejected
        SG_REQUIRE(p->numel[i] >= 0 && p->numel[i] <= (int64_t)1 << 40 && p->step[i] >= 1, SG_ERR_INVALID_ARGUMENT,
                   "adam_step_list: tensor %d: numel %lld, step %d", i, (long long)p->numel[i], p->step[i]);
        SG_REQUIRE(p->numel[i] == 0 || (p->param[i] && p->grad[i] && p->exp_avg[i] && p->exp_avg_sq[i]), SG_ERR_NULL_POINTER,
                   "adam_step_list: tensor %d has a NULL pointer", i);
    }
    AdamTable t;
    t.count = 0;
    t.beta1 = p->beta1; t.beta2 = p->beta2; t.eps = p->eps; t.grad_limit = p->grad_limit;
    int64_t blocks = 0;
    double bc1 = 0, bc2 = 0;
    int32_t bc_step = 0;
    for (int i = 0; i <= p->count; i++) {
        if (t.count == kMaxTensors || (i == p->count && t.count > 0)) {
            t.block_start[t.count] = (int)blocks;
            if (p->grad_scale)
                hipLaunchKernelGGL(adam_kernel<true>, dim3((unsigned)blocks), dim3(kThreads), 0, (hipStream_t)stream, t, p->grad_scale);
            else
                hipLaunchKernelGGL(adam_kernel<false>, dim3((unsigned)blocks), dim3(kThreads), 0, (hipStream_t)stream, t, (const float*)nullptr);
            const int rc = check_launch("sg_adam_step_list");
            if (rc != SG_OK) return rc;
            t.count = 0;
            blocks = 0;
        }
        if (i == p->count || p->numel[i] == 0) continue;
        const int k = t.count++;
        t.param[k] = p->param[i]; t.grad[k] = p->grad[i]; t.exp_avg[k] = p->exp_avg[i]; t.exp_avg_sq[k] = p->exp_avg_sq[i];
        if (p->step[i] != bc_step) {                        // (tensors of one optimizer mostly share their count)
            bc_step = p->step[i];
            bc1 = 1.0 - pow((double)p->beta1, (double)bc_step);
            bc2 = 1.0 - pow((double)p->beta2, (double)bc_step);
        }
        t.step_size[k] = (float)((double)p->lr / bc1);
        t.sqrt_bc2[k] = (float)sqrt(bc2);
        t.numel[k] = p->numel[i];
        t.block_start[k] = (int)blocks;
        blocks += (p->numel[i] + kBlockElems - 1) / kBlockElems;
        SG_REQUIRE(blocks <= INT32_MAX, SG_ERR_INVALID_ARGUMENT, "adam_step_list: too many elements");
    }
    return SG_OK;
}

extern "C" int sg_lerp_multi(const sg_lerp_params* p, sg_stream_t stream) {
    using namespace sg;
    SG_REQUIRE(p != nullptr, SG_ERR_NULL_POINTER, "params is NULL");
    SG_REQUIRE(p->count >= 0 && p->count <= kMaxTensors, SG_ERR_INVALID_ARGUMENT, "lerp_multi: %d tensors (at most %d per call)",
               p->count, kMaxTensors);
    if (p->count == 0) return SG_OK;
    SG_REQUIRE(p->tensors != nullptr, SG_ERR_NULL_POINTER, "lerp_multi: tensors is NULL");
    LerpTable t;
    t.count = 0;
    t.weight = p->beta;
    int64_t blocks = 0;
    for (int i = 0; i < p->count; i++) {
        const sg_lerp_tensor& e = p->tensors[i];
        SG_REQUIRE(e.numel >= 0, SG_ERR_INVALID_ARGUMENT, "lerp_multi: tensor %d: numel %lld", i, (long long)e.numel);
        if (e.numel == 0) continue;
        SG_REQUIRE(e.dst && e.src, SG_ERR_NULL_POINTER, "lerp_multi: tensor %d has a NULL pointer", i);
        const int k = t.count++;
        t.dst[k] = e.dst; t.src[k] = e.src; t.numel[k] = e.numel;
        t.block_start[k] = (int)blocks;
        blocks += (e.numel + kBlockElems - 1) / kBlockElems;
        SG_REQUIRE(blocks <= INT32_MAX, SG_ERR_INVALID_ARGUMENT, "lerp_multi: too many elements");
    }
    if (t.count == 0) return SG_OK;
    t.block_start[t.count] = (int)blocks;
    hipLaunchKernelGGL(lerp_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, (hipStream_t)stream, t);
    return check_launch("sg_lerp_multi");
}
