// Multi-tensor AdamW (decoupled weight decay), one pass over (p, g, m, v): 28 bytes per parameter.
// Replaces torch.optim.AdamW.step as the reference configures it (train.py:193-197: lr 1e-3, weight_decay 1e-4).
//
// The arithmetic follows torch's single-tensor AdamW step operation by operation, in fp32:
//   p *= 1 - lr*wd;  m = b1*m + (1-b1)*g  (as lerp);  v = b2*v + (1-b2)*g*g
//   denom = sqrt(v)/sqrt(1-b2^t) + eps;  p -= (lr/(1-b1^t)) * m/denom
//
// Up to MIA_ADAMW_CHUNK tensors travel in one launch's kernel arguments (pointers + sizes by value: no device-side
// table to allocate or upload). A workgroup owns BLOCK_ELEMS consecutive elements of one tensor; it finds its tensor
// by scanning the chunk's block prefix.
#include "common.h"

#define MIA_ADAMW_CHUNK 48
// Elements of a workgroup: 22 tensors of a head, 0.8 M in all, take 16.0 us with 4096 (208 workgroups), 10.9 with 2048, 9.0 with 1024;
// the launches of a whole model's 10.9 M take the same with 2048 and up to a tenth longer with 1024.
#define MIA_ADAMW_BLOCK_ELEMS 2048

struct AdamWChunk {
    float* p[MIA_ADAMW_CHUNK];
    const float* g[MIA_ADAMW_CHUNK];
    float* m[MIA_ADAMW_CHUNK];
    float* v[MIA_ADAMW_CHUNK];
    long long n[MIA_ADAMW_CHUNK];
    int first_block[MIA_ADAMW_CHUNK + 1];
    int count;
    float lr_wd_keep;   // 1 - lr*wd
    float beta1, beta2, eps;
    float omb1, omb2;   // 1 - beta, formed in double on the host
    float step_size;    // lr / (1 - beta1^t)
    float inv_sqrt_bc2; // 1 / sqrt(1 - beta2^t)
    float grad_scale;   // gradients are multiplied by this first (1 = none)
};

__global__ __launch_bounds__(256) void adamw_kernel(AdamWChunk c, const float* __restrict__ dev_hyper,
                                                    const float* __restrict__ dev_clip) {
    // step-dependent factors from device memory when given: a captured graph replays fixed kernel arguments.
    // (Kept in locals: assigning to fields of `c` would force a private copy of the whole 2 KB argument block in
    // every lane -- measured at 73 us instead of 13 us a launch.)
    float lr_wd_keep = c.lr_wd_keep, step_size = c.step_size, inv_sqrt_bc2 = c.inv_sqrt_bc2;
    const float grad_scale = dev_clip ? c.grad_scale * dev_clip[1] : c.grad_scale;
    if (dev_hyper) {
        lr_wd_keep = dev_hyper[0];
        step_size = dev_hyper[1];
        inv_sqrt_bc2 = dev_hyper[2];
    }
    // wave-uniform scan: which tensor does this block belong to
    int t = 0;
    while (t + 1 < c.count && (int)blockIdx.x >= c.first_block[t + 1]) ++t;
    const long long base = (long long)((int)blockIdx.x - c.first_block[t]) * MIA_ADAMW_BLOCK_ELEMS;
    const long long n = c.n[t];
    float* __restrict__ p = c.p[t];
    const float* __restrict__ g = c.g[t];
    float* __restrict__ m = c.m[t];
    float* __restrict__ v = c.v[t];
    const float omb1 = c.omb1, omb2 = c.omb2;
    auto upd = [&](float& pp, float gg, float& mm, float& vv) {
        gg *= grad_scale;
        pp *= lr_wd_keep;
        mm = mm + omb1 * (gg - mm);          // lerp(m, g, 1-b1)
        vv = vv * c.beta2 + omb2 * gg * gg;
        const float denom = sqrtf(vv) * inv_sqrt_bc2 + c.eps;
        pp -= step_size * (mm / denom);
    };
    const bool vec = ((((uintptr_t)p | (uintptr_t)g | (uintptr_t)m | (uintptr_t)v) & 15) == 0);
#pragma unroll
    for (int it = 0; it < MIA_ADAMW_BLOCK_ELEMS / (256 * 4); ++it) {
        const long long i = base + (long long)(it * 256 + threadIdx.x) * 4;
        if (i >= n) break;
        if (vec && i + 4 <= n) {
            float4 pv = *reinterpret_cast<float4*>(p + i);
            const float4 gv = *reinterpret_cast<const float4*>(g + i);
            float4 mv = *reinterpret_cast<float4*>(m + i);
            float4 vv = *reinterpret_cast<float4*>(v + i);
            upd(pv.x, gv.x, mv.x, vv.x);
            upd(pv.y, gv.y, mv.y, vv.y);
            upd(pv.z, gv.z, mv.z, vv.z);
            upd(pv.w, gv.w, mv.w, vv.w);
            *reinterpret_cast<float4*>(p + i) = pv;
            *reinterpret_cast<float4*>(m + i) = mv;
            *reinterpret_cast<float4*>(v + i) = vv;
        } else {
            for (long long j = i; j < n && j < i + 4; ++j) upd(p[j], g[j], m[j], v[j]);
        }
    }
}

// params/grads/exp_avg/exp_avg_sq: HOST arrays of n_tensors DEVICE pointers (fp32, contiguous); sizes: host array of
// element counts. step is the 1-based step number of this update.
// dev_hyper (nullable): 3 floats in DEVICE memory {1 - lr*weight_decay, lr/(1 - beta1^step), 1/sqrt(1 - beta2^step)}
// read at run time in place of the values derived from lr/weight_decay/step, for launches replayed from a HIP graph
// (the caller rewrites them before each replay, e.g. with mia_set_words).
static int adamw_step(int n_tensors, const void* const* params, const void* const* grads, const void* const* exp_avg,
                      const void* const* exp_avg_sq, const long long* sizes, double lr, double beta1, double beta2,
                      double eps, double weight_decay, int step, double grad_scale, const float* dev_hyper,
                      const float* dev_clip, void* stream) {
    MIA_CHECK_ARG(n_tensors >= 0 && (n_tensors == 0 || (params && grads && exp_avg && exp_avg_sq && sizes)),
                  "mia_adamw_step: null table");
    MIA_CHECK_ARG(step >= 1, "mia_adamw_step: step must be >= 1 (got %d)", step);
    MIA_CHECK_ARG(beta1 >= 0. && beta1 < 1. && beta2 >= 0. && beta2 < 1. && eps >= 0. && lr >= 0.,
                  "mia_adamw_step: bad hyper-parameters");
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const double bc1 = 1.0 - pow(beta1, (double)step), bc2 = 1.0 - pow(beta2, (double)step);
    AdamWChunk c;
    // hyper-parameters arrive as doubles (Python floats) and are rounded to fp32 once, after the derived
    // quantities are formed: 1 - 0.999 in fp32 would be off by 1e-5 relative
    c.lr_wd_keep = (float)(1.0 - lr * weight_decay);
    c.beta1 = (float)beta1; c.beta2 = (float)beta2; c.eps = (float)eps;
    c.omb1 = (float)(1.0 - beta1); c.omb2 = (float)(1.0 - beta2);
    c.step_size = (float)(lr / bc1);
    c.inv_sqrt_bc2 = (float)(1.0 / sqrt(bc2));
    c.grad_scale = (float)grad_scale;
    int i = 0;
    while (i < n_tensors) {
        c.count = 0;
        int blocks = 0;
        while (i < n_tensors && c.count < MIA_ADAMW_CHUNK) {
            MIA_CHECK_ARG(sizes[i] >= 0 && params[i] && grads[i] && exp_avg[i] && exp_avg_sq[i],
                          "mia_adamw_step: tensor %d has a null pointer or a negative size", i);
            if (sizes[i] > 0) {
                const int k = c.count++;
                c.p[k] = (float*)params[i]; c.g[k] = (const float*)grads[i];
                c.m[k] = (float*)exp_avg[i]; c.v[k] = (float*)exp_avg_sq[i];
                c.n[k] = sizes[i];
                c.first_block[k] = blocks;
                blocks += cdiv(sizes[i], MIA_ADAMW_BLOCK_ELEMS);
            }
            ++i;
        }
        if (c.count == 0) continue;
        c.first_block[c.count] = blocks;
        MIA_LAUNCH(adamw_kernel, dim3(blocks), dim3(256), 0, s, c, dev_hyper, dev_clip);
        MIA_CHECK_LAUNCH("mia_adamw_step");
    }
    return 0;
}

extern "C" int mia_adamw_step(int n_tensors, const void* const* params, const void* const* grads,
                              const void* const* exp_avg, const void* const* exp_avg_sq, const long long* sizes,
                              double lr, double beta1, double beta2, double eps, double weight_decay, int step,
                              double grad_scale, const float* dev_hyper, void* stream) {
    return adamw_step(n_tensors, params, grads, exp_avg, exp_avg_sq, sizes, lr, beta1, beta2, eps, weight_decay, step,
                      grad_scale, dev_hyper, nullptr, stream);
}

extern "C" int mia_adamw_step_clipped(int n_tensors, const void* const* params, const void* const* grads,
                                      const void* const* exp_avg, const void* const* exp_avg_sq, const long long* sizes,
                                      double lr, double beta1, double beta2, double eps, double weight_decay, int step,
                                      double grad_scale, const float* dev_hyper, const float* norm_and_factor,
                                      void* stream) {
    MIA_CHECK_ARG(norm_and_factor, "mia_adamw_step_clipped: norm_and_factor is null (mia_grad_norm writes it)");
    return adamw_step(n_tensors, params, grads, exp_avg, exp_avg_sq, sizes, lr, beta1, beta2, eps, weight_decay, step,
                      grad_scale, dev_hyper, norm_and_factor, stream);
}

// ------------------------------------------------------------------------------------------------
// Global gradient norm over many tensors, and clipping: n = sqrt(sum over all tensors of g^2), factor = min(1, max_norm /
// (n + 1e-6)), g *= factor. The squares are formed and added in double: a sum of fp32 squares overflows from gradients of
// 1.8e19 on, and the double FMAs cost nothing here (the pass is bound by its loads).
//
// Up to GRAD_ENTRIES tensors travel in one launch's kernel arguments. The launch's work is a list of blocks (GRAD_VECS
// 16-byte vectors of one tensor each, at least one block a tensor); a fixed number of workgroups walks it with a constant
// stride and each leaves ONE partial sum, so every sum is formed in an order that depends on the sizes alone. The scaling
// pass walks the same list, and every workgroup of it first adds up the partial sums for itself (a few KB from L2): that
// is cheaper than a launch of its own in between.
// Tensors need not be 16-byte aligned (views into an exchange buffer are not): the elements in front of the first 16-byte
// boundary and behind the last one are done one by one by the tensor's first block.
// ------------------------------------------------------------------------------------------------
#define GRAD_ENTRIES 200
#define GRAD_VECS 2048            // 16-byte vectors of a block: eight per thread
#define GRAD_SLOTS 512            // workgroups (= partial sums) of one launch at most
#define GRAD_ENTRY_MAX (1ll << 30)   // elements of one entry; longer tensors take several

struct GradEntry {
    unsigned long long p;   // address; bit 0 set for bf16
    unsigned n;
    int first;              // first block
};
struct GradChunk {
    GradEntry e[GRAD_ENTRIES];
    int count, blocks;
};

template <typename T>
struct GradSpan {
    T *head, *tail;      // elements outside the 16-byte vectors
    int n_head, n_tail;
    T* body;
    long long nv;
    static constexpr int PER = 16 / (int)sizeof(T);
    __device__ __forceinline__ GradSpan(unsigned long long p, unsigned n) {
        T* base = reinterpret_cast<T*>(p);
        const unsigned lead = (unsigned)((16 - (p & 15)) & 15) / (unsigned)sizeof(T);
        n_head = (int)(lead < n ? lead : n);
        head = base;
        body = base + n_head;
        nv = (n - n_head) / PER;
        n_tail = (int)((n - n_head) - nv * PER);
        tail = body + nv * PER;
    }
};

// which tensor a block belongs to (uniform over the wave: scalar loads from the kernel arguments)
__device__ __forceinline__ int grad_find(const GradChunk& c, int blk) {
    int lo = 0, hi = c.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (c.e[mid].first <= blk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double grad_block_sum(double v, double* sm) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
    __syncthreads();
    return (sm[0] + sm[1]) + (sm[2] + sm[3]);
}

template <typename T>
__device__ __forceinline__ void grad_unpack(const uint4& v, float* o);
template <>
__device__ __forceinline__ void grad_unpack<float>(const uint4& v, float* o) {
    o[0] = __uint_as_float(v.x); o[1] = __uint_as_float(v.y); o[2] = __uint_as_float(v.z); o[3] = __uint_as_float(v.w);
}
template <>
__device__ __forceinline__ void grad_unpack<bf16_t>(const uint4& v, float* o) {
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const v2f t = unpack_bf16x2(w[i]);
        o[2 * i] = t.x;
        o[2 * i + 1] = t.y;
    }
}

template <typename T>
__device__ __forceinline__ double grad_sumsq(unsigned long long p, unsigned n, int local) {
    const GradSpan<T> s(p, n);
    constexpr int PER = GradSpan<T>::PER;
    double acc = 0.0;
    if (local == 0) {
        if ((int)threadIdx.x < s.n_head) { const double x = to_f32<T>(s.head[threadIdx.x]); acc = x * x; }
        if ((int)threadIdx.x < s.n_tail) { const double x = to_f32<T>(s.tail[threadIdx.x]); acc = fma(x, x, acc); }
    }
    const uint4* v = reinterpret_cast<const uint4*>(s.body);
    const long long v0 = (long long)local * GRAD_VECS + threadIdx.x;
    uint4 r[GRAD_VECS / 256];
    if ((long long)(local + 1) * GRAD_VECS <= s.nv) {   // whole block: eight loads in flight
#pragma unroll
        for (int i = 0; i < GRAD_VECS / 256; ++i) r[i] = v[v0 + i * 256];
    } else {
#pragma unroll
        for (int i = 0; i < GRAD_VECS / 256; ++i) r[i] = v0 + i * 256 < s.nv ? v[v0 + i * 256] : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < GRAD_VECS / 256; ++i) {
        float f[PER];
        grad_unpack<T>(r[i], f);
#pragma unroll
        for (int k = 0; k < PER; ++k) acc = fma((double)f[k], (double)f[k], acc);
    }
    return acc;
}

__global__ __launch_bounds__(256) void grad_sumsq_kernel(GradChunk c, double* __restrict__ partial) {
    __shared__ double sm[4];
    double acc = 0.0;
    for (int blk = blockIdx.x; blk < c.blocks; blk += gridDim.x) {
        const int t = grad_find(c, blk);
        const unsigned long long p = c.e[t].p;
        const int local = blk - c.e[t].first;
        acc += (p & 1) ? grad_sumsq<bf16_t>(p & ~1ull, c.e[t].n, local) : grad_sumsq<float>(p, c.e[t].n, local);
    }
    const double total = grad_block_sum(acc, sm);
    if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

// norm and factor from the partial sums; every thread of a 256-thread workgroup gets both
__device__ __forceinline__ void grad_finish(const double* __restrict__ partial, int slots, double mult, double max_norm,
                                            double* sm, double& norm, float& factor) {
    double acc = 0.0;
    for (int i = threadIdx.x; i < slots; i += 256) acc += partial[i];
    norm = sqrt(grad_block_sum(acc, sm)) * mult;
    const double f = max_norm / (norm + 1e-6);
    factor = f >= 1.0 ? 1.0f : (float)f;    // a NaN norm gives a NaN factor
}

__global__ __launch_bounds__(256) void grad_norm_finish_kernel(const double* __restrict__ partial, int slots, double mult,
                                                               double max_norm, float* __restrict__ out) {
    __shared__ double sm[4];
    double norm;
    float factor;
    grad_finish(partial, slots, mult, max_norm, sm, norm, factor);
    if (threadIdx.x == 0) {
        out[0] = (float)norm;
        out[1] = factor;
    }
}

template <typename T>
__device__ __forceinline__ uint4 grad_scaled(const uint4& v, float factor);
template <>
__device__ __forceinline__ uint4 grad_scaled<float>(const uint4& v, float factor) {
    return make_uint4(__float_as_uint(__uint_as_float(v.x) * factor), __float_as_uint(__uint_as_float(v.y) * factor),
                      __float_as_uint(__uint_as_float(v.z) * factor), __float_as_uint(__uint_as_float(v.w) * factor));
}
template <>
__device__ __forceinline__ uint4 grad_scaled<bf16_t>(const uint4& v, float factor) {
    return make_uint4(pack_bf16x2(unpack_bf16x2(v.x) * factor), pack_bf16x2(unpack_bf16x2(v.y) * factor),
                      pack_bf16x2(unpack_bf16x2(v.z) * factor), pack_bf16x2(unpack_bf16x2(v.w) * factor));
}

template <typename T>
__device__ __forceinline__ void grad_scale_block(unsigned long long p, unsigned n, int local, float factor) {
    const GradSpan<T> s(p, n);
    if (local == 0) {
        if ((int)threadIdx.x < s.n_head) s.head[threadIdx.x] = from_f32<T>(to_f32<T>(s.head[threadIdx.x]) * factor);
        if ((int)threadIdx.x < s.n_tail) s.tail[threadIdx.x] = from_f32<T>(to_f32<T>(s.tail[threadIdx.x]) * factor);
    }
    uint4* v = reinterpret_cast<uint4*>(s.body);
    const long long v0 = (long long)local * GRAD_VECS + threadIdx.x;
    if ((long long)(local + 1) * GRAD_VECS <= s.nv) {
        uint4 r[GRAD_VECS / 256];
#pragma unroll
        for (int i = 0; i < GRAD_VECS / 256; ++i) r[i] = v[v0 + i * 256];
#pragma unroll
        for (int i = 0; i < GRAD_VECS / 256; ++i) v[v0 + i * 256] = grad_scaled<T>(r[i], factor);
    } else {
        for (long long i = v0; i < s.nv; i += 256) v[i] = grad_scaled<T>(v[i], factor);
    }
}

__global__ __launch_bounds__(256) void grad_scale_kernel(GradChunk c, const double* __restrict__ partial, int slots,
                                                         double max_norm, float* __restrict__ out) {
    __shared__ double sm[4];
    double norm;
    float factor;
    grad_finish(partial, slots, 1.0, max_norm, sm, norm, factor);
    if (out && blockIdx.x == 0 && threadIdx.x == 0) {
        out[0] = (float)norm;
        out[1] = factor;
    }
    if (factor == 1.0f) return;
    for (int blk = blockIdx.x; blk < c.blocks; blk += gridDim.x) {
        const int t = grad_find(c, blk);
        const unsigned long long p = c.e[t].p;
        const int local = blk - c.e[t].first;
        if (p & 1) grad_scale_block<bf16_t>(p & ~1ull, c.e[t].n, local, factor);
        else grad_scale_block<float>(p, c.e[t].n, local, factor);
    }
}

// Walks the host tables and fills one chunk at a time; `at` / `off` = next tensor and the element it goes on from.
// Returns false when nothing is left.
static bool grad_fill(GradChunk& c, int n_tensors, const void* const* grads, const int* dtypes, const long long* sizes,
                      int& at, long long& off) {
    c.count = c.blocks = 0;
    while (at < n_tensors && c.count < GRAD_ENTRIES) {
        const long long left = sizes[at] - off;
        if (left <= 0) {
            ++at;
            off = 0;
            continue;
        }
        const bool half = dtypes && dtypes[at] == MIA_BF16;
        const int es = half ? 2 : 4, per = 16 / es;
        const long long n = left < GRAD_ENTRY_MAX ? left : GRAD_ENTRY_MAX;
        GradEntry& e = c.e[c.count++];
        const unsigned long long p = (unsigned long long)(uintptr_t)grads[at] + (unsigned long long)off * es;
        e.p = p | (half ? 1ull : 0ull);
        e.n = (unsigned)n;
        e.first = c.blocks;
        long long lead = (long long)((16 - (p & 15)) & 15) / es;
        if (lead > n) lead = n;
        const long long nv = (n - lead) / per;
        c.blocks += nv > GRAD_VECS ? cdiv(nv, GRAD_VECS) : 1;
        off += n;
    }
    return c.count > 0;
}

static int grad_slots(const GradChunk& c) { return c.blocks < GRAD_SLOTS ? c.blocks : GRAD_SLOTS; }

extern "C" long long mia_grad_norm_ws_doubles(int n_tensors, const long long* sizes) {
    long long entries = 0;
    for (int i = 0; i < n_tensors; ++i) entries += sizes[i] > 0 ? (sizes[i] + GRAD_ENTRY_MAX - 1) / GRAD_ENTRY_MAX : 0;
    return ((entries + GRAD_ENTRIES - 1) / GRAD_ENTRIES) * GRAD_SLOTS + 1;
}

static int grad_checks(const char* name, int n_tensors, const void* const* grads, const int* dtypes, const long long* sizes,
                       const double* ws, long long ws_doubles, const float* out) {
    MIA_CHECK_ARG(n_tensors >= 0 && (n_tensors == 0 || (grads && sizes)), "%s: null table", name);
    MIA_CHECK_ARG(ws && out, "%s: null workspace or output", name);
    for (int i = 0; i < n_tensors; ++i) {
        MIA_CHECK_ARG(sizes[i] >= 0 && (sizes[i] == 0 || grads[i]), "%s: tensor %d has a null pointer or a negative size", name, i);
        MIA_CHECK_ARG(!dtypes || dtypes[i] == MIA_F32 || dtypes[i] == MIA_BF16, "%s: tensor %d has a bad dtype %d", name, i, dtypes[i]);
        const unsigned long long es = dtypes && dtypes[i] == MIA_BF16 ? 2 : 4;
        MIA_CHECK_ARG((unsigned long long)(uintptr_t)grads[i] % es == 0, "%s: tensor %d is not aligned to its elements", name, i);
    }
    MIA_CHECK_ARG(ws_doubles >= mia_grad_norm_ws_doubles(n_tensors, sizes), "%s: workspace of %lld doubles is too small (%lld needed)",
                  name, ws_doubles, mia_grad_norm_ws_doubles(n_tensors, sizes));
    return 0;
}

// one partial sum per workgroup, over all chunks; returns how many through `slots`
static int grad_partials(const char* name, int n_tensors, const void* const* grads, const int* dtypes,
                         const long long* sizes, double* ws, int& slots, hipStream_t s) {
    GradChunk c;
    int at = 0;
    long long off = 0;
    slots = 0;
    while (grad_fill(c, n_tensors, grads, dtypes, sizes, at, off)) {
        const int g = grad_slots(c);
        MIA_LAUNCH(grad_sumsq_kernel, dim3(g), dim3(256), 0, s, c, ws + slots);
        MIA_CHECK_LAUNCH(name);
        slots += g;
    }
    return 0;
}

extern "C" int mia_grad_norm(int n_tensors, const void* const* grads, const int* dtypes, const long long* sizes,
                             double grad_scale, double max_norm, double* ws, long long ws_doubles, float* norm_and_factor,
                             void* stream) {
    if (grad_checks("mia_grad_norm", n_tensors, grads, dtypes, sizes, ws, ws_doubles, norm_and_factor)) return -1;
    MIA_CHECK_ARG(max_norm >= 0., "mia_grad_norm: max_norm must not be negative (got %g)", max_norm);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    int slots = 0;
    if (int rc = grad_partials("mia_grad_norm", n_tensors, grads, dtypes, sizes, ws, slots, s)) return rc;
    MIA_LAUNCH(grad_norm_finish_kernel, dim3(1), dim3(256), 0, s, ws, slots, fabs(grad_scale), max_norm, norm_and_factor);
    MIA_CHECK_LAUNCH("mia_grad_norm");
    return 0;
}

extern "C" int mia_grad_clip(int n_tensors, const void* const* grads, const int* dtypes, const long long* sizes,
                             double max_norm, double* ws, long long ws_doubles, float* norm_and_factor, void* stream) {
    if (grad_checks("mia_grad_clip", n_tensors, grads, dtypes, sizes, ws, ws_doubles, norm_and_factor)) return -1;
    MIA_CHECK_ARG(max_norm >= 0., "mia_grad_clip: max_norm must not be negative (got %g)", max_norm);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    int slots = 0;
    if (int rc = grad_partials("mia_grad_clip", n_tensors, grads, dtypes, sizes, ws, slots, s)) return rc;
    if (slots == 0) {
        MIA_LAUNCH(grad_norm_finish_kernel, dim3(1), dim3(256), 0, s, ws, 0, 1.0, max_norm, norm_and_factor);
        MIA_CHECK_LAUNCH("mia_grad_clip");
        return 0;
    }
    GradChunk c;
    int at = 0;
    long long off = 0;
    bool first = true;
    while (grad_fill(c, n_tensors, grads, dtypes, sizes, at, off)) {
        const int g = c.blocks < 4 * GRAD_SLOTS ? c.blocks : 4 * GRAD_SLOTS;
        MIA_LAUNCH(grad_scale_kernel, dim3(g), dim3(256), 0, s, c, ws, slots, max_norm, first ? norm_and_factor : nullptr);
        MIA_CHECK_LAUNCH("mia_grad_clip");
        first = false;
    }
    return 0;
}

// ---- small by-value upload: n 32-bit words travel in the kernel arguments and are stored to dst by one wave.
// Unlike an asynchronous copy from host memory, the values are fixed when the call returns, so the caller may
// overwrite its buffer at once; used to refresh the per-step words a replayed graph reads (seed offset, dev_hyper).
#define MIA_SET_WORDS_MAX 64
struct WordPack {
    unsigned w[MIA_SET_WORDS_MAX];
};

__global__ __launch_bounds__(64) void set_words_kernel(unsigned* __restrict__ dst, int n, WordPack v) {
    const int i = threadIdx.x;
    if (i < n) dst[i] = v.w[i];
}

extern "C" int mia_set_words(void* dst, int n, const unsigned* host_words, void* stream) {
    MIA_CHECK_ARG(n >= 0 && n <= MIA_SET_WORDS_MAX, "mia_set_words: n must be 0..%d (got %d)", MIA_SET_WORDS_MAX, n);
    if (n == 0) return 0;
    MIA_CHECK_ARG(dst && host_words, "mia_set_words: null pointer");
    WordPack v;
    for (int i = 0; i < MIA_SET_WORDS_MAX; ++i) v.w[i] = i < n ? host_words[i] : 0u;
    MIA_LAUNCH(set_words_kernel, dim3(1), dim3(64), 0, reinterpret_cast<hipStream_t>(stream), (unsigned*)dst, n,
                       v);
    MIA_CHECK_LAUNCH("mia_set_words");
    return 0;
}
