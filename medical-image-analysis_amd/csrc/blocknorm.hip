// The end of a residual branch fused with the norm in front of the next one, forward and backward (gfx950):
//
//   u = norm1(f) (or f),   y = x + scale * gate * u,   z = norm2(y)
//
// norm(t) = (t - mean) * r * w + b with r = 1 / sqrt(mean((t - mean)^2) + eps) (layer norm), or the same with mean = 0
// (RMS norm). scale is per channel, gate per image and channel; both, the norms and their weights are fp32.
//
// Backward, with that = (t - mean) * r and N^T(g) = r * (g - mean(g) [layer norm only] - that * mean(g * that)):
//   dy' = dy + N2^T(dz * w2);   dx = dy';   du = dy' * scale * gate;   df = N1^T(du * w1)
// and every parameter gradient follows from four column sums per image n: S1 = sum dy' * fhat, S2 = sum dy',
// S3 = sum dz * yhat, S4 = sum dz:
//   dgate_n = scale * (w1 S1_n + b1 S2_n)      dscale = sum_n gate_n * (w1 S1_n + b1 S2_n)
//   dw1 = scale * sum_n gate_n S1_n            db1 = scale * sum_n gate_n S2_n
//   dw2 = sum_n S3_n                           db2 = sum_n S4_n
// (fhat = f, w1 = 1, b1 = 0 where there is no norm1).
//
// A row lives in the registers of one wave (up to 64 * V * 2 channels) or one workgroup, V = channels of a 16-byte access, so
// every tensor is read once and written once: two in, two out forward; four in, two out backward. The statistics of both
// norms are kept (16 bytes a row). The next row is requested while one is worked on: a wave has one or two rows in flight instead of
// waiting out every load (32 images of 1444 rows of 1024 bf16 channels, two RMS norms: forward 91 -> 73 us, backward 164 -> 131;
// now 65, 5.8 TB/s, and 125, 4.5 TB/s). Long batches of rows are bound by HBM, short ones (a head's 100 tokens) by latency.
// The backward keeps its column sums in registers over all rows of a workgroup and leaves one slab row; two small kernels add
// the slab up in double, in a fixed order (no atomics).
#include "common.h"

enum { BNORM_NONE = 0, BNORM_RMS = 1, BNORM_LAYER = 2 };

struct BNormArgs {
    const void *x, *f, *dy, *dz;
    void *y, *z, *dx, *df;
    const float *scale, *gate, *w1, *b1, *w2, *b2;
    float* stats;   // [rows][4] = mean1, r1, mean2, r2
    float* slab;    // [N * S][4][C]
    int N, S, C, post, pre;
    long long T;    // rows of an image
    float eps, inv_c;
};

// V consecutive elements of a row as they lie in memory (one 16-byte access, or one element) and as fp32
template <typename T, int V>
struct BNormRaw {
    uint4 v;
};
template <typename T>
struct BNormRaw<T, 1> {
    T v;
};
template <typename T, int V>
__device__ __forceinline__ void bn_unpack(const BNormRaw<T, V>& r, float* o) {
    if constexpr (V == 8) {
        const unsigned w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const v2f t = unpack_bf16x2(w[i]);
            o[2 * i] = t.x;
            o[2 * i + 1] = t.y;
        }
    } else if constexpr (V == 4) {
        o[0] = __uint_as_float(r.v.x); o[1] = __uint_as_float(r.v.y);
        o[2] = __uint_as_float(r.v.z); o[3] = __uint_as_float(r.v.w);
    } else {
        o[0] = to_f32<T>(r.v);
    }
}
template <typename T, int V>
__device__ __forceinline__ void bn_store(T* p, const float* v) {
    if constexpr (V == 8) store44<T>(p, {v2f{v[0], v[1]}, v2f{v[2], v[3]}}, {v2f{v[4], v[5]}, v2f{v[6], v[7]}});
    else if constexpr (V == 4) store4<T>(p, {v[0], v[1], v[2], v[3]});
    else *p = from_f32<T>(v[0]);
}

// One row of a tensor on its way into registers: requested while the row before it is worked on. Lanes past the last channel load
// the row's first vector and count as zeros when it is unpacked.
template <typename T, int V, int R, int TPR>
struct BNormRow {
    BNormRaw<T, V> r[R];
    __device__ __forceinline__ void fetch(const void* base, long long row, int C, int lane) {
        const T* p = (const T*)base + row * C;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int c = (i * TPR + lane) * V;
            r[i] = *reinterpret_cast<const BNormRaw<T, V>*>(p + (c < C ? c : 0));
        }
    }
    __device__ __forceinline__ void take(float (&o)[R * V], int C, int lane) const {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            bn_unpack<T, V>(r[i], o + i * V);
            if (TPR * R * V != C && (i * TPR + lane) * V >= C)
#pragma unroll
                for (int k = 0; k < V; ++k) o[i * V + k] = 0.f;
        }
    }
};

// Sum of two values over the threads of one row. Workgroup rows take turns on two LDS buffers, so one barrier a round is
// enough: whoever writes round r + 2 has passed the barrier of round r + 1, which everyone reaches after reading round r.
template <int TPR>
struct RowSum {
    float2* sm;   // [2][waves]
    int turn;
    __device__ __forceinline__ void operator()(float& a, float& b) {
        a = wave_sum(a);
        b = wave_sum(b);
        if constexpr (TPR > 64) {
            constexpr int WAVES = TPR / 64;
            float2* buf = sm + turn * WAVES;
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = make_float2(a, b);
            __syncthreads();
            a = b = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float2 t = buf[w];
                a += t.x;
                b += t.y;
            }
        }
    }
};

// the fp32 vector of one parameter for this thread's channels (`none` where the parameter is absent)
template <int V, int R, int TPR>
__device__ __forceinline__ void bn_param(const float* p, float none, int lane, int C, float (&o)[R * V]) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int c = (r * TPR + lane) * V;
        if constexpr (V >= 4) {
#pragma unroll
            for (int k = 0; k < V; k += 4) {
                const float4 t = p && c < C ? *reinterpret_cast<const float4*>(p + c + k) : make_float4(none, none, none, none);
                o[r * V + k] = t.x; o[r * V + k + 1] = t.y; o[r * V + k + 2] = t.z; o[r * V + k + 3] = t.w;
            }
        } else {
            o[r] = p && c < C ? p[c] : none;
        }
    }
}

// mean and 1/deviation of a row held in registers; centred sums (a second round) for a layer norm
template <int V, int R, int TPR>
__device__ __forceinline__ void bn_stats(const float (&t)[R * V], int kind, int lane, const BNormArgs& a, RowSum<TPR>& sum,
                                         float& mean, float& r) {
    float s = 0.f, q = 0.f;
    mean = 0.f;
    if (kind == BNORM_LAYER) {
#pragma unroll
        for (int i = 0; i < R * V; ++i) s += t[i];
        sum(s, q);
        mean = s * a.inv_c;
        s = 0.f;
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float d = (i * TPR + lane) * V + k < a.C ? t[i * V + k] - mean : 0.f;
            s = fmaf(d, d, s);
        }
    q = 0.f;
    sum(s, q);
    r = 1.0f / sqrtf(fmaf(s, a.inv_c, a.eps));
}

// The branch's affine part as it is used, y = x + (mul * fhat + add): mul = scale * gate * w1, add = scale * gate * b1. Two vectors
// instead of three, and both directions form the same y; 200000 rows of 384 bf16 channels, two RMS norms: backward 236 -> 194 us.
template <int V, int R, int TPR>
__device__ __forceinline__ void bn_affine(const BNormArgs& a, int n, int lane, float (&mul)[R * V], float (&add)[R * V]) {
    float t[R * V];
    bn_param<V, R, TPR>(a.scale, 1.f, lane, a.C, mul);
    if (a.gate) {
        bn_param<V, R, TPR>(a.gate + (size_t)n * a.C, 1.f, lane, a.C, t);
#pragma unroll
        for (int i = 0; i < R * V; ++i) mul[i] *= t[i];
    }
    bn_param<V, R, TPR>(a.b1, 0.f, lane, a.C, t);
#pragma unroll
    for (int i = 0; i < R * V; ++i) add[i] = mul[i] * t[i];
    bn_param<V, R, TPR>(a.w1, 1.f, lane, a.C, t);
#pragma unroll
    for (int i = 0; i < R * V; ++i) mul[i] *= t[i];
}

template <typename T, int V, int R, int TPR, int WG>
__global__ __launch_bounds__(WG) void blocknorm_fwd_kernel(BNormArgs a) {
    __shared__ float2 sm[2 * (WG / 64)];
    RowSum<TPR> sum{sm, 0};
    const int n = blockIdx.x / a.S, s = blockIdx.x % a.S;
    const int lane = threadIdx.x % TPR, row_of = __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);   // a row is whole waves: scalar addresses
    const long long lo = a.T * s / a.S, hi = a.T * (s + 1) / a.S;
    float mul[R * V], add[R * V], w2[R * V], b2[R * V];
    bn_affine<V, R, TPR>(a, n, lane, mul, add);
    bn_param<V, R, TPR>(a.w2, 1.f, lane, a.C, w2);
    bn_param<V, R, TPR>(a.b2, 0.f, lane, a.C, b2);
    BNormRow<T, V, R, TPR> fr, xr;
    const long long first = (long long)n * a.T;
    if (lo + row_of < hi) {
        fr.fetch(a.f, first + lo + row_of, a.C, lane);
        xr.fetch(a.x, first + lo + row_of, a.C, lane);
    }
    for (long long t = lo + row_of; t < hi; t += WG / TPR) {
        const long long row = first + t;
        float f[R * V], y[R * V];
        fr.take(f, a.C, lane);
        xr.take(y, a.C, lane);
        if (t + WG / TPR < hi) {
            fr.fetch(a.f, row + WG / TPR, a.C, lane);
            xr.fetch(a.x, row + WG / TPR, a.C, lane);
        }
        float m1 = 0.f, r1 = 1.f, m2 = 0.f, r2 = 1.f;
        if (a.post) {
            bn_stats<V, R, TPR>(f, a.post, lane, a, sum, m1, r1);
#pragma unroll
            for (int i = 0; i < R * V; ++i) f[i] = (f[i] - m1) * r1;
        }
#pragma unroll
        for (int i = 0; i < R * V; ++i) y[i] += fmaf(mul[i], f[i], add[i]);
        if (TPR * R * V != a.C) {   // channels behind the last one stay zero for the statistics' plain sum
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int k = 0; k < V; ++k)
                    if ((r * TPR + lane) * V + k >= a.C) y[r * V + k] = 0.f;
        }
        T* yp = (T*)a.y + row * a.C;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * TPR + lane) * V;
            if (c < a.C) bn_store<T, V>(yp + c, y + r * V);
        }
        if (a.pre) {
            bn_stats<V, R, TPR>(y, a.pre, lane, a, sum, m2, r2);
            T* zp = (T*)a.z + row * a.C;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int c = (r * TPR + lane) * V;
                float z[V];
#pragma unroll
                for (int k = 0; k < V; ++k) z[k] = fmaf((y[r * V + k] - m2) * r2, w2[r * V + k], b2[r * V + k]);
                if (c < a.C) bn_store<T, V>(zp + c, z);
            }
        }
        if (a.stats && lane == 0) *reinterpret_cast<float4*>(a.stats + row * 4) = make_float4(m1, r1, m2, r2);
    }
}

template <typename T, int V, int R, int TPR, int WG>
__global__ __launch_bounds__(WG) void blocknorm_bwd_kernel(BNormArgs a) {
    __shared__ float2 sm[2 * (WG / 64)];
    RowSum<TPR> sum{sm, 0};
    const int n = blockIdx.x / a.S, s = blockIdx.x % a.S;
    const int lane = threadIdx.x % TPR, row_of = __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);   // a row is whole waves: scalar addresses
    const long long lo = a.T * s / a.S, hi = a.T * (s + 1) / a.S;
    // The threads of a row of 1024 have 128 registers each: with eight channels they neither request rows ahead nor keep the
    // parameters, but read those again (from L2) where a row needs them (2048 rows of 8192, two RMS norms: 169 -> 97 us in
    // bf16, 251 -> 167 us in fp32). Single elements spill either way (353 us, 517 us so).
    // (dy and dz were one tensor there; with two of them 182 us in fp32, 374 for rows of 8190 in single elements.)
    constexpr bool SLIM = TPR == 1024 && V > 1 && R * V == 8;
    float mul[R * V], add[R * V], w2[R * V];
    auto load_w2 = [&]() { bn_param<V, R, TPR>(a.w2, 1.f, lane, a.C, w2); };
    if constexpr (!SLIM) {
        bn_affine<V, R, TPR>(a, n, lane, mul, add);
        load_w2();
    }
    float s1[R * V], s2[R * V], s3[R * V], s4[R * V];
#pragma unroll
    for (int i = 0; i < R * V; ++i) s1[i] = s2[i] = s3[i] = s4[i] = 0.f;
    BNormRow<T, V, R, TPR> fr, gr, zr, xr;
    float4 sr = make_float4(0.f, 0.f, 0.f, 0.f);
    const long long first = (long long)n * a.T;
    auto fetch = [&](long long row) {   // of an absent gradient the branch itself, which is not used
        sr = *reinterpret_cast<const float4*>(a.stats + row * 4);
        fr.fetch(a.f, row, a.C, lane);
        gr.fetch(a.dy ? a.dy : a.f, row, a.C, lane);
        if (a.dz) {
            zr.fetch(a.dz, row, a.C, lane);
            xr.fetch(a.x, row, a.C, lane);
        }
    };
    if (!SLIM && lo + row_of < hi) fetch(first + lo + row_of);
    for (long long t = lo + row_of; t < hi; t += WG / TPR) {
        const long long row = first + t, at = row * a.C;
        if constexpr (SLIM) fetch(row);
        const float4 st = sr;
        float f[R * V], g[R * V], z[R * V], y[R * V];   // f -> fhat; g: dy -> dy'; z: dz; y: x -> yhat
        fr.take(f, a.C, lane);
        gr.take(g, a.C, lane);
        if (!a.dy)
#pragma unroll
            for (int i = 0; i < R * V; ++i) g[i] = 0.f;
        if (a.dz) {
            zr.take(z, a.C, lane);
            xr.take(y, a.C, lane);
        }
        if (!SLIM && t + WG / TPR < hi) fetch(row + WG / TPR);
        if (a.post) {
#pragma unroll
            for (int i = 0; i < R * V; ++i) f[i] = (f[i] - st.x) * st.y;
        }
        if (a.dz) {
            float p = 0.f, q = 0.f;
            if constexpr (SLIM) {
                bn_affine<V, R, TPR>(a, n, lane, mul, add);
                load_w2();
            }
#pragma unroll
            for (int i = 0; i < R * V; ++i) {
                y[i] = (y[i] + fmaf(mul[i], f[i], add[i]) - st.z) * st.w;
                const float d = z[i] * w2[i];   // zero behind the last channel, where dz was not loaded
                p += d;
                q = fmaf(d, y[i], q);
            }
            sum(p, q);
            p = a.pre == BNORM_LAYER ? p * a.inv_c : 0.f;
            q *= a.inv_c;
#pragma unroll
            for (int i = 0; i < R * V; ++i) {
                s3[i] = fmaf(z[i], y[i], s3[i]);
                s4[i] += z[i];
                g[i] += (fmaf(z[i], w2[i], -p) - y[i] * q) * st.w;
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * TPR + lane) * V;
            if (c < a.C) bn_store<T, V>((T*)a.dx + at + c, g + r * V);
        }
        if constexpr (SLIM) bn_affine<V, R, TPR>(a, n, lane, mul, add);
#pragma unroll
        for (int i = 0; i < R * V; ++i) {
            s1[i] = fmaf(g[i], f[i], s1[i]);
            s2[i] += g[i];
            g[i] *= mul[i];
        }
        if (a.post) {
            float p = 0.f, q = 0.f;
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const int i = r * V + k;
                    if ((r * TPR + lane) * V + k >= a.C) g[i] = 0.f;
                    p += g[i];
                    q = fmaf(g[i], f[i], q);
                }
            sum(p, q);
            p = a.post == BNORM_LAYER ? p * a.inv_c : 0.f;
            q *= a.inv_c;
#pragma unroll
            for (int i = 0; i < R * V; ++i) g[i] = (g[i] - p - f[i] * q) * st.y;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * TPR + lane) * V;
            if (c < a.C) bn_store<T, V>((T*)a.df + at + c, g + r * V);
        }
    }
    // one slab row per workgroup; the waves of a wave-per-row workgroup are added in LDS first, in wave order
    float* out = a.slab + (size_t)blockIdx.x * 4 * a.C;
    auto flush = [&](const float (&v)[R * V], float* dst) {
        if constexpr (TPR == WG) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const int c = (r * TPR + lane) * V + k;
                    if (c < a.C) dst[c] = v[r * V + k];
                }
        } else {
            constexpr int ROWS = WG / TPR, W = R * V * TPR;
            __shared__ float cols[ROWS * W];
            __syncthreads();
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int k = 0; k < V; ++k) cols[row_of * W + (r * TPR + lane) * V + k] = v[r * V + k];
            __syncthreads();
            for (int c = threadIdx.x; c < a.C; c += WG) {
                float acc = cols[c];
#pragma unroll
                for (int w = 1; w < ROWS; ++w) acc += cols[w * W + c];
                dst[c] = acc;
            }
        }
    };
    flush(s1, out);
    flush(s2, out + a.C);
    flush(s3, out + 2 * (size_t)a.C);
    flush(s4, out + 3 * (size_t)a.C);
}

// sums[group] = slab rows [group * per, (group + 1) * per) added up; dgate of the group's image where there is a gate.
// grid (groups, ceil(C / 64)), 16 row lanes x 64 columns.
__global__ __launch_bounds__(1024) void blocknorm_fold_kernel(const float* __restrict__ slab, int rows, int per, int C,
                                                              const float* __restrict__ scale, const float* __restrict__ w1,
                                                              const float* __restrict__ b1, double* __restrict__ sums,
                                                              float* __restrict__ dgate) {
    __shared__ double sm[16][4][64];
    const int col = threadIdx.x & 63, g = threadIdx.x >> 6, c = blockIdx.y * 64 + col;
    const int r0 = blockIdx.x * per, r1 = min(rows, r0 + per);
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    if (c < C)
        for (int r = r0 + g; r < r1; r += 16)
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] += (double)slab[((size_t)r * 4 + k) * C + c];
#pragma unroll
    for (int k = 0; k < 4; ++k) sm[g][k][col] = v[k];
    __syncthreads();
    if (g != 0 || c >= C) return;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        for (int w = 1; w < 16; ++w) v[k] += sm[w][k][col];
#pragma unroll
    for (int k = 0; k < 4; ++k) sums[((size_t)blockIdx.x * 4 + k) * C + c] = v[k];
    if (dgate) dgate[(size_t)blockIdx.x * C + c] = (float)((scale ? scale[c] : 1.f) * ((w1 ? w1[c] : 1.f) * v[0] + (b1 ? b1[c] : 0.f) * v[1]));
}

// Parameter gradients from the group sums (S = double) or from the slab's rows themselves (float); gate (nullable): [groups][C].
// 64 row lanes x 16 columns: few rounds of loads, each of which waits for memory.
template <typename S>
__global__ __launch_bounds__(1024) void blocknorm_params_kernel(const S* __restrict__ sums, int groups, int C,
                                                                const float* __restrict__ gate, const float* __restrict__ scale,
                                                                const float* __restrict__ w1, const float* __restrict__ b1,
                                                                float* dscale, float* dw1, float* db1, float* dw2, float* db2) {
    __shared__ double sm[64][4][16];
    const int col = threadIdx.x & 15, g = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    if (c < C)
        for (int n = g; n < groups; n += 64) {
            const S* p = sums + (size_t)n * 4 * C + c;
            const double gt = gate ? gate[(size_t)n * C + c] : 1.f;
            v[0] = fma(gt, (double)p[0], v[0]);
            v[1] = fma(gt, (double)p[C], v[1]);
            v[2] += (double)p[2 * (size_t)C];
            v[3] += (double)p[3 * (size_t)C];
        }
#pragma unroll
    for (int k = 0; k < 4; ++k) sm[g][k][col] = v[k];
    __syncthreads();
    if (threadIdx.x < 64) {   // one sum a thread; only it reads and writes its column of sm[..][g]
        double t = sm[0][g][col];
#pragma unroll 8
        for (int w = 1; w < 64; ++w) t += sm[w][g][col];
        sm[0][g][col] = t;
    }
    __syncthreads();
    if (g != 0 || c >= C) return;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = sm[0][k][col];
    const double sc = scale ? scale[c] : 1.f;
    if (dscale) dscale[c] = (float)((w1 ? w1[c] : 1.f) * v[0] + (b1 ? b1[c] : 0.f) * v[1]);
    if (dw1) dw1[c] = (float)(sc * v[0]);
    if (db1) db1[c] = (float)(sc * v[1]);
    if (dw2) dw2[c] = (float)v[2];
    if (db2) db2[c] = (float)v[3];
}

// ------------------------------------------------------------------------------------------------
// Row layout of a launch. V channels a 16-byte access where C and the pointers allow it, else single elements. A wave per
// row while two accesses a lane cover it (four rows a workgroup, no barrier), a workgroup per row above (1024 bf16 channels:
// forward 73 us, 88 with two waves a row and a barrier for each sum).
// ------------------------------------------------------------------------------------------------
#define BNORM_MAX_C 8192

// (the parameters are read 16 bytes at a time then, too)
static bool bn_vec(int dtype, int C, const void* const* ptrs, int n) {
    if (C % (dtype == MIA_BF16 ? 8 : 4)) return false;
    for (int i = 0; i < n; ++i)
        if ((uintptr_t)ptrs[i] & 15) return false;
    return true;
}

template <typename T, int V, int R, int TPR, int WG>
static void bn_launch(bool fwd, const BNormArgs& a, hipStream_t s) {
    if (fwd) MIA_LAUNCH((blocknorm_fwd_kernel<T, V, R, TPR, WG>), dim3(a.N * a.S), dim3(WG), 0, s, a);
    else MIA_LAUNCH((blocknorm_bwd_kernel<T, V, R, TPR, WG>), dim3(a.N * a.S), dim3(WG), 0, s, a);
}

template <typename T>
static void bn_dispatch(bool fwd, bool vec, const BNormArgs& a, hipStream_t s) {
    constexpr int V = 16 / (int)sizeof(T);
    if (vec) {
        const int u = (a.C + V - 1) / V;   // accesses of a row
        if (u <= 64) bn_launch<T, V, 1, 64, 256>(fwd, a, s);
        else if (u <= 128) bn_launch<T, V, 2, 64, 256>(fwd, a, s);
        else if (u <= 256) bn_launch<T, V, 1, 256, 256>(fwd, a, s);
        else if (u <= 512) bn_launch<T, V, 1, 512, 512>(fwd, a, s);
        else if (u <= 1024) bn_launch<T, V, 1, 1024, 1024>(fwd, a, s);
        else if constexpr (V == 4) bn_launch<T, V, 2, 1024, 1024>(fwd, a, s);
    } else {
        if (a.C <= 64) bn_launch<T, 1, 1, 64, 256>(fwd, a, s);
        else if (a.C <= 512) bn_launch<T, 1, 8, 64, 256>(fwd, a, s);
        else if (a.C <= 2048) bn_launch<T, 1, 8, 256, 256>(fwd, a, s);
        else bn_launch<T, 1, 8, 1024, 1024>(fwd, a, s);
    }
}

// Workgroups an image's rows are split over: as many in all as are resident at once, so that the rows come out even, with at
// least one row a wave forward and two backward, two where a workgroup has a row (100 rows of 384 bf16 channels: forward 3.6 us,
// 7.2 with four rows a wave; backward 6.7 and 8.7).
// Backward three a CU up to 512 channels (100000 rows of 256 fp32 channels: 126 us, 134 with 512 workgroups; 200000 of 384 in bf16:
// 194 and 196), else two (32 images of 1444 rows of 1024 bf16 channels: 125 us; 142 with 1024 workgroups and 134 with 512
// before the affine part was kept as two vectors). Forward four a CU with eight channels a lane (200000 rows of 384 bf16 channels:
// 120 us, 143 with 512), three with sixteen (rows of 1024: 65 us, 70 with 1024, 67 with 512), two with a workgroup a row (8000
// rows of 2048: 28 us, 45 with 256).
static int bn_splits(bool fwd, int dtype, long long images, long long rows, int C) {
    const long long want = !fwd ? (C <= 512 ? 768 : 512) : C > 1024 ? 512 : dtype == MIA_BF16 && C > 512 ? 768 : 1024, per = C > 512 ? 2 : fwd ? 4 : 8;
    long long s = (want + images - 1) / images;
    if (s > rows / per) s = rows / per;
    return s < 1 ? 1 : (int)s;
}

static int bn_groups(int gated, int N, int S) { return gated ? N : (N * S + 15) / 16; }

extern "C" long long mia_blocknorm_ws_floats(int images, long long rows_per_image, int C, int gated) {
    const int S = bn_splits(false, MIA_F32, gated ? images : 1, gated ? rows_per_image : rows_per_image * images, C), N = gated ? images : 1;
    return ((long long)N * S + 2ll * bn_groups(gated, N, S)) * 4 * C;   // slab rows | group sums (doubles)
}

static int bn_checks(const char* name, int dtype, int images, long long rows, int C, const float* gate, int post, int pre, float eps) {
    MIA_CHECK_ARG(dtype == MIA_F32 || dtype == MIA_BF16, "%s: bad dtype %d", name, dtype);
    MIA_CHECK_ARG(images > 0 && rows > 0 && C > 0 && C <= BNORM_MAX_C, "%s: bad shape images=%d rows=%lld C=%d (C <= %d)", name,
                  images, rows, C, BNORM_MAX_C);
    MIA_CHECK_ARG((long long)images * rows <= 0x7fffffffll, "%s: %lld rows are too many", name, (long long)images * rows);
    MIA_CHECK_ARG(!gate || images < 1 << 22, "%s: gates of %d images are too many", name, images);   // a workgroup each, 1024 threads
    MIA_CHECK_ARG(post >= 0 && post <= 2 && pre >= 0 && pre <= 2, "%s: bad norm kind (%d, %d)", name, post, pre);
    MIA_CHECK_ARG(eps >= 0.f, "%s: eps must not be negative", name);
    return 0;
}

static void bn_shape(BNormArgs& a, bool fwd, int dtype, int images, long long rows, int C, int post, int pre, float eps) {
    a.N = a.gate ? images : 1;
    a.T = a.gate ? rows : rows * images;
    a.S = bn_splits(fwd, dtype, a.N, a.T, C);
    a.C = C; a.post = post; a.pre = pre; a.eps = eps; a.inv_c = 1.0f / (float)C;
}

extern "C" int mia_blocknorm_fwd(int dtype, const void* x, const void* f, int images, long long rows_per_image, int C,
                                 const float* scale, const float* gate, int post, const float* post_w, const float* post_b,
                                 int pre, const float* pre_w, const float* pre_b, float eps, void* y, void* z, float* stats,
                                 void* stream) {
    if (bn_checks("mia_blocknorm_fwd", dtype, images, rows_per_image, C, gate, post, pre, eps)) return -1;
    MIA_CHECK_ARG(x && f && y && (!pre || z), "mia_blocknorm_fwd: null");
    MIA_CHECK_ARG(((uintptr_t)stats & 15) == 0, "mia_blocknorm_fwd: stats must start at a multiple of 16 bytes");
    MIA_CHECK_ARG(!post == !post_w && !pre == !pre_w && (post || !post_b) && (pre || !pre_b),
                  "mia_blocknorm_fwd: a norm comes with its weight, and only then with a bias");
    BNormArgs a = {};
    a.x = x; a.f = f; a.y = y; a.z = z; a.stats = stats;
    a.scale = scale; a.gate = gate; a.w1 = post_w; a.b1 = post_b; a.w2 = pre_w; a.b2 = pre_b;
    bn_shape(a, true, dtype, images, rows_per_image, C, post, pre, eps);
    const void* ptrs[] = {x, f, y, pre ? z : y, scale, gate, post_w, post_b, pre_w, pre_b};
    const bool vec = bn_vec(dtype, C, ptrs, 10);
    if (dtype == MIA_BF16) bn_dispatch<bf16_t>(true, vec, a, reinterpret_cast<hipStream_t>(stream));
    else bn_dispatch<float>(true, vec, a, reinterpret_cast<hipStream_t>(stream));
    MIA_CHECK_LAUNCH("mia_blocknorm_fwd");
    return 0;
}

extern "C" int mia_blocknorm_bwd(int dtype, const void* dy, const void* dz, const void* x, const void* f, const float* stats,
                                 int images, long long rows_per_image, int C, const float* scale, const float* gate, int post,
                                 const float* post_w, const float* post_b, int pre, const float* pre_w, float* ws,
                                 long long ws_floats, void* dx, void* df, float* dscale, float* dgate, float* dpost_w,
                                 float* dpost_b, float* dpre_w, float* dpre_b, void* stream) {
    if (bn_checks("mia_blocknorm_bwd", dtype, images, rows_per_image, C, gate, post, pre, 0.f)) return -1;
    MIA_CHECK_ARG((dy || dz) && x && f && stats && ws && dx && df, "mia_blocknorm_bwd: null");
    MIA_CHECK_ARG((((uintptr_t)ws | (uintptr_t)stats) & 15) == 0, "mia_blocknorm_bwd: stats and the workspace must start at multiples of 16 bytes");
    MIA_CHECK_ARG(!post == !post_w && !pre == !pre_w && (post || !post_b) && (pre || !dz),
                  "mia_blocknorm_bwd: a norm comes with its weight, and only then with a gradient");
    MIA_CHECK_ARG(ws_floats >= mia_blocknorm_ws_floats(images, rows_per_image, C, gate != nullptr),
                  "mia_blocknorm_bwd: workspace of %lld floats is too small (%lld needed)", ws_floats,
                  mia_blocknorm_ws_floats(images, rows_per_image, C, gate != nullptr));
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    BNormArgs a = {};
    a.dy = dy; a.dz = dz; a.x = x; a.f = f; a.dx = dx; a.df = df; a.stats = const_cast<float*>(stats); a.slab = ws;
    a.scale = scale; a.gate = gate; a.w1 = post_w; a.b1 = post_b; a.w2 = pre_w;
    bn_shape(a, false, dtype, images, rows_per_image, C, post, pre, 0.f);
    const void* ptrs[] = {x, f, dx, df, dy, dz, scale, gate, post_w, post_b, pre_w};
    const bool vec = bn_vec(dtype, C, ptrs, 11);
    if (dtype == MIA_BF16) bn_dispatch<bf16_t>(false, vec, a, s);
    else bn_dispatch<float>(false, vec, a, s);
    MIA_CHECK_LAUNCH("mia_blocknorm_bwd");
    // up to 64 slab rows without a gate are added up by the parameter kernel itself (four to a lane): one launch less
    const int rows = a.N * a.S;
    const bool fold = gate || rows > 64;
    const int groups = fold ? bn_groups(gate != nullptr, a.N, a.S) : rows;
    if (fold) {
        double* sums = reinterpret_cast<double*>(ws + (size_t)rows * 4 * C);
        MIA_LAUNCH(blocknorm_fold_kernel, dim3(groups, cdiv(C, 64)), dim3(1024), 0, s, ws, rows, gate ? a.S : 16, C, scale, post_w,
                   post_b, sums, gate ? dgate : nullptr);
        MIA_CHECK_LAUNCH("mia_blocknorm_bwd");
        MIA_LAUNCH(blocknorm_params_kernel<double>, dim3(cdiv(C, 16)), dim3(1024), 0, s, sums, groups, C, gate, scale, post_w, post_b, dscale,
                   dpost_w, dpost_b, dpre_w, dpre_b);
    } else {
        MIA_LAUNCH(blocknorm_params_kernel<float>, dim3(cdiv(C, 16)), dim3(1024), 0, s, ws, groups, C, gate, scale, post_w, post_b, dscale,
                   dpost_w, dpost_b, dpre_w, dpre_b);
    }
    MIA_CHECK_LAUNCH("mia_blocknorm_bwd");
    return 0;
}
