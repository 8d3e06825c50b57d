// Attention with a learned relative position bias, forward and backward (gfx950).
//
//   s_ij = scale * q_i . k_j + table[bucket(pos_j - pos_i)][head],  P = softmax over the unmasked keys,  O = P V
//   dV = P^T dO,  dP = dO V^T,  D_i = sum_j P_ij dP_ij,  dS = P o (dP - D),  dQ = scale dS K,  dK = scale dS^T Q,
//   dtable[k][head] = sum of dS over the batch and over all pairs whose offset lies in bucket k
//
// Tokens are the positions of an H x W map in row order (a sequence is a map of one row). With c(p) = (p / W)(2W - 1) + p % W
// the offset of a pair is the single number c(j) - c(i): it names (dy, dx) uniquely, so one fp32 vector per head over the
// (2H - 1)(2W - 1) offsets holds the whole bias. relpos_expand_kernel forms it from the table (divided by scale, because
// the matrix accumulators start from it: acc = q.k + bias / scale), and a tile of pairs needs only the short window of it
// that its tokens' c span, which is staged in LDS next to the tile.
//
// Matrix cores: S^T = K Q^T with keys as rows leaves a lane of v_mfma_f32_16x16x* four consecutive keys of ONE query: the
// softmax runs down registers plus two lane exchanges, and the four values are already the B operand of O^T = V^T P^T (V^T
// read from the row-major tile by the transposing LDS read). fp32 runs the same code on 16x16x4. Scores and weights never
// exist in memory (the table's gradient needs rows of offsets, see rp_slab_ld); the backward recomputes P from the row statistics, once with queries as columns (dQ) and once with keys as
// columns (dK, dV, dtable). P and dS become bf16 only as operands of bf16 products, as two numbers each (what the first
// rounding took off is the second); statistics and D stay fp32, the bias gradient is added up in double.
//
// D is needed to fp32 accuracy because the rows of dS sum to zero and a bucket's gradient is what is left of many terms. The
// output a bf16 caller holds is too coarse for it: the forward keeps what its rounding took off beside it, the dQ kernel starts from
// D~ = dO . (out + out_low), good to 2^-16, and leaves D~ + sum_j P_ij (dP_ij - D~_i) = D_i, added up in fp32 on the way, for
// the dK / dV / dtable kernel.
#include "common.h"

typedef __attribute__((ext_vector_type(4))) float rp_f32x4;
typedef __attribute__((ext_vector_type(4))) short rp_s16x4;
typedef __attribute__((ext_vector_type(8))) short rp_s16x8;
typedef __attribute__((ext_vector_type(8))) __bf16 rp_bf16x8;

#define RP_LOG2E 1.4426950408889634f
#define RP_TILE 64          // tokens that one round of products works on
// Largest maximum, in units of the exponent, up to which P = exp2(acc * sl2 - shift) is formed by one FMA with shift rounded to
// fp32 (64 * 2^-24 = 4e-6 relative in P at worst); rows beyond it subtract first.
#define RP_FAR 64.f
#define RP_MAX_WIDTH 896    // of a map of several rows: keeps the dK/dV kernel's rings (RP_RING_MAX offsets) in LDS
#define RP_RING_MAX 2048

struct RpStride {
    long long b, t, h;   // elements
};
struct RpArgs {
    const void *q, *k, *v, *dout, *out, *out_low;
    void *o, *o_low, *dq, *dk, *dv;   // o_low: what rounding o to bf16 took off it, for the backward's D; nullable
    RpStride sq, sk, sv, sdq, sdk, sdv;
    const float* bias;            // [heads][n_off]
    float2* stat;                 // [B][heads][Lq]: maximum of acc, log2 of the sum of exponentials
    float* dsum;                  // [B][heads][Lq]
    const uint8_t* mask;          // [B][Lk], nullable
    float* slab;                  // dK/dV kernel: [B * heads * key blocks][slab_ld], nullable
    float *po, *pml;              // split forward: [splits][B * heads * Lq][D], [..][2]
    int B, heads, Lq, Lk, D, W, off, n_off, q_start;
    unsigned inv_w;               // ceil(2^32 / W)
    int tiles, splits, acc_mask, slab_ld, few;
    float scale, sl2, pdrop;
    unsigned long long seed;
    const unsigned long long* seed_off;
};

__device__ __forceinline__ unsigned long long rp_seed(const RpArgs& a) {
    return a.seed_off ? a.seed + a.seed_off[0] * 0x9E3779B97F4A7C15ull : a.seed;
}
// the same counter-based mask as the other dropout kernels of the library
__device__ __forceinline__ float rp_drop(unsigned long long seed, unsigned long long idx, float p) {
    unsigned long long z = idx + seed * 0x9E3779B97F4A7C15ull + 0xD1B54A32D192ED03ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    z = z ^ (z >> 31);
    const float u = (float)(z >> 40) * (1.0f / 16777216.0f);
    return u >= p ? 1.0f / (1.0f - p) : 0.f;
}

// c(p) = p + (p / W)(W - 1); the quotient by a multiplication (rp_fill: exact for maps of up to 2^22 tokens, and 0 where there
// is one row, or one column and so no step)
__device__ __forceinline__ int rp_c(const RpArgs& a, int p) { return p + (int)__umulhi((unsigned)p, a.inv_w) * (a.W - 1); }

// ------------------------------------------------------------------------------------------------
// Matrix operands. A Frag is 16 bytes of one row (8 bf16 or 4 fp32): lane (g = lane / 16, l = lane % 16) holds elements
// PER * g .. of row l in the current chunk of 4 * PER elements. Both operands of a product use the same assignment of elements
// to reduction indices, so any assignment is right; this one makes every operand load one 16-byte access.
// ------------------------------------------------------------------------------------------------
template <typename T>
struct RpOp;

template <>
struct RpOp<bf16_t> {
    typedef rp_bf16x8 Frag;
    typedef rp_bf16x8 Pair;    // two 16-row blocks of a D-layout result as one B operand (reduction length 32)
    typedef rp_bf16x8 TFrag;
    static constexpr int PER = 8, CHUNK = 32;
    static __device__ __forceinline__ rp_f32x4 dot(Frag a, Frag b, rp_f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ Pair pack(const rp_f32x4& x, const rp_f32x4& y) {
        return __builtin_bit_cast(Pair, make_uint4(pack_bf16x2(v2f{x[0], x[1]}), pack_bf16x2(v2f{x[2], x[3]}),
                                                   pack_bf16x2(v2f{y[0], y[1]}), pack_bf16x2(v2f{y[2], y[3]})));
    }
    // what pack rounded off x and y
    static __device__ __forceinline__ Pair rest(const rp_f32x4& x, const rp_f32x4& y, const Pair& p) {
        const uint4 w = __builtin_bit_cast(uint4, p);
        const v2f a = unpack_bf16x2(w.x), b = unpack_bf16x2(w.y), c = unpack_bf16x2(w.z), d = unpack_bf16x2(w.w);
        return pack(rp_f32x4{x[0] - a.x, x[1] - a.y, x[2] - b.x, x[3] - b.y}, rp_f32x4{y[0] - c.x, y[1] - c.y, y[2] - d.x, y[3] - d.y});
    }
    // A operand of a product over rows: rows ra .. ra+3 and rb .. rb+3 (per 16-lane group) of columns col0 .. col0+15.
    // ra_ptr / rb_ptr: element [ra][col0] of this lane's group.
    static __device__ __forceinline__ TFrag load_t(const bf16_t* ra_ptr, const bf16_t* rb_ptr, int ld, int l) {
        typedef __attribute__((address_space(3))) rp_s16x4 lds4;
        const int at = (l >> 2) * ld + 4 * (l & 3);
        const rp_s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(ra_ptr + at));
        const rp_s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(rb_ptr + at));
        const rp_s16x8 r = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        return __builtin_bit_cast(TFrag, r);
    }
    static __device__ __forceinline__ rp_f32x4 dot_t(const TFrag& a, const Pair& b, rp_f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ float inner(Frag a, Frag b) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf((float)a[i], (float)b[i], s);
        return s;
    }
};

template <>
struct RpOp<float> {
    typedef rp_f32x4 Frag;
    struct Pair {
        rp_f32x4 x, y;
    };
    typedef Pair TFrag;
    static constexpr int PER = 4, CHUNK = 16;
    static __device__ __forceinline__ rp_f32x4 dot(Frag a, Frag b, rp_f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ Pair pack(const rp_f32x4& x, const rp_f32x4& y) { return {x, y}; }
    static __device__ __forceinline__ TFrag load_t(const float* ra_ptr, const float* rb_ptr, int ld, int l) {
        TFrag r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            r.x[i] = ra_ptr[i * ld + l];
            r.y[i] = rb_ptr[i * ld + l];
        }
        return r;
    }
    static __device__ __forceinline__ rp_f32x4 dot_t(const TFrag& a, const Pair& b, rp_f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x[i], b.x[i], c, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.y[i], b.y[i], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ float inner(Frag a, Frag b) {
        return fmaf(a[0], b[0], fmaf(a[1], b[1], fmaf(a[2], b[2], a[3] * b[3])));
    }
};

template <typename T, int DP>
struct RpDim {
    static constexpr int ES = (int)sizeof(T), PER = RpOp<T>::PER;
    static constexpr int NCH = (DP + RpOp<T>::CHUNK - 1) / RpOp<T>::CHUNK;   // operand chunks of a row
    static constexpr int LD = NCH * RpOp<T>::CHUNK + PER;                    // LDS row stride: 16 bytes of padding
    static constexpr int CPR = DP / PER;                                     // 16-byte pieces of a staged row
    // keys that the query kernels stage between two barriers: the fixed cost of a round of staging is a third of a 64-key tile's
    // instructions, so two tiles share it where registers and LDS allow
    static constexpr int HALVES = ES == 2 && DP <= 64 ? 2 : 1, STAGE = HALVES * RP_TILE;
    static constexpr int DB = DP / 16;                                       // 16-wide output blocks
    static constexpr bool EARLY = ES == 2 && DP <= 64;                       // registers for operands requested ahead
};

// 16-byte pieces of one row for this lane: elements beyond D are zeros (D is a multiple of 8)
template <typename T, int DP>
__device__ __forceinline__ void rp_row_frags(const T* row, bool ok, int D, int g, typename RpOp<T>::Frag (&f)[RpDim<T, DP>::NCH]) {
    typedef typename RpOp<T>::Frag Frag;
#pragma unroll
    for (int s = 0; s < RpDim<T, DP>::NCH; ++s) {
        const int col = s * RpOp<T>::CHUNK + g * RpOp<T>::PER;
        f[s] = ok && col < D ? *reinterpret_cast<const Frag*>(row + col) : Frag{};
    }
}

// One tile of rows on its way to LDS, kept in registers while the tile before it is worked on; a group of 256 threads, tid its
// thread. The loads are unconditional (rows past the end read the last row, columns past D the first): what counts is
// decided when the tile is put down. Their addresses are one scalar per tile plus 32-bit offsets that never change.
template <typename T, int DP, int ROWS>
struct RpTile {
    static constexpr int CPR = RpDim<T, DP>::CPR, NST = (ROWS * CPR + 255) / 256, WORDS = ROWS / 64;   // 16-byte pieces per thread
    uint4 r[NST];
    unsigned off[NST];   // bytes
    __device__ __forceinline__ void init(long long st, int D, int tid) {
#pragma unroll
        for (int i = 0; i < NST; ++i) {
            const int id = i * 256 + tid, row = min(id / CPR, ROWS - 1), col = (id % CPR) * RpOp<T>::PER;
            off[i] = ((unsigned)row * (unsigned)st + (unsigned)(col < D ? col : 0)) * (unsigned)sizeof(T);
        }
    }
    // rows first .. first + ROWS - 1 of src (row stride st), of `limit` rows in all
    __device__ __forceinline__ void fetch(const T* src, long long st, int first, int limit, int D, int tid) {
        const char* base = reinterpret_cast<const char*>(src + (long long)first * st);
        if (first + ROWS <= limit) {
#pragma unroll
            for (int i = 0; i < NST; ++i) r[i] = *reinterpret_cast<const uint4*>(base + off[i]);
        } else {
#pragma unroll
            for (int i = 0; i < NST; ++i) {
                const int id = i * 256 + tid, row = min(id / CPR, limit - 1 - first), col = (id % CPR) * RpOp<T>::PER;
                r[i] = *reinterpret_cast<const uint4*>(base + ((unsigned)row * (unsigned)st + (unsigned)(col < D ? col : 0)) * (unsigned)sizeof(T));
            }
        }
    }
    // bit i of valid (64 to a word) clear: row i becomes zeros. Columns past D are not written (rp_zero_pad). INS: extra elements after every
    // 16 rows
    template <int INS>
    __device__ __forceinline__ void put(T* lds, const unsigned long long (&valid)[WORDS], int D, int tid) const {
        if (valid[0] == ~0ull && valid[WORDS - 1] == ~0ull) {
#pragma unroll
            for (int i = 0; i < NST; ++i)
                if (used(i, D, tid)) *place<INS>(lds, i, tid) = r[i];
        } else {
#pragma unroll
            for (int i = 0; i < NST; ++i)
                if (used(i, D, tid)) {
                    const int row = (i * 256 + tid) / CPR;
                    const unsigned long long word = WORDS == 1 || row < 64 ? valid[0] : valid[WORDS - 1];
                    *place<INS>(lds, i, tid) = (word >> (row & 63)) & 1 ? r[i] : make_uint4(0u, 0u, 0u, 0u);
                }
        }
    }
    static __device__ __forceinline__ bool used(int i, int D, int tid) {
        const int id = i * 256 + tid;
        return ((ROWS * CPR) % 256 == 0 || id < ROWS * CPR) && (id % CPR) * RpOp<T>::PER < D;
    }
    template <int INS>
    static __device__ __forceinline__ uint4* place(T* lds, int i, int tid) {
        const int id = i * 256 + tid, row = id / CPR;
        return reinterpret_cast<uint4*>(lds + row * RpDim<T, DP>::LD + (row >> 4) * INS + (id - row * CPR) * RpOp<T>::PER);
    }
};

// a value loaded before a loop is waited for here: without it the wait falls on its first use inside the loop, where it also
// waits for whatever the loop has in flight
template <typename V>
__device__ __forceinline__ void rp_settle(V& v) {
    asm volatile("" : "+v"(v));
}

// Four channels of the output, and of what rounding took off them where the backward will want it.
template <typename T>
__device__ __forceinline__ void rp_store_out(const RpArgs& a, size_t at, rp_f32x4 x) {
    store4<T>((T*)a.o + at, {x[0], x[1], x[2], x[3]});
    if (sizeof(T) == 2 && a.o_low) {
        rp_f32x4 y;
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = x[r] - to_f32<T>(from_f32<T>(x[r]));
        store4<T>((T*)a.o_low + at, {y[0], y[1], y[2], y[3]});
    }
}

// Barrier between the waves' LDS work on one tile and the next. The wait is explicit because LDS additions return nothing that a
// later instruction would wait for, and the compiler has been seen to leave none of its own in front of the barrier at a loop's
// top: the ring below was then read before the last additions had arrived.
__device__ __forceinline__ void rp_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __syncthreads();
}

__device__ __forceinline__ void rp_lds_add(double* p, float v) {
    __hip_atomic_fetch_add(p, (double)v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}

enum { RP_FWD, RP_BWD_Q, RP_BWD_KV };
// Waves a SIMD has room for: the most that leave a kernel with at most a few registers in scratch (48 bytes at most). Asking for two
// already keeps the compiler from spreading over the accumulation registers, whose moves cost issue slots (38x38 maps, batch
// 4, 8 heads of 64: dK/dV 140 -> 103 us, 110 since its weights are two numbers, forward unchanged).
constexpr int rp_waves(int what, bool half, int DP, int cols) {
    if (what == RP_FWD)
        return half ? (cols == 1 ? (DP <= 32 ? 4 : DP <= 64 ? 3 : 2) : 2) : (DP <= 32 ? 4 : DP <= 64 ? 3 : 2);
    if (what == RP_BWD_Q) return half ? (cols == 1 ? (DP <= 32 ? 4 : DP <= 64 ? 3 : 2) : (DP <= 32 ? 3 : 2)) : (DP <= 32 ? 4 : DP <= 96 ? 2 : 1);
    return half ? (cols == 1 ? (DP <= 32 ? 4 : DP <= 64 ? 3 : 2) : (DP <= 16 ? 3 : 2)) : (DP <= 16 ? 4 : DP <= 32 ? 3 : DP <= 64 ? 2 : 1);
}

// columns between D and the padded reduction length are read as operands and never staged: zero once
template <typename T, int DP, int INS, int ROWS>
__device__ __forceinline__ void rp_zero_pad(T* lds, int D, int tid) {
    const int pad = RpDim<T, DP>::NCH * RpOp<T>::CHUNK - D;
    if (pad > 0)
#pragma unroll 1
        for (int i = tid; i < ROWS * pad; i += 256) {
            const int row = i / pad;
            lds[row * RpDim<T, DP>::LD + (row >> 4) * INS + D + (i - row * pad)] = from_f32<T>(0.f);
        }
}

// reductions over the four lanes l, l + 16, l + 32, l + 48 that share a column, in all of them: the row swaps leave the two halves
// of each pair in the two results
template <typename F>
__device__ __forceinline__ float rp_cross(float v, F f) {
    typedef unsigned u2 __attribute__((ext_vector_type(2)));
    u2 t = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(t[0]), __uint_as_float(t[1]));
    t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
__device__ __forceinline__ float rp_xor_max(float v) {
    return rp_cross(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float rp_xor_sum(float v) {
    return rp_cross(v, [](float a, float b) { return a + b; });
}

// A row's statistics for the backward pass: P = exp2((acc - max) * scale * log2(e) - log2(sum)). The maximum is subtracted before
// anything else, so that rows whose scores are all at the lowest value come out right (their maximum times a constant, rounded,
// would be off by more than any exponent); a row without keys gets an infinite sum, and so weights of zero.
__device__ __forceinline__ float2 rp_stat(float m, float total) {
    return total == 0.f ? make_float2(0.f, INFINITY) : make_float2(m, __builtin_amdgcn_logf(total));
}

// this lane's key of the tile at k0: its mask byte (1 without a mask), and the tile's existing keys as bits
__device__ __forceinline__ int rp_mask_byte(const RpArgs& a, int b, int k0) {
    return a.mask ? a.mask[(size_t)b * a.Lk + min(k0 + (int)(threadIdx.x & 63), a.Lk - 1)] : 1;
}
__device__ __forceinline__ unsigned long long rp_valid(const RpArgs& a, int k0, int byte) {
    return __ballot(byte != 0 && k0 + (int)(threadIdx.x & 63) < a.Lk);
}

// Which block (of `per` blocks of each (image, head)) a workgroup works on. Consecutive hardware workgroup ids go to the eight XCDs
// in turn; the blocks of one (image, head) stay on one XCD, whose L2 then holds that head's keys and values. Images are dealt to
// the XCDs in turn when their number is a multiple of eight (the heads of a packed token share cache lines: 10x10 maps, batch 128,
// 8 heads of 48: forward 20 us, 23 with heads dealt out), else (image, head)s are (an image that is masked out then costs
// every XCD the same: 38x38 maps, batch 4, one of them empty: forward 46 us, 48 with a run for each XCD), else each XCD gets an
// equal run of blocks. (Times from before P was split in two numbers.) The grid is a multiple of 8; ids past the last block have
// nothing to do.
__device__ __forceinline__ int rp_block(const RpArgs& a, int per) {
    const int id = blockIdx.x, bhs = a.B * a.heads;
    if (bhs & 7) return (id & 7) * ((int)gridDim.x >> 3) + (id >> 3);
    const int unit = a.B & 7 ? per : per * a.heads, j = id >> 3, q = j / unit;
    return (q * 8 + (id & 7)) * unit + (j - q * unit);
}

// ------------------------------------------------------------------------------------------------
// bias[h][o] = table[bucket[o]][h] / scale. Finite values stay finite (the largest ones are clamped): a table entry at the
// type's lowest value is a very low score, not a forbidden one.
// ------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void relpos_expand_kernel(const float* __restrict__ table, const int* __restrict__ bucket,
                                                            int n_off, int heads, float inv_scale, float limit,
                                                            float* __restrict__ bias) {
    const int o = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y;
    if (o >= n_off) return;
    float t = table[(size_t)bucket[o] * heads + h];
    if (fabsf(t) < INFINITY) t = fminf(fmaxf(t, -limit), limit) * inv_scale;
    bias[(size_t)h * n_off + o] = t;
}

// the bias window of one tile on its way to LDS
struct RpWindow {
    float r[2];
    __device__ __forceinline__ void fetch(const float* src, int n, int tid) {
#pragma unroll
        for (int i = 0; i < 2; ++i) r[i] = src[min(i * 256 + tid, n - 1)];
    }
    __device__ __forceinline__ void put(float* dst, const float* src, int n, int tid) const {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i * 256 + tid < n) dst[i * 256 + tid] = r[i];
#pragma unroll 1
        for (int i = 512 + tid; i < n; i += 256) dst[i] = src[i];
    }
};
// four entries of the window: c4 holds byte offsets of four rows, cq that of the column
__device__ __forceinline__ rp_f32x4 rp_bias4(const float* bw, const int4& c4, int cq) {
    const char* p = reinterpret_cast<const char*>(bw) - cq;
    return rp_f32x4{*reinterpret_cast<const float*>(p + c4.x), *reinterpret_cast<const float*>(p + c4.y),
                    *reinterpret_cast<const float*>(p + c4.z), *reinterpret_cast<const float*>(p + c4.w)};
}

// ------------------------------------------------------------------------------------------------
// forward: a workgroup owns 64 * QB queries of one (image, head), 16 * QB a wave, and walks the keys in tiles of 64 with the
// running maximum and sum of a softmax. With several splits (few queries, many keys) it walks one range of the tiles and
// leaves an unnormalised partial result.
// ------------------------------------------------------------------------------------------------
template <typename T, int DP, int QB>
__global__ __launch_bounds__(256, rp_waves(RP_FWD, sizeof(T) == 2, DP, QB)) void relpos_fwd_kernel(RpArgs a) {
    typedef RpOp<T> Op;
    typedef RpDim<T, DP> Dim;
    constexpr int LD = Dim::LD, QT = 64 * QB, ST = Dim::STAGE, HV = Dim::HALVES;
    extern __shared__ __attribute__((aligned(16))) char rp_sm[];
    const int tid = threadIdx.x;
    T* Ks = reinterpret_cast<T*>(rp_sm);
    T* Vs = Ks + ST * LD;
    int* ck = reinterpret_cast<int*>(Vs + ST * LD);
    float* cap = reinterpret_cast<float*>(ck + ST);   // scores end at this: -inf for a key that does not exist
    float* bw = cap + ST;
    const int qtiles = (a.Lq + QT - 1) / QT, id = rp_block(a, qtiles);
    if (id >= a.B * a.heads * qtiles) return;
    const int bh = id / qtiles, b = bh / a.heads, h = bh - b * a.heads, q0 = (id - bh * qtiles) * QT;
    const int lane = tid & 63, wave = tid >> 6, l = lane & 15, g = lane >> 4;
    const T* kp = (const T*)a.k + b * a.sk.b + h * a.sk.h;
    const T* vp = (const T*)a.v + b * a.sv.b + h * a.sv.h;
    const float* bias = a.bias + (size_t)h * a.n_off;
    const int q_hi = min(q0 + QT, a.Lq) - 1;
    const int cq_lo = rp_c(a, a.q_start + q0), cq_hi = rp_c(a, a.q_start + q_hi);

    typename Op::Frag qf[QB][Dim::NCH];
    int qi[QB], cq[QB];
    float m[QB], sum[QB];
    rp_f32x4 o[QB][Dim::DB];
#pragma unroll
    for (int i = 0; i < QB; ++i) {
        qi[i] = q0 + (wave * QB + i) * 16 + l;
        cq[i] = 4 * (rp_c(a, a.q_start + min(qi[i], q_hi)) - cq_hi);
        rp_row_frags<T, DP>((const T*)a.q + b * a.sq.b + (long long)min(qi[i], q_hi) * a.sq.t + h * a.sq.h, qi[i] < a.Lq, a.D, g, qf[i]);
        m[i] = -INFINITY;
        sum[i] = 0.f;
#pragma unroll
        for (int d = 0; d < Dim::DB; ++d) o[i][d] = rp_f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int i = 0; i < QB; ++i)
#pragma unroll
        for (int c = 0; c < Dim::NCH; ++c) rp_settle(qf[i][c]);
    const bool idle = q0 + wave * QB * 16 >= a.Lq;   // a wave without queries only helps to stage
    const unsigned long long seed = a.pdrop > 0.f ? rp_seed(a) : 0ull;
    rp_zero_pad<T, DP, 0, Dim::STAGE>(Ks, a.D, tid);
    rp_zero_pad<T, DP, 0, Dim::STAGE>(Vs, a.D, tid);

    RpTile<T, DP, ST> kt, vt;
    kt.init(a.sk.t, a.D, tid);
    vt.init(a.sv.t, a.D, tid);
    RpWindow wt;
    unsigned long long valid[HV];
    int byte[HV], ck_lo = 0, n_win = 0, base = 0;
    auto fetch = [&](int t) {
        const int k0 = t * ST;
#pragma unroll
        for (int i = 0; i < HV; ++i) byte[i] = rp_mask_byte(a, b, k0 + 64 * i);
        kt.fetch(kp, a.sk.t, k0, a.Lk, a.D, tid);
        vt.fetch(vp, a.sv.t, k0, a.Lk, a.D, tid);
        ck_lo = rp_c(a, k0);
        base = ck_lo - cq_hi + a.off;
        n_win = rp_c(a, min(k0 + ST, a.Lk) - 1) - ck_lo + cq_hi - cq_lo + 1;
        wt.fetch(bias + base, n_win, tid);
    };
    const int t1 = (int)((long long)a.tiles * (blockIdx.y + 1) / a.splits);
    int t = (int)((long long)a.tiles * blockIdx.y / a.splits);
    if (t < t1) fetch(t);
    for (; t < t1; ++t) {
        rp_barrier();
#pragma unroll
        for (int i = 0; i < HV; ++i) valid[i] = rp_valid(a, t * ST + 64 * i, byte[i]);
        kt.template put<0>(Ks, valid, a.D, tid);
        vt.template put<0>(Vs, valid, a.D, tid);
        wt.put(bw, bias + base, n_win, tid);
        if (tid < ST) {
            ck[tid] = 4 * (rp_c(a, min(t * ST + tid, a.Lk - 1)) - ck_lo);
            cap[tid] = ((tid < 64 ? valid[0] : valid[HV - 1]) >> (tid & 63)) & 1 ? INFINITY : -INFINITY;
        }
        rp_barrier();
        if (t + 1 < t1) fetch(t + 1);
        if (idle) continue;
#pragma unroll 1
        for (int hv = 0; hv < HV; ++hv) {
            const unsigned long long here = HV == 1 || hv == 0 ? valid[0] : valid[HV - 1];
            if (here == 0ull) continue;
            const T *Kh = Ks + hv * RP_TILE * LD, *Vh = Vs + hv * RP_TILE * LD;
            const int* ckh = ck + hv * RP_TILE;
            rp_f32x4 s[4][QB];
#pragma unroll
            for (int kb = 0; kb < 4; ++kb) {
                const int4 c4 = *reinterpret_cast<const int4*>(ckh + kb * 16 + g * 4);
#pragma unroll
                for (int i = 0; i < QB; ++i) s[kb][i] = rp_bias4(bw, c4, cq[i]);
            }
#pragma unroll
            for (int c = 0; c < Dim::NCH; ++c)
#pragma unroll
                for (int kb = 0; kb < 4; ++kb) {
                    const typename Op::Frag kf = *reinterpret_cast<const typename Op::Frag*>(Kh + (kb * 16 + l) * LD + c * Op::CHUNK + g * Op::PER);
#pragma unroll
                    for (int i = 0; i < QB; ++i) s[kb][i] = Op::dot(kf, qf[i][c], s[kb][i]);
                }
            // the value operands are requested here, so that they arrive while the softmax runs
            typename Op::TFrag vf[2][Dim::DB];
            auto values = [&](int kk) {
#pragma unroll
                for (int d = 0; d < Dim::DB; ++d) {
                    const T* v0 = Vh + (kk * 32 + g * 4) * LD + d * 16;
                    vf[kk][d] = Op::load_t(v0, v0 + 16 * LD, LD, l);
                }
            };
            if constexpr (Dim::EARLY) {
                values(0);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (here != ~0ull) {
#pragma unroll
                for (int kb = 0; kb < 4; ++kb) {
                    const rp_f32x4 c4 = *reinterpret_cast<const rp_f32x4*>(cap + hv * RP_TILE + kb * 16 + g * 4);
#pragma unroll
                    for (int i = 0; i < QB; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[kb][i][r] = fminf(s[kb][i][r], c4[r]);
                }
            }
#pragma unroll
            for (int i = 0; i < QB; ++i) {
                float mx = -INFINITY;
#pragma unroll
                for (int kb = 0; kb < 4; ++kb)
#pragma unroll
                    for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[kb][i][r]);
                mx = fmaxf(m[i], rp_xor_max(mx));
                const float use = mx == -INFINITY ? 0.f : mx;
                if (__any(mx > m[i])) {
                    const float alpha = __builtin_amdgcn_exp2f((m[i] - use) * a.sl2);
                    sum[i] *= alpha;
#pragma unroll
                    for (int d = 0; d < Dim::DB; ++d) o[i][d] *= alpha;
                }
                m[i] = mx;
                // one FMA where the rounding of use * sl2 cannot matter, the difference first where it would
                if (!__any(fabsf(use) * a.sl2 > RP_FAR)) {
                    const float shift = use * a.sl2;
#pragma unroll
                    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[kb][i][r] = __builtin_amdgcn_exp2f(fmaf(s[kb][i][r], a.sl2, -shift));
                } else {
#pragma unroll
                    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[kb][i][r] = __builtin_amdgcn_exp2f((s[kb][i][r] - use) * a.sl2);
                }
                float part[4];
#pragma unroll
                for (int kb = 0; kb < 4; ++kb) part[kb] = (s[kb][i][0] + s[kb][i][1]) + (s[kb][i][2] + s[kb][i][3]);
                sum[i] += (part[0] + part[1]) + (part[2] + part[3]);
                if (a.pdrop > 0.f) {
                    const unsigned long long at = ((unsigned long long)bh * a.Lq + qi[i]) * a.Lk + t * ST + hv * RP_TILE + g * 4;
#pragma unroll
                    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[kb][i][r] *= rp_drop(seed, at + kb * 16 + r, a.pdrop);
                }
            }
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                typename Op::Pair p[QB];
#pragma unroll
                for (int i = 0; i < QB; ++i) p[i] = Op::pack(s[2 * kk][i], s[2 * kk + 1][i]);
                typename Op::Pair more[QB];
                if constexpr (sizeof(T) == 2)
#pragma unroll
                    for (int i = 0; i < QB; ++i) more[i] = Op::rest(s[2 * kk][i], s[2 * kk + 1][i], p[i]);
                if (!Dim::EARLY) values(kk);
                else if (kk == 0) values(1);
#pragma unroll
                for (int d = 0; d < Dim::DB; ++d) {
#pragma unroll
                    for (int i = 0; i < QB; ++i) o[i][d] = Op::dot_t(vf[kk][d], p[i], o[i][d]);
                    if constexpr (sizeof(T) == 2)
#pragma unroll
                        for (int i = 0; i < QB; ++i) o[i][d] = Op::dot_t(vf[kk][d], more[i], o[i][d]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < QB; ++i) {
        const float total = rp_xor_sum(sum[i]);
        if (qi[i] >= a.Lq) continue;
        const size_t row = (size_t)bh * a.Lq + qi[i];
        if (a.splits > 1) {
            const size_t prow = (size_t)blockIdx.y * a.B * a.heads * a.Lq + row;
            if (g == 0) {
                a.pml[2 * prow] = m[i];
                a.pml[2 * prow + 1] = total;
            }
#pragma unroll
            for (int d = 0; d < Dim::DB; ++d) {
                const int col = d * 16 + g * 4;
                if (col < a.D) *reinterpret_cast<rp_f32x4*>(a.po + prow * a.D + col) = o[i][d];
            }
            continue;
        }
        const float inv = total == 0.f ? 0.f : 1.0f / total;   // a row without keys is zero
        if (a.stat && g == 0) a.stat[row] = rp_stat(m[i], total);
        const size_t at = (((size_t)b * a.Lq + qi[i]) * a.heads + h) * a.D;
#pragma unroll
        for (int d = 0; d < Dim::DB; ++d) {
            const int col = d * 16 + g * 4;
            if (col < a.D) rp_store_out<T>(a, at + col, o[i][d] * inv);
        }
    }
}

// ------------------------------------------------------------------------------------------------
// forward of at most 16 queries (one new token against a long series): reading the keys and values is all the work. Waves take
// chunks of KEYS keys in turn and never wait for each other: a wave's keys go from memory into the operand registers, its values
// through a piece of LDS of its own for the transposing read, and the next chunk is requested before the softmax of this one. The four
// waves of a workgroup share one head's keys or read four neighbouring heads (rp_plan); the waves of a head are joined in LDS at the end,
// workgroups by relpos_join_few_kernel. One query against 16384 keys, batch 8, 8 heads of 64 in bf16, keys and values not in any
// cache: 52 us = 5.2 TB/s with four heads a workgroup, 56 with two, 62 with one (128-byte pieces of memory), 64 with the tiled kernel
// above, of whose four waves one works; 155 keys, 8 heads of 48 in fp32: 7.5 us, 11.6 with that kernel.
// ------------------------------------------------------------------------------------------------
#define RP_FEW 16
template <typename T, int DP>
struct RpFew {
    static constexpr int KEYS = DP * (int)sizeof(T) <= 128 ? 64 : 32, LD = RpDim<T, DP>::LD, PIECES = KEYS * RpDim<T, DP>::CPR / 64;
    static constexpr size_t LDS = 4 * (size_t)KEYS * LD * sizeof(T);
    static_assert(LDS >= 4 * RP_FEW * (DP + 2) * sizeof(float), "the joining of the waves does not fit");
};
static int rp_few_keys(int dtype, int DP) { return DP * (dtype == MIA_BF16 ? 2 : 4) <= 128 ? 64 : 32; }

// LDS that only this wave's lanes share: its accesses are carried out in order, the compiler has to keep the order too
__device__ __forceinline__ void rp_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <typename T, int DP>
__global__ __launch_bounds__(256, DP * (int)sizeof(T) <= 64 ? 3 : DP * (int)sizeof(T) <= 384 ? 2 : 1) void relpos_few_kernel(RpArgs a) {
    typedef RpOp<T> Op;
    typedef RpDim<T, DP> Dim;
    typedef RpFew<T, DP> Few;
    constexpr int LD = Dim::LD, KEYS = Few::KEYS, KB = KEYS / 16, CPR = Dim::CPR;
    __shared__ __attribute__((aligned(16))) char sm[Few::LDS];
    const int groups = a.heads / a.few, ranks = 4 / a.few, split = blockIdx.x / (a.B * groups), id = blockIdx.x - split * a.B * groups;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 15, g = lane >> 4;
    const int b = id / groups, h0 = (id - b * groups) * a.few, h = h0 + wave % a.few;
    const T* kp = (const T*)a.k + b * a.sk.b + h * a.sk.h;
    const T* vp = (const T*)a.v + b * a.sv.b + h * a.sv.h;
    T* Vs = reinterpret_cast<T*>(sm) + wave * KEYS * LD;
    const int query = min(l, a.Lq - 1);
    const float* bias = a.bias + (size_t)h * a.n_off + (a.off - rp_c(a, a.q_start + query));   // of this lane's query, by c(key)
    typename Op::Frag qf[Dim::NCH];
    rp_row_frags<T, DP>((const T*)a.q + b * a.sq.b + (long long)query * a.sq.t + h * a.sq.h, l < a.Lq, a.D, g, qf);
    const unsigned long long seed = a.pdrop > 0.f ? rp_seed(a) : 0ull;

    typename Op::Frag kf[KB][Dim::NCH];
    uint4 vr[Few::PIECES];
    float br[KB][4];
    int byte = 0;
    auto fetch = [&](int t) {
        const int k0 = t * KEYS;
        byte = rp_mask_byte(a, b, k0);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const T* row = kp + (long long)min(k0 + kb * 16 + l, a.Lk - 1) * a.sk.t;
#pragma unroll
            for (int c = 0; c < Dim::NCH; ++c) {
                const int col = c * Op::CHUNK + g * Op::PER;
                kf[kb][c] = *reinterpret_cast<const typename Op::Frag*>(row + (col < a.D ? col : 0));
            }
        }
#pragma unroll
        for (int i = 0; i < Few::PIECES; ++i) {
            const int piece = i * 64 + lane, row = piece / CPR, col = (piece - row * CPR) * Op::PER;
            vr[i] = *reinterpret_cast<const uint4*>(vp + (long long)min(k0 + row, a.Lk - 1) * a.sv.t + (col < a.D ? col : 0));
        }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r) br[kb][r] = bias[rp_c(a, min(k0 + kb * 16 + g * 4 + r, a.Lk - 1))];
    };
    float m = -INFINITY, sum = 0.f;
    rp_f32x4 o[Dim::DB];
#pragma unroll
    for (int d = 0; d < Dim::DB; ++d) o[d] = rp_f32x4{0.f, 0.f, 0.f, 0.f};
    const int t1 = (int)((long long)a.tiles * (split + 1) / a.splits);
    int t = (int)((long long)a.tiles * split / a.splits) + wave / a.few;
    if (t < t1) fetch(t);
    for (; t < t1; t += ranks) {
        const unsigned long long all = KEYS == 64 ? ~0ull : (1ull << KEYS) - 1, here = rp_valid(a, t * KEYS, byte) & all;
        rp_f32x4 s[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) s[kb] = rp_f32x4{br[kb][0], br[kb][1], br[kb][2], br[kb][3]};
        // columns past D are zero in the query's operand; in the keys' they repeat the first ones, which may not be finite
#pragma unroll
        for (int c = 0; c < Dim::NCH; ++c)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                if (c * Op::CHUNK + g * Op::PER >= a.D) kf[kb][c] = typename Op::Frag{};
                s[kb] = Op::dot(kf[kb][c], qf[c], s[kb]);
            }
        rp_wave_sync();
#pragma unroll
        for (int i = 0; i < Few::PIECES; ++i) {
            const int piece = i * 64 + lane, row = piece / CPR;
            *reinterpret_cast<uint4*>(Vs + row * LD + (piece - row * CPR) * Op::PER) = (here >> row) & 1 ? vr[i] : make_uint4(0u, 0u, 0u, 0u);
        }
        rp_wave_sync();
        if (t + ranks < t1) fetch(t + ranks);
        if (here == 0ull) continue;
        if (here != all) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[kb][r] = (here >> (kb * 16 + g * 4 + r)) & 1 ? s[kb][r] : -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[kb][r]);
        mx = fmaxf(m, rp_xor_max(mx));
        const float use = mx == -INFINITY ? 0.f : mx, alpha = __builtin_amdgcn_exp2f((m - use) * a.sl2);
        sum *= alpha;
#pragma unroll
        for (int d = 0; d < Dim::DB; ++d) o[d] *= alpha;
        m = mx;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
            for (int r = 0; r < 4; ++r) s[kb][r] = __builtin_amdgcn_exp2f((s[kb][r] - use) * a.sl2);
            sum += (s[kb][0] + s[kb][1]) + (s[kb][2] + s[kb][3]);
        }
        if (a.pdrop > 0.f) {
            const unsigned long long at = ((unsigned long long)(b * a.heads + h) * a.Lq + query) * a.Lk + (unsigned)(t * KEYS) + g * 4;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[kb][r] *= rp_drop(seed, at + kb * 16 + r, a.pdrop);
        }
#pragma unroll
        for (int kk = 0; kk < KB / 2; ++kk) {
            const typename Op::Pair p = Op::pack(s[2 * kk], s[2 * kk + 1]);
            typename Op::Pair more;
            if constexpr (sizeof(T) == 2) more = Op::rest(s[2 * kk], s[2 * kk + 1], p);
#pragma unroll
            for (int d = 0; d < Dim::DB; ++d) {
                const T* v0 = Vs + (kk * 32 + g * 4) * LD + d * 16;
                const typename Op::TFrag vf = Op::load_t(v0, v0 + 16 * LD, LD, l);
                o[d] = Op::dot_t(vf, p, o[d]);
                if constexpr (sizeof(T) == 2) o[d] = Op::dot_t(vf, more, o[d]);
            }
        }
    }
    // maxima, sums and outputs of the waves of a head, joined in wave order
    sum = rp_xor_sum(sum);
    float* os = reinterpret_cast<float*>(sm);      // [wave][query][DP]
    float2* ml = reinterpret_cast<float2*>(os + 4 * RP_FEW * DP);
    __syncthreads();
    if (g == 0) ml[wave * RP_FEW + l] = make_float2(m, sum);
#pragma unroll
    for (int d = 0; d < Dim::DB; ++d) *reinterpret_cast<rp_f32x4*>(os + (wave * RP_FEW + l) * DP + d * 16 + g * 4) = o[d];
    __syncthreads();
    for (int i = threadIdx.x; i < a.few * a.Lq * (DP / 4); i += 256) {
        const int hq = i / (DP / 4), col = (i - hq * (DP / 4)) * 4, hh = hq / a.Lq, q = hq - hh * a.Lq;
        if (col >= a.D) continue;
        float top = -INFINITY, total = 0.f;
        for (int w = hh; w < 4; w += a.few) top = fmaxf(top, ml[w * RP_FEW + q].x);
        const float use = top == -INFINITY ? 0.f : top;
        rp_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int w = hh; w < 4; w += a.few) {
            const float2 x = ml[w * RP_FEW + q];
            const float weight = __builtin_amdgcn_exp2f((x.x - use) * a.sl2);
            total = fmaf(x.y, weight, total);
            acc += *reinterpret_cast<const rp_f32x4*>(os + (w * RP_FEW + q) * DP + col) * weight;
        }
        const size_t row = ((size_t)b * a.heads + h0 + hh) * a.Lq + q;
        if (a.splits > 1) {
            const size_t prow = (size_t)split * a.B * a.heads * a.Lq + row;
            if (col == 0) reinterpret_cast<float2*>(a.pml)[prow] = make_float2(top, total);
            *reinterpret_cast<rp_f32x4*>(a.po + prow * a.D + col) = acc;
        } else {
            const float inv = total == 0.f ? 0.f : 1.0f / total;
            rp_store_out<T>(a, (((size_t)b * a.Lq + q) * a.heads + h0 + hh) * a.D + col, acc * inv);
            if (a.stat && col == 0) a.stat[row] = rp_stat(top, total);
        }
    }
}

// Joins the partial results of relpos_few_kernel: few rows in many splits, so a workgroup per row, whose threads share the splits
// (64 rows of 64 in 16 splits: 5 us; 12 with a thread per four channels that walks the splits).
template <typename T, int DP>
__global__ __launch_bounds__(256) void relpos_join_few_kernel(RpArgs a) {
    constexpr int QUADS = DP <= 16 ? 4 : DP <= 32 ? 8 : DP <= 64 ? 16 : 32, LANES = 256 / QUADS;
    __shared__ rp_f32x4 os[LANES][QUADS];
    __shared__ float2 ml[LANES];
    const size_t rows = (size_t)a.B * a.heads * a.Lq, row = blockIdx.x;
    const int quad = threadIdx.x % QUADS, sl = threadIdx.x / QUADS, d = quad * 4;
    const float2* pml = reinterpret_cast<const float2*>(a.pml);
    float m = -INFINITY, total = 0.f;
    for (int s = sl; s < a.splits; s += LANES) m = fmaxf(m, pml[s * rows + row].x);
    float use = m == -INFINITY ? 0.f : m;
    rp_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s = sl; s < a.splits; s += LANES) {
        const float2 x = pml[s * rows + row];
        const float w = __builtin_amdgcn_exp2f((x.x - use) * a.sl2);
        total = fmaf(x.y, w, total);
        if (d < a.D) acc += *reinterpret_cast<const rp_f32x4*>(a.po + (s * rows + row) * a.D + d) * w;
    }
    os[sl][quad] = acc;
    if (quad == 0) ml[sl] = make_float2(m, total);
    __syncthreads();
    if (sl != 0 || d >= a.D) return;
    const int n = min(LANES, a.splits);
    m = -INFINITY;
    for (int i = 0; i < n; ++i) m = fmaxf(m, ml[i].x);
    use = m == -INFINITY ? 0.f : m;
    total = 0.f;
    acc = rp_f32x4{0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < n; ++i) {
        const float w = __builtin_amdgcn_exp2f((ml[i].x - use) * a.sl2);
        total = fmaf(ml[i].y, w, total);
        acc += os[i][quad] * w;
    }
    const size_t bh = row / a.Lq, b = bh / a.heads, h = bh - b * a.heads, t = row - bh * a.Lq;
    rp_store_out<T>(a, ((b * a.Lq + t) * a.heads + h) * a.D + d, acc * (total == 0.f ? 0.f : 1.0f / total));
    if (a.stat && d == 0) a.stat[row] = rp_stat(m, total);
}

// Joins the partial results of kernels that were split over the tokens they walk: a thread per four channels of a row, the
// partials of one row added in order of the splits.
//   RP_FWD    the running maxima and sums of the splits, their unnormalised outputs
//   RP_BWD_Q  dQ and the sums that make D exact
//   RP_BWD_KV dK and dV
template <typename T, int WHAT>
__global__ __launch_bounds__(256) void relpos_join_kernel(RpArgs a) {
    const int vecs = a.D >> 2, tokens = WHAT == RP_BWD_KV ? a.Lk : a.Lq;
    const size_t rows = (size_t)a.B * a.heads * tokens, i = (size_t)blockIdx.x * 256 + threadIdx.x, row = i / vecs;
    if (row >= rows) return;
    const int d = (int)(i - row * vecs) * 4;
    const size_t bh = row / tokens, b = bh / a.heads, h = bh - b * a.heads, t = row - bh * tokens;
    if constexpr (WHAT == RP_BWD_KV) {
        const size_t part = rows * a.D;
        rp_f32x4 k = {0.f, 0.f, 0.f, 0.f}, v = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < a.splits; ++s) {
            const float* p = a.po + 2 * s * part + row * a.D + d;
            k += *reinterpret_cast<const rp_f32x4*>(p);
            v += *reinterpret_cast<const rp_f32x4*>(p + part);
        }
        store4<T>((T*)a.dk + b * a.sdk.b + t * a.sdk.t + h * a.sdk.h + d, {k[0] * a.scale, k[1] * a.scale, k[2] * a.scale, k[3] * a.scale});
        store4<T>((T*)a.dv + b * a.sdv.b + t * a.sdv.t + h * a.sdv.h + d, {v[0], v[1], v[2], v[3]});
    } else {
        const float2* pml = reinterpret_cast<const float2*>(a.pml);
        float m = -INFINITY, total = 0.f;
        if (WHAT == RP_FWD)
            for (int s = 0; s < a.splits; ++s) m = fmaxf(m, pml[s * rows + row].x);
        const float use = m == -INFINITY ? 0.f : m;
        rp_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < a.splits; ++s) {
            const float2 ml = pml[s * rows + row];
            const float w = WHAT == RP_FWD ? __builtin_amdgcn_exp2f((ml.x - use) * a.sl2) : 1.f;
            total = fmaf(ml.y, w, total);
            acc += *reinterpret_cast<const rp_f32x4*>(a.po + (s * rows + row) * a.D + d) * w;
        }
        if (WHAT == RP_FWD) {
            const float inv = total == 0.f ? 0.f : 1.0f / total;
            rp_store_out<T>(a, ((b * a.Lq + t) * a.heads + h) * a.D + d, acc * inv);
            if (a.stat && d == 0) a.stat[row] = rp_stat(m, total);
        } else {
            store4<T>((T*)a.dq + b * a.sdq.b + t * a.sdq.t + h * a.sdq.h + d,
                      {acc[0] * a.scale, acc[1] * a.scale, acc[2] * a.scale, acc[3] * a.scale});
            if (d == 0) a.dsum[row] = pml[row].x + total;
        }
    }
}

// ------------------------------------------------------------------------------------------------
// backward, queries as columns: dQ and the exact D. The same walk as the forward.
//
// A row of dS sums to zero, so what the keys have in common drops out of dQ = dS K, but not out of what rounding dS to bf16, or an
// inexact D~, does to it. dS is therefore multiplied as two bf16 numbers, its rounding and what that took off, and the forward
// does the same with P (38x38 maps, batch 4, 8 heads of 64: 52 -> 57 us, forward 45 -> 49; 75x75, 4 heads of 32: 74 -> 87,
// forward 71 -> 86). The error of dQ is then that of its own last rounding, 1.7e-3; with single roundings it was 2.4e-3 for keys
// with nothing in common, 5.6e-3 for keys of mean 4 and deviation 1. dK and dV are sums over queries that cancel too, by
// chance: their products take P and dS as two numbers as well (2.4e-3 -> 1.7e-3 for 103 -> 109 us).
// ------------------------------------------------------------------------------------------------
template <typename T, int DP, int QB>
__global__ __launch_bounds__(256, rp_waves(RP_BWD_Q, sizeof(T) == 2, DP, QB)) void relpos_bwd_q_kernel(RpArgs a) {
    typedef RpOp<T> Op;
    typedef RpDim<T, DP> Dim;
    constexpr int LD = Dim::LD, QT = 64 * QB, ST = Dim::STAGE, HV = Dim::HALVES;
    extern __shared__ __attribute__((aligned(16))) char rp_sm[];
    const int tid = threadIdx.x;
    T* Ks = reinterpret_cast<T*>(rp_sm);
    T* Vs = Ks + ST * LD;
    int* ck = reinterpret_cast<int*>(Vs + ST * LD);
    float* cap = reinterpret_cast<float*>(ck + ST);   // scores end at this: -inf for a key that does not exist
    float* bw = cap + ST;
    const int qtiles = (a.Lq + QT - 1) / QT, id = rp_block(a, qtiles);
    if (id >= a.B * a.heads * qtiles) return;
    const int bh = id / qtiles, b = bh / a.heads, h = bh - b * a.heads, q0 = (id - bh * qtiles) * QT;
    const int lane = tid & 63, wave = tid >> 6, l = lane & 15, g = lane >> 4;
    const T* kp = (const T*)a.k + b * a.sk.b + h * a.sk.h;
    const T* vp = (const T*)a.v + b * a.sv.b + h * a.sv.h;
    const float* bias = a.bias + (size_t)h * a.n_off;
    const int q_hi = min(q0 + QT, a.Lq) - 1;
    const int cq_lo = rp_c(a, a.q_start + q0), cq_hi = rp_c(a, a.q_start + q_hi);

    typename Op::Frag qf[QB][Dim::NCH], gf[QB][Dim::NCH];
    int qi[QB], cq[QB];
    float mx[QB], lg[QB], shift[QB], D0[QB], extra[QB];
    bool far = false;
    rp_f32x4 dq[QB][Dim::DB];
#pragma unroll
    for (int i = 0; i < QB; ++i) {
        qi[i] = q0 + (wave * QB + i) * 16 + l;
        const int row = min(qi[i], q_hi);
        const bool ok = qi[i] < a.Lq;
        cq[i] = 4 * (rp_c(a, a.q_start + row) - cq_hi);
        rp_row_frags<T, DP>((const T*)a.q + b * a.sq.b + (long long)row * a.sq.t + h * a.sq.h, ok, a.D, g, qf[i]);
        const size_t orow = (((size_t)b * a.Lq + row) * a.heads + h) * a.D;
        typename Op::Frag of[Dim::NCH];
        rp_row_frags<T, DP>((const T*)a.dout + orow, ok, a.D, g, gf[i]);
        rp_row_frags<T, DP>((const T*)a.out + orow, ok, a.D, g, of);
        float d = 0.f;
#pragma unroll
        for (int c = 0; c < Dim::NCH; ++c) d += Op::inner(gf[i][c], of[c]);
        if (sizeof(T) == 2) {
            rp_row_frags<T, DP>((const T*)a.out_low + orow, ok, a.D, g, of);
#pragma unroll
            for (int c = 0; c < Dim::NCH; ++c) d += Op::inner(gf[i][c], of[c]);
        }
        D0[i] = rp_xor_sum(d);
        const float2 st = a.stat[(size_t)bh * a.Lq + row];
        mx[i] = st.x;
        lg[i] = ok ? st.y : INFINITY;
        extra[i] = 0.f;
#pragma unroll
        for (int c = 0; c < Dim::DB; ++c) dq[i][c] = rp_f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int i = 0; i < QB; ++i) {
#pragma unroll
        for (int c = 0; c < Dim::NCH; ++c) {
            rp_settle(qf[i][c]);
            rp_settle(gf[i][c]);
        }
        rp_settle(mx[i]);
        rp_settle(lg[i]);
        shift[i] = fmaf(mx[i], a.sl2, lg[i]);
        far |= fabsf(mx[i]) * a.sl2 > RP_FAR;
    }
    far = __any(far);
    const bool idle = q0 + wave * QB * 16 >= a.Lq;
    const unsigned long long seed = a.pdrop > 0.f ? rp_seed(a) : 0ull;
    rp_zero_pad<T, DP, 0, Dim::STAGE>(Ks, a.D, tid);
    rp_zero_pad<T, DP, 0, Dim::STAGE>(Vs, a.D, tid);

    RpTile<T, DP, ST> kt, vt;
    kt.init(a.sk.t, a.D, tid);
    vt.init(a.sv.t, a.D, tid);
    RpWindow wt;
    unsigned long long valid[HV];
    int byte[HV], ck_lo = 0, n_win = 0, base = 0;
    auto fetch = [&](int t) {
        const int k0 = t * ST;
#pragma unroll
        for (int i = 0; i < HV; ++i) byte[i] = rp_mask_byte(a, b, k0 + 64 * i);
        kt.fetch(kp, a.sk.t, k0, a.Lk, a.D, tid);
        vt.fetch(vp, a.sv.t, k0, a.Lk, a.D, tid);
        ck_lo = rp_c(a, k0);
        base = ck_lo - cq_hi + a.off;
        n_win = rp_c(a, min(k0 + ST, a.Lk) - 1) - ck_lo + cq_hi - cq_lo + 1;
        wt.fetch(bias + base, n_win, tid);
    };
    const int t1 = (int)((long long)a.tiles * (blockIdx.y + 1) / a.splits);
    int t = (int)((long long)a.tiles * blockIdx.y / a.splits);
    if (t < t1) fetch(t);
    for (; t < t1; ++t) {
        rp_barrier();
#pragma unroll
        for (int i = 0; i < HV; ++i) valid[i] = rp_valid(a, t * ST + 64 * i, byte[i]);
        kt.template put<0>(Ks, valid, a.D, tid);
        vt.template put<0>(Vs, valid, a.D, tid);
        wt.put(bw, bias + base, n_win, tid);
        if (tid < ST) {
            ck[tid] = 4 * (rp_c(a, min(t * ST + tid, a.Lk - 1)) - ck_lo);
            cap[tid] = ((tid < 64 ? valid[0] : valid[HV - 1]) >> (tid & 63)) & 1 ? INFINITY : -INFINITY;
        }
        rp_barrier();
        if (t + 1 < t1) fetch(t + 1);
        if (idle) continue;
#pragma unroll 1
        for (int hv = 0; hv < HV; ++hv) {
            const unsigned long long here = HV == 1 || hv == 0 ? valid[0] : valid[HV - 1];
            if (here == 0ull) continue;
            const T *Kh = Ks + hv * RP_TILE * LD, *Vh = Vs + hv * RP_TILE * LD;
            const int* ckh = ck + hv * RP_TILE;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                rp_f32x4 s[2][QB], ds[2][QB];   // ds: dP, then dS
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int4 c4 = *reinterpret_cast<const int4*>(ckh + (2 * kk + e) * 16 + g * 4);
#pragma unroll
                    for (int i = 0; i < QB; ++i) {
                        s[e][i] = rp_bias4(bw, c4, cq[i]);
                        ds[e][i] = rp_f32x4{0.f, 0.f, 0.f, 0.f};
                    }
                }
#pragma unroll
                for (int c = 0; c < Dim::NCH; ++c)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int at = ((2 * kk + e) * 16 + l) * LD + c * Op::CHUNK + g * Op::PER;
                        const typename Op::Frag kf = *reinterpret_cast<const typename Op::Frag*>(Kh + at);
                        const typename Op::Frag vf = *reinterpret_cast<const typename Op::Frag*>(Vh + at);
#pragma unroll
                        for (int i = 0; i < QB; ++i) {
                            s[e][i] = Op::dot(kf, qf[i][c], s[e][i]);
                            ds[e][i] = Op::dot(vf, gf[i][c], ds[e][i]);
                        }
                    }
                typename Op::TFrag kt_[Dim::DB];   // requested ahead of the exponentials
                if constexpr (Dim::EARLY) {
#pragma unroll
                    for (int d = 0; d < Dim::DB; ++d) {
                        const T* k0 = Kh + (kk * 32 + g * 4) * LD + d * 16;
                        kt_[d] = Op::load_t(k0, k0 + 16 * LD, LD, l);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (here != ~0ull) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const rp_f32x4 c4 = *reinterpret_cast<const rp_f32x4*>(cap + hv * RP_TILE + (2 * kk + e) * 16 + g * 4);
#pragma unroll
                        for (int i = 0; i < QB; ++i)
#pragma unroll
                            for (int r = 0; r < 4; ++r) s[e][i][r] = fminf(s[e][i][r], c4[r]);
                    }
                }
                if (a.pdrop > 0.f) {
#pragma unroll
                    for (int i = 0; i < QB; ++i) {
                        const unsigned long long at = ((unsigned long long)bh * a.Lq + qi[i]) * a.Lk + t * ST + hv * RP_TILE + kk * 32 + g * 4;
#pragma unroll
                        for (int e = 0; e < 2; ++e)
#pragma unroll
                            for (int r = 0; r < 4; ++r) ds[e][i][r] *= rp_drop(seed, at + e * 16 + r, a.pdrop);
                    }
                }
                if (far) {
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int i = 0; i < QB; ++i)
#pragma unroll
                            for (int r = 0; r < 4; ++r) s[e][i][r] = __builtin_amdgcn_exp2f(fmaf(s[e][i][r] - mx[i], a.sl2, -lg[i]));
                } else {
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int i = 0; i < QB; ++i)
#pragma unroll
                            for (int r = 0; r < 4; ++r) s[e][i][r] = __builtin_amdgcn_exp2f(fmaf(s[e][i][r], a.sl2, -shift[i]));
                }
#pragma unroll
                for (int i = 0; i < QB; ++i) {
                    float part[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) ds[e][i][r] = s[e][i][r] * (ds[e][i][r] - D0[i]);
                        part[e] = (ds[e][i][0] + ds[e][i][1]) + (ds[e][i][2] + ds[e][i][3]);
                    }
                    extra[i] += part[0] + part[1];
                }
                typename Op::Pair p[QB];
#pragma unroll
                for (int i = 0; i < QB; ++i) p[i] = Op::pack(ds[0][i], ds[1][i]);
                typename Op::Pair more[QB];
                if constexpr (sizeof(T) == 2)
#pragma unroll
                    for (int i = 0; i < QB; ++i) more[i] = Op::rest(ds[0][i], ds[1][i], p[i]);
#pragma unroll
                for (int d = 0; d < Dim::DB; ++d) {
                    if constexpr (!Dim::EARLY) {
                        const T* k0 = Kh + (kk * 32 + g * 4) * LD + d * 16;
                        kt_[d] = Op::load_t(k0, k0 + 16 * LD, LD, l);
                    }
#pragma unroll
                    for (int i = 0; i < QB; ++i) dq[i][d] = Op::dot_t(kt_[d], p[i], dq[i][d]);
                    if constexpr (sizeof(T) == 2)
#pragma unroll
                        for (int i = 0; i < QB; ++i) dq[i][d] = Op::dot_t(kt_[d], more[i], dq[i][d]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < QB; ++i) {
        const float more = rp_xor_sum(extra[i]);
        if (qi[i] >= a.Lq) continue;
        const size_t row = (size_t)bh * a.Lq + qi[i];
        if (a.splits > 1) {
            const size_t prow = (size_t)blockIdx.y * a.B * a.heads * a.Lq + row;
            if (g == 0) *reinterpret_cast<float2*>(a.pml + 2 * prow) = make_float2(D0[i], more);
#pragma unroll
            for (int d = 0; d < Dim::DB; ++d) {
                const int col = d * 16 + g * 4;
                if (col < a.D) *reinterpret_cast<rp_f32x4*>(a.po + prow * a.D + col) = dq[i][d];
            }
            continue;
        }
        if (g == 0) a.dsum[row] = D0[i] + more;
        T* out = (T*)a.dq + b * a.sdq.b + (long long)qi[i] * a.sdq.t + h * a.sdq.h;
#pragma unroll
        for (int d = 0; d < Dim::DB; ++d) {
            const int col = d * 16 + g * 4;
            if (col < a.D)
                store4<T>(out + col, {dq[i][d][0] * a.scale, dq[i][d][1] * a.scale, dq[i][d][2] * a.scale, dq[i][d][3] * a.scale});
        }
    }
}

// ------------------------------------------------------------------------------------------------
// backward, keys as columns: dK, dV and the bias gradient per offset. A workgroup owns 64 * KB keys of one (image, head), 16 *
// KB a wave, whose K and V operands stay in registers, and walks the queries in tiles of 64.
//
// Row a = 4 g + r of the m-th 16-row block of a tile is query 16 g + 4 m + r. In register r of a block the 64 lanes then hold
// four queries 16 apart against 16 consecutive keys: 64 different token distances, hence 64 different offsets. So one LDS
// add instruction never meets an address twice, and each wave adds its dS into an accumulator array of its OWN: the additions
// to one address come from one wave in program order, and the result does not depend on timing. The array is a ring over the
// offsets; offsets that later tiles cannot reach any more (queries only go up, so offsets only go down) are added over
// the waves in wave order and leave for the slab after every tile. The sums are doubles because LDS adds those at
// 11.5 cycles a wave instruction and floats at 194 (measured): 481 -> 152 us for this kernel on 38x38 maps, batch 4, 8 heads of 64.
// ------------------------------------------------------------------------------------------------
template <typename T, int DP, int KB>
__global__ __launch_bounds__(256, rp_waves(RP_BWD_KV, sizeof(T) == 2, DP, KB)) void relpos_bwd_kv_kernel(RpArgs a) {
    typedef RpOp<T> Op;
    typedef RpDim<T, DP> Dim;
    constexpr int LD = Dim::LD, KT = 64 * KB;
    constexpr int INS = 64 / (int)sizeof(T);   // 16 rows apart = 64 bytes further in the banks: the transposing reads' four row groups
    constexpr int TILE = RP_TILE * LD + 4 * INS;
    extern __shared__ __attribute__((aligned(16))) char rp_sm[];
    T* Qs = reinterpret_cast<T*>(rp_sm);
    T* Gs = Qs + TILE;
    float* ms = reinterpret_cast<float*>(Gs + TILE);
    float* ls = ms + RP_TILE;
    float* sh = ls + RP_TILE;
    float* dsm = sh + RP_TILE;
    int* cqs = reinterpret_cast<int*>(dsm + RP_TILE);
    float* bw = reinterpret_cast<float*>(cqs + RP_TILE);   // ring, acc_mask + 1 floats
    const int ring = a.acc_mask + 1;
    double* acc = reinterpret_cast<double*>(bw + ring);    // [4 waves][ring]
    const int ktiles = (a.Lk + KT - 1) / KT, id = rp_block(a, ktiles);
    if (id >= a.B * a.heads * ktiles) return;
    const int bh = id / ktiles, b = bh / a.heads, h = bh - b * a.heads, k0 = (id - bh * ktiles) * KT;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
    const T* qp = (const T*)a.q + b * a.sq.b + h * a.sq.h;
    const T* gp = (const T*)a.dout + ((size_t)b * a.Lq * a.heads + h) * a.D;
    const long long gst = (long long)a.heads * a.D;
    const float* bias = a.bias + (size_t)h * a.n_off;
    const float2* stat = a.stat + (size_t)bh * a.Lq;
    const float* dsum = a.dsum + (size_t)bh * a.Lq;
    const int k_hi = min(k0 + KT, a.Lk) - 1;
    const int ck_lo = rp_c(a, k0) + a.off, ck_hi = rp_c(a, k_hi) + a.off;   // offset of a pair = this - c(query)
    const bool grad_bias = a.slab != nullptr;
    const int qtiles = (a.Lq + RP_TILE - 1) / RP_TILE;
    const int t0 = (int)((long long)qtiles * blockIdx.y / a.splits), t1 = (int)((long long)qtiles * (blockIdx.y + 1) / a.splits);
    float* slab = grad_bias ? a.slab + ((size_t)id * a.splits + blockIdx.y) * a.slab_ld : nullptr;
    const int slab_lo = ck_lo - rp_c(a, a.q_start + min(t1 * RP_TILE, a.Lq) - 1);
    double* mine = acc + wave * ring;

    typename Op::Frag kf[KB][Dim::NCH], vf[KB][Dim::NCH];
    int key[KB], ck[KB];
    bool ok[KB], any_bad = false, any_ok = false;
    rp_f32x4 dk[KB][Dim::DB], dv[KB][Dim::DB];
#pragma unroll
    for (int j = 0; j < KB; ++j) {
        key[j] = k0 + (wave * KB + j) * 16 + l;
        const int row = min(key[j], k_hi);
        ok[j] = key[j] < a.Lk && (!a.mask || a.mask[(size_t)b * a.Lk + row] != 0);
        any_bad |= !ok[j];
        any_ok |= ok[j];
        ck[j] = rp_c(a, row) + a.off;
        rp_row_frags<T, DP>((const T*)a.k + b * a.sk.b + (long long)row * a.sk.t + h * a.sk.h, ok[j], a.D, g, kf[j]);
        rp_row_frags<T, DP>((const T*)a.v + b * a.sv.b + (long long)row * a.sv.t + h * a.sv.h, ok[j], a.D, g, vf[j]);
#pragma unroll
        for (int d = 0; d < Dim::DB; ++d) dk[j][d] = dv[j][d] = rp_f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int j = 0; j < KB; ++j)
#pragma unroll
        for (int c = 0; c < Dim::NCH; ++c) {
            rp_settle(kf[j][c]);
            rp_settle(vf[j][c]);
        }
    any_bad = __any(any_bad);
    any_ok = __any(any_ok);
    const unsigned long long seed = a.pdrop > 0.f ? rp_seed(a) : 0ull;
    rp_zero_pad<T, DP, INS, RP_TILE>(Qs, a.D, threadIdx.x);
    rp_zero_pad<T, DP, INS, RP_TILE>(Gs, a.D, threadIdx.x);
    if (grad_bias)
        for (int i = threadIdx.x; i < 4 * ring; i += 256) acc[i] = 0.0;

    // offsets (from, to] leave the ring for the slab
    auto flush = [&](int from, int to) {
        for (int i = from + 1 + (int)threadIdx.x; i <= to; i += 256) {
            double* p = acc + (i & a.acc_mask);
            const double v = (p[0] + p[ring]) + (p[2 * ring] + p[3 * ring]);
            p[0] = p[ring] = p[2 * ring] = p[3 * ring] = 0.0;
            slab[i - slab_lo] = (float)v;
        }
    };

    RpTile<T, DP, RP_TILE> qt, gt;
    qt.init(a.sq.t, a.D, threadIdx.x);
    gt.init(gst, a.D, threadIdx.x);
    float2 sr = make_float2(0.f, 0.f);
    float dr = 0.f, br[2];
    int b_lo = 0, b_hi = 0;
    auto fetch = [&](int t) {
        const int first = t * RP_TILE, left = a.Lq - first;
        qt.fetch(qp, a.sq.t, first, a.Lq, a.D, threadIdx.x);
        gt.fetch(gp, gst, first, a.Lq, a.D, threadIdx.x);
        if (threadIdx.x < RP_TILE) {
            const bool in = (int)threadIdx.x < left;
            sr = in ? stat[first + threadIdx.x] : make_float2(0.f, INFINITY);
            dr = in ? dsum[first + threadIdx.x] : 0.f;
        }
        // the offsets that this tile is the first to reach: below those of the tile before it
        b_lo = ck_lo - rp_c(a, a.q_start + min(first + RP_TILE, a.Lq) - 1);
        b_hi = t == t0 ? ck_hi - rp_c(a, a.q_start + first) : ck_lo - rp_c(a, a.q_start + first - 1) - 1;
#pragma unroll
        for (int i = 0; i < 2; ++i) br[i] = bias[min(b_lo + i * 256 + (int)threadIdx.x, b_hi)];
    };
    fetch(t0);
    int top = ck_hi - rp_c(a, a.q_start + t0 * RP_TILE);   // highest offset still in the ring
    for (int t = t0; t < t1; ++t) {
        const int first = t * RP_TILE, q_hi = min(first + RP_TILE, a.Lq) - 1;
        const int cq_lo = rp_c(a, a.q_start + first);
        rp_barrier();
        if (grad_bias) {
            const int reach = ck_hi - cq_lo;
            flush(reach, top);
            top = reach;
        }
        const int left = a.Lq - first;
        const unsigned long long rows[1] = {left >= 64 ? ~0ull : (1ull << left) - 1};
        qt.template put<INS>(Qs, rows, a.D, threadIdx.x);
        gt.template put<INS>(Gs, rows, a.D, threadIdx.x);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (b_lo + i * 256 + (int)threadIdx.x <= b_hi) bw[(b_lo + i * 256 + threadIdx.x) & a.acc_mask] = br[i];
        for (int i = b_lo + 512 + (int)threadIdx.x; i <= b_hi; i += 256) bw[i & a.acc_mask] = bias[i];
        if (threadIdx.x < RP_TILE) {
            ms[threadIdx.x] = sr.x;
            ls[threadIdx.x] = sr.y;
            sh[threadIdx.x] = fmaf(sr.x, a.sl2, sr.y);
            dsm[threadIdx.x] = dr;
            cqs[threadIdx.x] = rp_c(a, a.q_start + min(first + (int)threadIdx.x, q_hi));
        }
        rp_barrier();
        const bool far = __any(fabsf(ms[lane]) * a.sl2 > RP_FAR);
        if (t + 1 < t1) fetch(t + 1);
        if (!any_ok) continue;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            rp_f32x4 p[2][KB], ds[2][KB];   // scores, then P (dropped); dP, then dS
            int at[2][KB][4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int4 c4 = *reinterpret_cast<const int4*>(cqs + g * 16 + (2 * kk + e) * 4);
                const int cr[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
                for (int j = 0; j < KB; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        at[e][j][r] = (ck[j] - cr[r]) & a.acc_mask;
                        p[e][j][r] = bw[at[e][j][r]];
                        ds[e][j][r] = 0.f;
                    }
            }
#pragma unroll
            for (int c = 0; c < Dim::NCH; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = (l >> 2) * (16 * LD + INS) + ((2 * kk + e) * 4 + (l & 3)) * LD + c * Op::CHUNK + g * Op::PER;
                    const typename Op::Frag qf = *reinterpret_cast<const typename Op::Frag*>(Qs + row);
                    const typename Op::Frag gf = *reinterpret_cast<const typename Op::Frag*>(Gs + row);
#pragma unroll
                    for (int j = 0; j < KB; ++j) {
                        p[e][j] = Op::dot(qf, kf[j][c], p[e][j]);
                        ds[e][j] = Op::dot(gf, vf[j][c], ds[e][j]);
                    }
                }
            if (any_bad) {
#pragma unroll
                for (int j = 0; j < KB; ++j)
                    if (!ok[j]) p[0][j] = p[1][j] = rp_f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            }
            unsigned kept = 0u;   // dropout: bit (e * KB + j) * 4 + r
            if (a.pdrop > 0.f) {
                const float up = 1.0f / (1.0f - a.pdrop);
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int j = 0; j < KB; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const unsigned long long q = (unsigned long long)bh * a.Lq + first + g * 16 + (2 * kk + e) * 4 + r;
                            const bool keep = rp_drop(seed, q * a.Lk + key[j], a.pdrop) != 0.f;
                            ds[e][j][r] = keep ? ds[e][j][r] * up : 0.f;
                            kept |= (unsigned)keep << ((e * KB + j) * 4 + r);
                        }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = g * 16 + (2 * kk + e) * 4;
                const rp_f32x4 d4 = *reinterpret_cast<const rp_f32x4*>(dsm + row);
                if (far) {
                    const rp_f32x4 m4 = *reinterpret_cast<const rp_f32x4*>(ms + row);
                    const rp_f32x4 l4 = *reinterpret_cast<const rp_f32x4*>(ls + row);
#pragma unroll
                    for (int j = 0; j < KB; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) p[e][j][r] = __builtin_amdgcn_exp2f(fmaf(p[e][j][r] - m4[r], a.sl2, -l4[r]));
                } else {
                    const rp_f32x4 s4 = *reinterpret_cast<const rp_f32x4*>(sh + row);
#pragma unroll
                    for (int j = 0; j < KB; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) p[e][j][r] = __builtin_amdgcn_exp2f(fmaf(p[e][j][r], a.sl2, -s4[r]));
                }
#pragma unroll
                for (int j = 0; j < KB; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) ds[e][j][r] = p[e][j][r] * (ds[e][j][r] - d4[r]);
            }
            if (grad_bias) {
                if (!any_bad && left >= RP_TILE) {
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int j = 0; j < KB; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) rp_lds_add(mine + at[e][j][r], ds[e][j][r]);
                } else {
                    // keys and queries past the last have its offset: many lanes on one address (10x10 maps, batch 128, 8 heads of
                    // 48: 53 us with their zeros added, 36 without)
#pragma unroll
                    for (int j = 0; j < KB; ++j)
                        if (ok[j]) {
#pragma unroll
                            for (int e = 0; e < 2; ++e)
#pragma unroll
                                for (int r = 0; r < 4; ++r)
                                    if (g * 16 + (2 * kk + e) * 4 + r < left) rp_lds_add(mine + at[e][j][r], ds[e][j][r]);
                        }
                }
            }
            if (a.pdrop > 0.f) {
                const float up = 1.0f / (1.0f - a.pdrop);
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int j = 0; j < KB; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) p[e][j][r] = (kept >> ((e * KB + j) * 4 + r)) & 1 ? p[e][j][r] * up : 0.f;
            }
            typename Op::Pair pp[KB], pd[KB], pp2[KB], pd2[KB];
#pragma unroll
            for (int j = 0; j < KB; ++j) {
                pp[j] = Op::pack(p[0][j], p[1][j]);
                pd[j] = Op::pack(ds[0][j], ds[1][j]);
                if constexpr (sizeof(T) == 2) {
                    pp2[j] = Op::rest(p[0][j], p[1][j], pp[j]);
                    pd2[j] = Op::rest(ds[0][j], ds[1][j], pd[j]);
                }
            }
            const int trow = g * (16 * LD + INS) + kk * 8 * LD;
#pragma unroll
            for (int d = 0; d < Dim::DB; ++d) {
                const typename Op::TFrag qa = Op::load_t(Qs + trow + d * 16, Qs + trow + 4 * LD + d * 16, LD, l);
                const typename Op::TFrag ga = Op::load_t(Gs + trow + d * 16, Gs + trow + 4 * LD + d * 16, LD, l);
#pragma unroll
                for (int j = 0; j < KB; ++j) {
                    dk[j][d] = Op::dot_t(qa, pd[j], dk[j][d]);
                    dv[j][d] = Op::dot_t(ga, pp[j], dv[j][d]);
                }
                if constexpr (sizeof(T) == 2)
#pragma unroll
                    for (int j = 0; j < KB; ++j) {
                        dk[j][d] = Op::dot_t(qa, pd2[j], dk[j][d]);
                        dv[j][d] = Op::dot_t(ga, pp2[j], dv[j][d]);
                    }
            }
        }
    }
    if (grad_bias) {
        rp_barrier();
        flush(slab_lo - 1, top);
    }
#pragma unroll
    for (int j = 0; j < KB; ++j) {
        if (key[j] >= a.Lk) continue;
        if (a.splits > 1) {
            const size_t part = (size_t)a.B * a.heads * a.Lk * a.D;
            float* p = a.po + 2 * blockIdx.y * part + ((size_t)bh * a.Lk + key[j]) * a.D;
#pragma unroll
            for (int d = 0; d < Dim::DB; ++d) {
                const int col = d * 16 + g * 4;
                if (col >= a.D) continue;
                *reinterpret_cast<rp_f32x4*>(p + col) = ok[j] ? dk[j][d] : rp_f32x4{0.f, 0.f, 0.f, 0.f};
                *reinterpret_cast<rp_f32x4*>(p + part + col) = ok[j] ? dv[j][d] : rp_f32x4{0.f, 0.f, 0.f, 0.f};
            }
            continue;
        }
        T* kd = (T*)a.dk + b * a.sdk.b + (long long)key[j] * a.sdk.t + h * a.sdk.h;
        T* vd = (T*)a.dv + b * a.sdv.b + (long long)key[j] * a.sdv.t + h * a.sdv.h;
#pragma unroll
        for (int d = 0; d < Dim::DB; ++d) {
            const int col = d * 16 + g * 4;
            if (col >= a.D) continue;
            if (ok[j]) {
                store4<T>(kd + col, {dk[j][d][0] * a.scale, dk[j][d][1] * a.scale, dk[j][d][2] * a.scale, dk[j][d][3] * a.scale});
                store4<T>(vd + col, {dv[j][d][0], dv[j][d][1], dv[j][d][2], dv[j][d][3]});
            } else {   // a masked key has no gradient, whatever its own values are
                store4<T>(kd + col, {0.f, 0.f, 0.f, 0.f});
                store4<T>(vd + col, {0.f, 0.f, 0.f, 0.f});
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------
// bias gradient: offsets over images and key blocks, then buckets over their offsets (the offsets of bucket k are
// order[start[k]] .. order[start[k + 1] - 1]). Fixed order everywhere; in double, because a bucket's gradient is what is left of many
// terms of both signs: only a slab row and the result are fp32.
// ------------------------------------------------------------------------------------------------
// Slab rows are [image][head][key block][query range]; the offsets that a row covers depend on the last two alone. A workgroup: 64
// * PER offsets, 16 waves that share the rows where there are at least 16 of them (PER = 4: a row's four loads are in flight
// together), else the images (PER = 1, four images in flight). A lane works out what one row covers, a ballot finds the rows
// that reach the workgroup's offsets. 75x75 map, 4 heads, 704 rows: 12 us in double (11 in fp32; there 18 to 20 with PER = 1, 31 with every
// row tested by every wave); 38x38, 8 heads, 23 rows, 4 images: 5.7 us (5.5 in fp32, 7.7 with PER = 1).
template <int PER>
__global__ __launch_bounds__(1024) void relpos_offsets_kernel(RpArgs a, int ktiles, int kt, double* __restrict__ per_off) {
    __shared__ double sm[16][64 * PER];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), o0 = blockIdx.x * 64 * PER, h = blockIdx.y;
    const int rows = ktiles * a.splits, qtiles = (a.Lq + RP_TILE - 1) / RP_TILE;
    const size_t image = (size_t)a.heads * rows * a.slab_ld;
    double v[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) v[u] = 0.0;
    for (int first = 0; first < rows; first += 1024) {
        const int r = first + (PER == 4 ? lane * 16 + wave : lane), kb = (int)((unsigned)r / (unsigned)a.splits), sp = r - kb * a.splits, k0 = kb * kt;
        int lo = 0, hi = -1;
        if (r < rows) {
            const unsigned t0 = (unsigned)(qtiles * sp) / (unsigned)a.splits, t1 = (unsigned)(qtiles * (sp + 1)) / (unsigned)a.splits;   // at most 2^21 * 64
            lo = rp_c(a, k0) + a.off - rp_c(a, a.q_start + min((int)t1 * RP_TILE, a.Lq) - 1);
            hi = rp_c(a, min(k0 + kt, a.Lk) - 1) + a.off - rp_c(a, a.q_start + (int)t0 * RP_TILE);
        }
        unsigned long long reach = __ballot(r < rows && hi >= o0 && lo < o0 + 64 * PER);
        for (; reach != 0ull; reach &= reach - 1) {
            const int j = __builtin_ctzll(reach), from = __builtin_amdgcn_readlane(lo, j), to = __builtin_amdgcn_readlane(hi, j);
            const float* p = a.slab + ((size_t)h * rows + first + (PER == 4 ? j * 16 + wave : j)) * a.slab_ld;
            if constexpr (PER == 4) {
                int at[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) at[u] = min(max(o0 + u * 64 + lane, from), to) - from;
                for (int b = 0; b < a.B; ++b, p += image) {
                    float x[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) x[u] = p[at[u]];
#pragma unroll
                    for (int u = 0; u < 4; ++u) v[u] += (double)(at[u] == o0 + u * 64 + lane - from ? x[u] : 0.f);
                }
            } else {
                const int o = o0 + lane;
                const bool in = o >= from && o <= to;
                p += in ? o - from : 0;
                int b = wave;
                for (; b + 48 < a.B; b += 64) {
                    float x[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) x[u] = p[(b + u * 16) * image];
                    if (in) v[0] += ((double)x[0] + (double)x[1]) + ((double)x[2] + (double)x[3]);
                }
                for (; b < a.B; b += 16) {
                    const float x = p[b * image];
                    if (in) v[0] += (double)x;
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < PER; ++u) sm[wave][u * 64 + lane] = v[u];
    __syncthreads();
    if ((int)threadIdx.x >= 64 * PER || o0 + (int)threadIdx.x >= a.n_off) return;
    double total = sm[0][threadIdx.x];
    for (int w = 1; w < 16; ++w) total += sm[w][threadIdx.x];
    per_off[(size_t)h * a.n_off + o0 + threadIdx.x] = total;
}

__global__ __launch_bounds__(256) void relpos_buckets_kernel(const double* __restrict__ per_off, int n_off, int heads,
                                                             const int* __restrict__ order, const int* __restrict__ start,
                                                             float* __restrict__ dtable) {
    __shared__ double sm[4];
    const int k = blockIdx.x, h = blockIdx.y;
    double v = 0.0;
    for (int i = start[k] + threadIdx.x; i < start[k + 1]; i += 256) v += per_off[(size_t)h * n_off + order[i]];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) dtable[(size_t)k * heads + h] = (float)((sm[0] + sm[1]) + (sm[2] + sm[3]));
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
// largest difference of c between two of n consecutive tokens
static int rp_span(const RpArgs& a, int n, int tokens) {
    if (n > tokens) n = tokens;
    if (n <= 1) return 0;
    const int wraps = tokens <= a.W ? 0 : (n - 1 + a.W - 1) / a.W;
    return (n - 1) + wraps * (a.W - 1);
}

static int rp_dp(int D) { return D <= 16 ? 16 : D <= 32 ? 32 : D <= 48 ? 48 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }

static int rp_ld(int dtype, int DP) {   // RpDim::LD
    const int chunk = dtype == MIA_BF16 ? 32 : 16;
    return (DP + chunk - 1) / chunk * chunk + chunk / 4;
}
static int rp_stage(int dtype, int DP) { return dtype == MIA_BF16 && DP <= 64 ? 2 * RP_TILE : RP_TILE; }   // RpDim::STAGE
static size_t rp_es(int dtype) { return dtype == MIA_BF16 ? 2 : 4; }

// How the kernels are laid out over a problem: the pair with the lowest estimate of
//   cols: 16-wide columns of a wave, so 64 * cols queries (keys) of a workgroup. Two serve more products with every operand read from
//     LDS, but a round of them is 1.85 times as long (1.95 backward with heads of up to 32, whose two-column kernels have half as
//     many waves a SIMD; forward 2.1, so such heads keep one). fp32 and wide heads keep one: their operands do not fit.
//   splits: ranges of the tokens a workgroup walks, of at least four rounds, joined afterwards.
// The kernels are bound by issue, so what counts is the busiest of the 256 CUs: ceil(workgroups * splits / 256) of them, for
// ceil(rounds / splits) rounds each; a workgroup alone on its CU takes 1.25 times its share, and joining about 3 rounds plus what the
// partial results weigh. Measured (us, kernel + join), with the choice first: forward on a 75x75 map, 4 heads of 32: one column, 5
// splits 73 + 6, 2 splits 82 + 5, 3 splits 85 + 5; two columns, 4 splits 85 + 6. 4096 tokens, 4 heads of 64: two columns, 4 splits
// 54 + 7, 3 splits 66 + 6, 5 splits 65 + 7; one column, 3 splits 57 + 6. 38x38, batch 4, 8 heads of 64: one column unsplit 50, 3
// splits 50 + 11; two columns unsplit 58. 10x10, batch 128, 8 heads of 48: two columns 27, one 30.
// At most 16 queries (cols = 0): `few` heads of a workgroup's four waves. With enough keys for 2048 waves of four chunks or more, the
// waves read neighbouring heads, whose rows are one piece of memory, in ranges that make about 2048 waves; else the waves share one
// head's keys, four chunks each, which is what a second workgroup and the joining would cost.
#define RP_FEW_WAVES 2048
constexpr bool rp_two_columns(int what, int DP) { return what == RP_FWD ? DP > 32 && DP <= 96 : DP <= 64; }
struct RpPlan {
    int cols, splits, few;
};
static RpPlan rp_plan(int what, int dtype, int B, int heads, int Lq, int Lk, int D) {
    const int DP = rp_dp(D), owned = what == RP_BWD_KV ? Lk : Lq, walked = what == RP_BWD_KV ? Lq : Lk;
    const int round = what == RP_BWD_KV ? RP_TILE : rp_stage(dtype, DP);
    const long long rounds = (walked + round - 1) / round, most = rounds / 4 < 1 ? 1 : rounds / 4 < 64 ? rounds / 4 : 64;
    const int max_cols = dtype == MIA_F32 || owned <= 64 || !rp_two_columns(what, DP) ? 1 : 2;
    RpPlan p = {1, 1, 0};
    if (what == RP_FWD && Lq <= RP_FEW) {
        const int keys = rp_few_keys(dtype, DP);
        const long long bh = (long long)B * heads, chunks = (Lk + keys - 1) / keys;
        p.cols = 0;
        p.few = 1;
        long long s = (chunks + 15) / 16;
        if (bh * chunks >= 4 * RP_FEW_WAVES) {
            p.few = heads % 4 == 0 ? 4 : heads % 2 == 0 ? 2 : 1;
            s = (RP_FEW_WAVES * p.few / 4 + bh - 1) / bh;
        }
        p.splits = (int)(s < 1 ? 1 : s > 256 ? 256 : s);
        return p;
    }
    double best = 1e300;
    for (int cols = 1; cols <= max_cols; ++cols) {
        const long long wgs = (long long)B * heads * ((owned + 64 * cols - 1) / (64 * cols));
        const double length = cols == 1 ? 1.0 : DP > 32 ? 1.85 : 1.95;
        for (long long s = 1; s <= most; ++s) {
            const long long busiest = (wgs * s + 255) / 256, walk = (rounds + s - 1) / s;
            double t = length * walk * (busiest == 1 ? 1.25 : (double)busiest);
            if (s > 1) t += 3.0 + 0.6 * s * wgs * cols / 256;
            if (t < best) best = t, p.cols = cols, p.splits = (int)s;
        }
    }
    return p;
}

extern "C" int mia_relpos_plan(int direction, int dtype, int B, int heads, int Lq, int Lk, int D, int* plan) {
    MIA_CHECK_ARG(plan && direction >= RP_FWD && direction <= RP_BWD_KV && (dtype == MIA_F32 || dtype == MIA_BF16), "mia_relpos_plan: bad arguments");
    MIA_CHECK_ARG(B > 0 && heads > 0 && Lq > 0 && Lk > 0 && D > 0 && D % 8 == 0 && D <= 128, "mia_relpos_plan: bad shape");
    const RpPlan p = rp_plan(direction, dtype, B, heads, Lq, Lk, D);
    plan[0] = p.cols;
    plan[1] = p.splits;
    plan[2] = p.few;
    return 0;
}

template <typename K>
static int rp_launch(const char* name, K kernel, dim3 grid, size_t lds, const RpArgs& a, hipStream_t s) {
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        MIA_CHECK_ARG(e == hipSuccess, "%s: %zu bytes of LDS refused: %s", name, lds, hipGetErrorString(e));
    }
    MIA_LAUNCH(kernel, grid, dim3(256), lds, s, a);
    MIA_CHECK_LAUNCH(name);
    return 0;
}

template <typename T, int DP>
static int rp_few(const char* name, dim3 grid, const RpArgs& a, hipStream_t s) {
    MIA_LAUNCH((relpos_few_kernel<T, DP>), grid, dim3(256), 0, s, a);
    MIA_CHECK_LAUNCH(name);
    if (a.splits > 1) {
        MIA_LAUNCH((relpos_join_few_kernel<T, DP>), dim3(a.B * a.heads * a.Lq), dim3(256), 0, s, a);
        MIA_CHECK_LAUNCH(name);
    }
    return 0;
}

// COLS: 16-wide columns of a wave
template <typename T, int DP, int COLS>
static int rp_run(int what, const char* name, dim3 grid, size_t lds, const RpArgs& a, hipStream_t s) {
    if constexpr (COLS == 1 || rp_two_columns(RP_FWD, DP)) {
        if (what == RP_FWD) return rp_launch(name, relpos_fwd_kernel<T, DP, COLS>, grid, lds, a, s);
    }
    if constexpr (COLS == 1 || rp_two_columns(RP_BWD_Q, DP)) {
        if (what == RP_BWD_Q) return rp_launch(name, relpos_bwd_q_kernel<T, DP, COLS>, grid, lds, a, s);
        if (what == RP_BWD_KV) return rp_launch(name, relpos_bwd_kv_kernel<T, DP, COLS>, grid, lds, a, s);
    }
    mia_set_error("%s: dispatch failed", name);
    return -1;
}

static int rp_dispatch(int what, const char* name, int dtype, int cols, dim3 grid, size_t lds, const RpArgs& a, hipStream_t s) {
#define RP_CASE(DP_)                                                                                      \
    case DP_:                                                                                             \
        if (cols == 0) return dtype == MIA_F32 ? rp_few<float, DP_>(name, grid, a, s) : rp_few<bf16_t, DP_>(name, grid, a, s); \
        if (dtype == MIA_F32) return rp_run<float, DP_, 1>(what, name, grid, lds, a, s);          \
        return cols == 2 ? rp_run<bf16_t, DP_, 2>(what, name, grid, lds, a, s)                    \
                         : rp_run<bf16_t, DP_, 1>(what, name, grid, lds, a, s);
    switch (rp_dp(a.D)) {
        RP_CASE(16)
        RP_CASE(32)
        RP_CASE(48)
        RP_CASE(64)
        RP_CASE(96)
        RP_CASE(128)
    }
#undef RP_CASE
    return -1;
}

// LDS of a query kernel: two tiles, the keys' c and caps, the bias window
static size_t rp_query_lds(const RpArgs& a, int dtype, int DP, int cols, int tokens) {
    const int stage = rp_stage(dtype, DP), win = rp_span(a, stage, tokens) + rp_span(a, 64 * cols, tokens) + 1;
    return 2 * (size_t)stage * rp_ld(dtype, DP) * rp_es(dtype) + stage * 8 + (size_t)win * 4;
}

static dim3 rp_grid(long long blocks, int splits) { return dim3((unsigned)((blocks + 7) / 8 * 8), (unsigned)splits); }

static int rp_checks(const char* name, int dtype, int B, int heads, int Lq, int Lk, int D, int height, int width, int q_start,
                     float scale, float pdrop) {
    MIA_CHECK_ARG(dtype == MIA_F32 || dtype == MIA_BF16, "%s: bad dtype %d", name, dtype);
    MIA_CHECK_ARG(B > 0 && heads > 0 && Lq > 0 && Lk > 0 && D > 0, "%s: bad shape B=%d heads=%d queries=%d keys=%d D=%d", name, B, heads, Lq, Lk, D);
    MIA_CHECK_ARG(D % 8 == 0 && D <= 128, "%s: head width %d is not a multiple of 8 up to 128", name, D);
    MIA_CHECK_ARG(height > 0 && width > 0 && (height == 1 || width <= RP_MAX_WIDTH), "%s: bad map %d x %d (at most %d wide if of several rows)", name,
                  height, width, RP_MAX_WIDTH);
    MIA_CHECK_ARG((2ll * height - 1) * (2ll * width - 1) <= (1ll << 27), "%s: a map of %d x %d has too many offsets", name, height, width);
    const long long tokens = (long long)height * width;
    MIA_CHECK_ARG(height == 1 || tokens <= (1ll << 22), "%s: a map of %d x %d has too many tokens", name, height, width);
    MIA_CHECK_ARG(Lk <= tokens && q_start >= 0 && (long long)q_start + Lq <= tokens,
                  "%s: %d keys and %d queries from %d on do not fit a map of %lld tokens", name, Lk, Lq, q_start, tokens);
    MIA_CHECK_ARG(scale > 0.f && scale < 1e30f, "%s: scale must be positive (got %g)", name, (double)scale);
    MIA_CHECK_ARG(pdrop >= 0.f && pdrop < 1.f, "%s: dropout %g is not in [0, 1)", name, (double)pdrop);
    // 256 threads a block of 64 tokens, less than 2^32 of them in a launch
    MIA_CHECK_ARG((long long)B * heads * ((Lq + 63ll) / 64) < (1ll << 24) - 8 && (long long)B * heads * ((Lk + 63ll) / 64) < (1ll << 24) - 8,
                  "%s: too many workgroups", name);
    return 0;
}

static int rp_aligned(const char* name, int dtype, const void* p, const RpStride& s) {
    const long long per = dtype == MIA_BF16 ? 8 : 4;
    MIA_CHECK_ARG(((uintptr_t)p & 15) == 0 && s.b % per == 0 && s.t % per == 0 && s.h % per == 0,
                  "%s: rows must start at multiples of 16 bytes", name);
    MIA_CHECK_ARG(s.t >= 0 && s.t < (1ll << 24), "%s: token stride %lld is not in 0 .. 2^24 - 1", name, s.t);
    return 0;
}

static void rp_fill(RpArgs& a, int B, int heads, int Lq, int Lk, int D, int height, int width, int q_start, float scale,
                    float pdrop, unsigned long long seed, const unsigned long long* seed_offset) {
    a.B = B; a.heads = heads; a.Lq = Lq; a.Lk = Lk; a.D = D; a.W = width;
    a.inv_w = height == 1 || width == 1 ? 0u : (unsigned)(((1ull << 32) + width - 1) / width);
    a.off = (height - 1) * (2 * width - 1) + width - 1;
    a.n_off = (2 * height - 1) * (2 * width - 1);
    a.q_start = q_start; a.scale = scale; a.sl2 = scale * RP_LOG2E;
    a.pdrop = pdrop; a.seed = seed; a.seed_off = seed_offset;
    a.splits = 1;
}

static RpStride rp_stride(const long long* s) { return {s[0], s[1], s[2]}; }

extern "C" int mia_relpos_bias(const float* table, const int* bucket, int height, int width, int heads, float scale, float* bias,
                               void* stream) {
    MIA_CHECK_ARG(table && bucket && bias, "mia_relpos_bias: null");
    MIA_CHECK_ARG(height > 0 && width > 0 && heads > 0 && heads <= 65535 && (2ll * height - 1) * (2ll * width - 1) <= (1ll << 27) && scale > 0.f,
                  "mia_relpos_bias: bad arguments");
    const int n_off = (2 * height - 1) * (2 * width - 1);
    // after the division by scale and the later product with scale * log2(e) everything has to stay finite
    const float limit = 1e38f * fminf(1.f, scale);
    MIA_LAUNCH(relpos_expand_kernel, dim3(cdiv(n_off, 256), heads), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), table, bucket,
               n_off, heads, 1.0f / scale, limit, bias);
    MIA_CHECK_LAUNCH("mia_relpos_bias");
    return 0;
}

// floats of the partial results of a split launch (rows of D and two more per query; dK and dV rows of D)
static long long rp_part_floats(int what, const RpPlan& p, int B, int heads, int Lq, int Lk, int D) {
    if (p.splits == 1) return 0;
    return (long long)p.splits * B * heads * (what == RP_BWD_KV ? 2ll * Lk * D : (long long)Lq * (D + 2));
}

template <int WHAT>
static int rp_join(const char* name, int dtype, const RpArgs& a, hipStream_t s) {
    const long long threads = (long long)a.B * a.heads * (WHAT == RP_BWD_KV ? a.Lk : a.Lq) * (a.D / 4);
    const dim3 grid((unsigned)((threads + 255) / 256));
    if (dtype == MIA_BF16) MIA_LAUNCH((relpos_join_kernel<bf16_t, WHAT>), grid, dim3(256), 0, s, a);
    else MIA_LAUNCH((relpos_join_kernel<float, WHAT>), grid, dim3(256), 0, s, a);
    MIA_CHECK_LAUNCH(name);
    return 0;
}

extern "C" long long mia_relpos_fwd_ws_floats(int dtype, int B, int heads, int Lq, int Lk, int D) {
    return rp_part_floats(RP_FWD, rp_plan(RP_FWD, dtype, B, heads, Lq, Lk, D), B, heads, Lq, Lk, D);
}

extern "C" int mia_relpos_fwd(int dtype, const void* q, const void* k, const void* v, const long long* strides, int B, int heads,
                              int Lq, int Lk, int D, const float* bias, int height, int width, int q_start,
                              const uint8_t* key_mask, float scale, float pdrop, unsigned long long seed,
                              const unsigned long long* seed_offset, float* ws, long long ws_floats, void* out, void* out_low,
                              float* stat, void* stream) {
    if (rp_checks("mia_relpos_fwd", dtype, B, heads, Lq, Lk, D, height, width, q_start, scale, pdrop)) return -1;
    MIA_CHECK_ARG(q && k && v && strides && bias && out, "mia_relpos_fwd: null");
    MIA_CHECK_ARG(((uintptr_t)stat & 7) == 0, "mia_relpos_fwd: stat must start at a multiple of 8 bytes");
    RpArgs a = {};
    a.q = q; a.k = k; a.v = v; a.o = out; a.o_low = out_low; a.bias = bias; a.mask = key_mask; a.stat = reinterpret_cast<float2*>(stat);
    a.sq = rp_stride(strides); a.sk = rp_stride(strides + 3); a.sv = rp_stride(strides + 6);
    if (rp_aligned("mia_relpos_fwd", dtype, q, a.sq) || rp_aligned("mia_relpos_fwd", dtype, k, a.sk) ||
        rp_aligned("mia_relpos_fwd", dtype, v, a.sv) || rp_aligned("mia_relpos_fwd", dtype, out, RpStride{0, 0, 0}) ||
        rp_aligned("mia_relpos_fwd", dtype, out_low, RpStride{0, 0, 0}))
        return -1;
    rp_fill(a, B, heads, Lq, Lk, D, height, width, q_start, scale, pdrop, seed, seed_offset);
    const RpPlan plan = rp_plan(RP_FWD, dtype, B, heads, Lq, Lk, D);
    const int cols = plan.cols, tile = cols == 0 ? rp_few_keys(dtype, rp_dp(D)) : rp_stage(dtype, rp_dp(D));
    a.tiles = (Lk + tile - 1) / tile;
    a.splits = plan.splits;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const long long rows = (long long)B * heads * Lq;
    if (a.splits > 1) {
        MIA_CHECK_ARG(ws && ws_floats >= mia_relpos_fwd_ws_floats(dtype, B, heads, Lq, Lk, D),
                      "mia_relpos_fwd: workspace of %lld floats is too small (%lld needed)", ws_floats,
                      mia_relpos_fwd_ws_floats(dtype, B, heads, Lq, Lk, D));
        MIA_CHECK_ARG(((uintptr_t)ws & 15) == 0, "mia_relpos_fwd: the workspace must start at a multiple of 16 bytes");
        a.po = ws;
        a.pml = ws + (long long)a.splits * rows * D;
    }
    const int tokens = height * width, DP = rp_dp(D);
    const size_t lds = cols == 0 ? 0 : rp_query_lds(a, dtype, DP, cols, tokens);
    a.few = plan.few;
    const long long blocks = cols == 0 ? (long long)B * heads / a.few : (long long)B * heads * ((Lq + 64 * cols - 1) / (64 * cols));
    const dim3 grid = cols == 0 ? dim3((unsigned)(blocks * a.splits)) : rp_grid(blocks, a.splits);
    const int rc = rp_dispatch(RP_FWD, "mia_relpos_fwd", dtype, cols, grid, lds, a, s);
    if (rc || a.splits == 1 || cols == 0) return rc;
    return rp_join<RP_FWD>("mia_relpos_fwd", dtype, a, s);
}

// Floats of one slab row: the offsets between the keys of a block and the queries of a split's range. A map's offsets span about
// twice its tokens, so the rows of an (image, head) are L^2 / 32 floats on a map with blocks of 64 keys, L^2 / 128 on a sequence
// with blocks of 128, and the ranges' ends (75x75, 4 heads of 32: 18 MB; 127 with room for all queries in every range's row).
static int rp_slab_ld(const RpArgs& a, int tokens, const RpPlan& p) {
    const int qtiles = (a.Lq + RP_TILE - 1) / RP_TILE, range = RP_TILE * ((qtiles + p.splits - 1) / p.splits);
    return rp_span(a, range < a.Lq ? range : a.Lq, tokens) + rp_span(a, 64 * p.cols, tokens) + 1;
}

// The backward's workspace: D of every row | the bias gradient per offset (doubles) | slab rows | partial results (those of dQ are
// joined before the dK / dV kernel writes its own over them)
struct RpWs {
    long long per_off, slab, part, total;
};
static RpWs rp_bwd_ws(int dtype, int B, int heads, int Lq, int Lk, int D, int height, int width, int want_bias) {
    RpArgs a = {};
    rp_fill(a, B, heads, Lq, Lk, D, height, width, 0, 1.f, 0.f, 0, nullptr);
    const RpPlan q = rp_plan(RP_BWD_Q, dtype, B, heads, Lq, Lk, D), kv = rp_plan(RP_BWD_KV, dtype, B, heads, Lq, Lk, D);
    const long long bh = (long long)B * heads, kt = 64 * kv.cols;
    RpWs w;
    w.per_off = (bh * Lq + 3) / 4 * 4;
    w.slab = w.per_off + (want_bias ? 2ll * heads * a.n_off : 0);
    w.part = w.slab + (want_bias ? bh * ((Lk + kt - 1) / kt) * kv.splits * rp_slab_ld(a, height * width, kv) : 0);
    w.part = (w.part + 3) / 4 * 4;
    const long long pq = rp_part_floats(RP_BWD_Q, q, B, heads, Lq, Lk, D), pk = rp_part_floats(RP_BWD_KV, kv, B, heads, Lq, Lk, D);
    w.total = w.part + (pq > pk ? pq : pk);
    return w;
}

extern "C" long long mia_relpos_bwd_ws_floats(int dtype, int B, int heads, int Lq, int Lk, int D, int height, int width, int want_bias) {
    const RpWs w = rp_bwd_ws(dtype, B, heads, Lq, Lk, D, height, width, want_bias);
    return w.total;
}

extern "C" int mia_relpos_bwd(int dtype, const void* q, const void* k, const void* v, const long long* strides, const void* dout,
                              const void* out, const void* out_low, const float* stat, int B, int heads, int Lq, int Lk, int D, const float* bias,
                              int height, int width, int q_start, const uint8_t* key_mask, float scale, float pdrop,
                              unsigned long long seed, const unsigned long long* seed_offset, const int* order, const int* start,
                              int buckets, float* ws, long long ws_floats, void* dq, void* dk, void* dv,
                              const long long* grad_strides, float* dtable, void* stream) {
    if (rp_checks("mia_relpos_bwd", dtype, B, heads, Lq, Lk, D, height, width, q_start, scale, pdrop)) return -1;
    MIA_CHECK_ARG(q && k && v && strides && dout && out && stat && bias && ws && dq && dk && dv && grad_strides, "mia_relpos_bwd: null");
    MIA_CHECK_ARG(dtype != MIA_BF16 || out_low, "mia_relpos_bwd: bf16 needs the forward's out_low");
    MIA_CHECK_ARG(((uintptr_t)stat & 7) == 0, "mia_relpos_bwd: stat must start at a multiple of 8 bytes");
    MIA_CHECK_ARG(!dtable || (order && start && buckets > 0), "mia_relpos_bwd: the bias gradient needs the bucket lists");
    MIA_CHECK_ARG(heads <= 65535, "mia_relpos_bwd: %d heads are too many", heads);
    const RpWs w = rp_bwd_ws(dtype, B, heads, Lq, Lk, D, height, width, dtable != nullptr);
    MIA_CHECK_ARG(ws_floats >= w.total, "mia_relpos_bwd: workspace of %lld floats is too small (%lld needed)", ws_floats, w.total);
    MIA_CHECK_ARG(((uintptr_t)ws & 15) == 0, "mia_relpos_bwd: the workspace must start at a multiple of 16 bytes");
    RpArgs a = {};
    a.q = q; a.k = k; a.v = v; a.dout = dout; a.out = out; a.out_low = out_low; a.bias = bias; a.mask = key_mask;
    a.stat = reinterpret_cast<float2*>(const_cast<float*>(stat));
    a.dq = dq; a.dk = dk; a.dv = dv; a.dsum = ws;
    a.sq = rp_stride(strides); a.sk = rp_stride(strides + 3); a.sv = rp_stride(strides + 6);
    a.sdq = rp_stride(grad_strides); a.sdk = rp_stride(grad_strides + 3); a.sdv = rp_stride(grad_strides + 6);
    const void* ptrs[] = {q, k, v, dq, dk, dv, dout, out, out_low};
    const RpStride sts[] = {a.sq, a.sk, a.sv, a.sdq, a.sdk, a.sdv, {0, 0, 0}, {0, 0, 0}, {0, 0, 0}};
    for (int i = 0; i < 9; ++i)
        if (rp_aligned("mia_relpos_bwd", dtype, ptrs[i], sts[i])) return -1;
    rp_fill(a, B, heads, Lq, Lk, D, height, width, q_start, scale, pdrop, seed, seed_offset);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const long long bh = (long long)B * heads;
    const int tokens = height * width, DP = rp_dp(D);
    const size_t tile = (size_t)RP_TILE * rp_ld(dtype, DP) * rp_es(dtype);
    const RpPlan qp = rp_plan(RP_BWD_Q, dtype, B, heads, Lq, Lk, D), kp = rp_plan(RP_BWD_KV, dtype, B, heads, Lq, Lk, D);
    const int stage = rp_stage(dtype, DP), kt = 64 * kp.cols, ktiles = (Lk + kt - 1) / kt;
    a.tiles = (Lk + stage - 1) / stage;
    a.splits = qp.splits;
    a.po = ws + w.part;
    a.pml = a.po + (long long)qp.splits * bh * Lq * D;
    if (int rc = rp_dispatch(RP_BWD_Q, "mia_relpos_bwd", dtype, qp.cols, rp_grid(bh * ((Lq + 64 * qp.cols - 1) / (64 * qp.cols)), qp.splits),
                             rp_query_lds(a, dtype, DP, qp.cols, tokens), a, s))
        return rc;
    if (qp.splits > 1)
        if (int rc = rp_join<RP_BWD_Q>("mia_relpos_bwd", dtype, a, s)) return rc;
    int ring = 64;
    while (ring < rp_span(a, RP_TILE, tokens) + rp_span(a, kt, tokens) + 1) ring *= 2;
    MIA_CHECK_ARG(ring <= RP_RING_MAX, "mia_relpos_bwd: ring of %d offsets", ring);
    a.acc_mask = ring - 1;
    a.splits = kp.splits;
    double* per_off = reinterpret_cast<double*>(ws + w.per_off);
    if (dtable) {
        a.slab_ld = rp_slab_ld(a, tokens, kp);
        a.slab = ws + w.slab;
    }
    const size_t kv_lds = 2 * (tile + 256) + 5 * RP_TILE * 4 + (size_t)ring * (dtable ? 4 + 4 * 8 : 4);
    if (int rc = rp_dispatch(RP_BWD_KV, "mia_relpos_bwd", dtype, kp.cols, rp_grid(bh * ktiles, kp.splits), kv_lds, a, s)) return rc;
    if (kp.splits > 1)
        if (int rc = rp_join<RP_BWD_KV>("mia_relpos_bwd", dtype, a, s)) return rc;
    if (!dtable) return 0;
    if (ktiles * a.splits >= 16) MIA_LAUNCH((relpos_offsets_kernel<4>), dim3(cdiv(a.n_off, 256), heads), dim3(1024), 0, s, a, ktiles, kt, per_off);
    else MIA_LAUNCH((relpos_offsets_kernel<1>), dim3(cdiv(a.n_off, 64), heads), dim3(1024), 0, s, a, ktiles, kt, per_off);
    MIA_CHECK_LAUNCH("mia_relpos_bwd");
    MIA_LAUNCH(relpos_buckets_kernel, dim3(buckets, heads), dim3(256), 0, s, per_off, a.n_off, heads, order, start, dtable);
    MIA_CHECK_LAUNCH("mia_relpos_bwd");
    return 0;
}
