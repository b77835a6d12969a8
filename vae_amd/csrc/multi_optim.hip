// Gradient-norm clipping and AdamW over MANY separate tensors (torch.nn.utils.clip_grad_norm_ and torch.optim.AdamW,
// vae/training/train.py:310,336,338, for a model whose parameters are separate allocations, as the drafts' U-Nets' are),
// with fp32 or bf16 parameters and both moments in 32 or in 8 bits.
//
// A launch carries the table of its tensors (addresses, lengths, place of their state) in its kernel arguments: gradients
// are new allocations every step, and arguments are the one way to hand over their addresses that needs no copy, no buffer
// whose lifetime somebody has to watch, and that a captured graph replays as recorded.
//
// State layout.  Every tensor's state starts on a block of 256 elements of its group's flat state buffers; `block` is that block.
//
// 8-bit moments.  A block has one base per moment.  The fp32 bits of a magnitude shifted right by 20 are its LEVEL: exponent
// and three mantissa bits, 8 levels per octave.  Code c > 0 stands for level base + c, code 0 for zero.
//   exp_avg    : bit 7 = sign, c = 1..127 (15.9 octaves below the block's largest magnitude); 0x80 = not finite
//   exp_avg_sq : c = 1..254 (31.75 octaves); a positive value always gets c >= 1, because m / (sqrt(0) + eps) of a value
//                that had only been rounded to zero would be a step of size lr * m / eps; 255 = not finite
// The base depends on the finite values only, so a NaN in a gradient stays in its own element.
// Rounding adds d in [0, 2^20) to the bits before the shift.  To nearest (d = 2^19) would not do: with beta2 = 0.999 a step moves
// exp_avg_sq by at most 0.1 % where its gradient has stopped, a level is 6 to 12 % wide, and it would stay where it is for good.
// d is the top 20 bits of (i * 2^32 / golden ratio + t * 2^32 * frac(sqrt 3 or sqrt 2)) mod 2^32, i the element's index in its
// tensor and t the step: for a fixed element an additive recurrence with an irrational rate, equidistributed over t (Weyl), so that
// a constant is rounded without bias, and 1, sqrt 2, sqrt 3 are independent over the rationals, so the two moments' pairs are too.
// It needs no generator state, costs one addition per value, and is the same on every data-parallel rank.  In the loop, where the
// value depends on the dither of the steps before, it is not unbiased to the last percent but nearer than independent random numbers:
// exp_avg_sq over 4096 elements against 64 bits after 2000 steps (constant gradient / noise / gradient every other step / 1500 steps
// without one): off by 5 / 16 / 10 / 10 % rms with means of +2 / -1 / -7 / -9 %; random numbers 10 / 20 / 21 / 42 % rms with means
// of 0; to nearest the means are -97 / -73 / -95 / -74 %.
//
// bf16 parameters.  Steps of lr are far below half a last place of bf16, so the parameter alone would not move.  A 16-bit
// remainder r makes it a 32-bit master: |master| bits = (|p| bits << 16) + r, with p = (|master| bits + 0x8000) >> 16 (nearest, ties
// away).  That is 2 bytes a parameter instead of 4, and a parameter that somebody else writes needs no bookkeeping: any
// (p, r) stands for p to within half of its last place.
#include "common.h"
#include "prof.h"
#include "../../include/vae_hip.h"

namespace vae {

#define MT_TENSORS 192           // tensors one launch takes: 32 + 4 bytes of kernel arguments each
#define MT_CHUNK 4096            // elements a workgroup takes at a time
#define MT_BLOCK 256             // elements of one tensor that share a base; a wave's 64 lanes x 4
#define MT_PARTIALS 256          // workgroups (= partial sums) of the norm; every launch of a longer list has at least one

struct MtJob {
    void* p;
    const void* g;
    long n;
    uint32_t block;
    uint32_t slot_flags;         // slot << 2 | VAE_MT_*
};
struct MtTable {
    int count;
    uint32_t nchunk;
    uint32_t first[MT_TENSORS];  // first chunk of each tensor; 0xFFFFFFFF behind the last
    MtJob job[MT_TENSORS];
};
struct MtHyper {
    void *m, *v;
    short2* base;
    short* rem;
    const float* scal;
    float b1, omb1, b2, omb2, eps;
};
// what makes the per-tensor numbers of a step (prep_tensors)
struct MtPrep {
    long* steps;
    float* scal;
    const float* lr_dev;
    double lr, b1, b2, wd;
};
// per-tensor numbers of a step, 8 floats at scal + 8 * slot
struct MtScal {
    float decay, step, inv_bc2;
    uint32_t phase_m, phase_v;
};

#define DITHER_I 0x9E3779B9u     // 2^32 / golden ratio
#define DITHER_M 0xBB67AE85u     // 2^32 * frac(sqrt 3)
#define DITHER_V 0x6A09E667u     // 2^32 * frac(sqrt 2)

// vectors whose address is only as aligned as one element: the memory system takes any 4-byte (fp32) or 2-byte (bf16) address
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x4u __attribute__((ext_vector_type(4), aligned(2)));

// Which tensor a chunk belongs to: the last one whose first chunk is not behind it.  All lanes compare at once.
struct MtFind {
    uint32_t f[MT_TENSORS / 64];
    __device__ __forceinline__ MtFind(const MtTable& t) {
#pragma unroll
        for (int k = 0; k < MT_TENSORS / 64; ++k) f[k] = t.first[k * 64 + (threadIdx.x & 63)];
    }
    __device__ __forceinline__ int operator()(uint32_t chunk) const {
        int n = 0;
#pragma unroll
        for (int k = 0; k < MT_TENSORS / 64; ++k) n += __popcll(__ballot(f[k] <= chunk));
        return __builtin_amdgcn_readfirstlane(n - 1);
    }
};

// four consecutive elements from index i of n; elements behind the end read as 0
template <bool BF>
__device__ __forceinline__ void load4(const void* p, long i, long n, float x[4]) {
    if (i + 4 <= n) {
        if (BF) {
            const u16x4u q = *(const u16x4u*)((const bf16_t*)p + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = bf2f(q[k]);
        } else {
            const f32x4u q = *(const f32x4u*)((const float*)p + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = q[k];
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = i + k < n ? (BF ? bf2f(((const bf16_t*)p)[i + k]) : ((const float*)p)[i + k]) : 0.f;
    }
}
__device__ __forceinline__ void store4(float* p, long i, long n, const float x[4]) {
    if (i + 4 <= n) {
        f32x4u q;
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = x[k];
        *(f32x4u*)(p + i) = q;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) p[i + k] = x[k];
    }
}
__device__ __forceinline__ void store4(bf16_t* p, long i, long n, const bf16_t x[4]) {
    if (i + 4 <= n) {
        u16x4u q;
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = x[k];
        *(u16x4u*)(p + i) = q;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) p[i + k] = x[k];
    }
}

// ---------------------------------------------------------------- global norm
// Squares and sums in 64 bits: a square of an fp32 gradient can pass fp32's range, and the sum runs over the whole model.
template <bool BF>
__device__ __forceinline__ double sumsq_chunk(const void* g, long c0, long n) {
    double a = 0.0;
    float x[4][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) load4<BF>(g, c0 + (u * 256 + (int)threadIdx.x) * 4L, n, x[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int k = 0; k < 4; ++k) a = __builtin_fma((double)x[u][k], (double)x[u][k], a);
    return a;
}

// beta^t, t >= 1, by squaring: 2 log2(t) multiplications, off by less than t * 2^-53 of its value
__device__ __forceinline__ double int_pow(double b, unsigned long t) {
    double r = 1.0;
    for (; t; t >>= 1) {
        if (t & 1) r *= b;
        b *= b;
    }
    return r;
}

// Advances each tensor's step count and works out what depends on it alone, in 64 bits.  The counts live on the device, so
// that a captured step counts on when it is replayed.
__device__ __forceinline__ void prep_tensors(const MtTable& tab, const MtPrep& h) {
    for (int i = threadIdx.x; i < tab.count; i += blockDim.x) {
        const uint32_t slot = tab.job[i].slot_flags >> 2;
        const long t = h.steps[slot] + 1;
        h.steps[slot] = t;
        const double lr = h.lr_dev ? (double)*h.lr_dev : h.lr;
        float* s = h.scal + 8 * (size_t)slot;
        s[0] = (float)(1.0 - lr * h.wd);
        s[1] = (float)(lr / (1.0 - int_pow(h.b1, t)));
        s[2] = (float)(1.0 / sqrt(1.0 - int_pow(h.b2, t)));
        s[3] = __uint_as_float((uint32_t)t * DITHER_M);
        s[4] = __uint_as_float((uint32_t)t * DITHER_V);
    }
}

// workgroups 0..nsum-1: partial sums; with PREP one more, which prepares the step of the same tensors
template <bool PREP>
__global__ __launch_bounds__(256) void multi_sumsq_kernel(const MtTable tab, double* __restrict__ partial, int nsum, const MtPrep prep) {
    if (PREP && (int)blockIdx.x >= nsum) {
        prep_tensors(tab, prep);
        return;
    }
    __shared__ double red[4];
    const MtFind find(tab);
    double a = 0.0;
    for (uint32_t c = blockIdx.x; c < tab.nchunk; c += nsum) {
        const int j = find(c);
        const MtJob& jb = tab.job[j];
        const long c0 = (long)(c - tab.first[j]) * MT_CHUNK;
        a += (jb.slot_flags & VAE_MT_GRAD_BF16) ? sumsq_chunk<true>(jb.g, c0, jb.n) : sumsq_chunk<false>(jb.g, c0, jb.n);
    }
    a = wave_sum_d(a);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

struct MtClip {
    const double* partial;
    int npartial;                // 0: no norm was taken
    float grad_mul, max_norm;    // max_norm < 0: no clipping
    float* norm_out;
};

// What gradients are multiplied with; every wave folds the partial sums itself (no barrier).  A norm that is NaN makes every
// gradient NaN and an infinite one makes them 0 or NaN, as torch's clip_grad_norm_ does.
__device__ __forceinline__ float clip_coef(const MtClip& c) {
    if (c.npartial == 0) return c.grad_mul;
    double a = 0.0;
    for (int i = threadIdx.x & 63; i < c.npartial; i += 64) a += c.partial[i];
    a = wave_sum_d(a);
    const double norm = sqrt(a) * fabs((double)c.grad_mul);
    if (blockIdx.x == 0 && threadIdx.x == 0 && c.norm_out) *c.norm_out = (float)norm;
    if (c.max_norm < 0.f) return c.grad_mul;
    const double q = (double)c.max_norm / (norm + 1e-6);
    return (float)(q >= 1.0 ? 1.0 : q) * c.grad_mul;
}

template <bool BF>
__device__ __forceinline__ void scale_chunk(void* g, long c0, long n, float coef) {
    float x[4][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) load4<BF>(g, c0 + (u * 256 + (int)threadIdx.x) * 4L, n, x[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const long i = c0 + (u * 256 + (int)threadIdx.x) * 4L;
        if (BF) {
            bf16_t y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = f2bf(x[u][k] * coef);
            store4((bf16_t*)g, i, n, y);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) x[u][k] *= coef;
            store4((float*)g, i, n, x[u]);
        }
    }
}

__global__ __launch_bounds__(256) void multi_scale_kernel(const MtTable tab, const MtClip clip) {
    const MtFind find(tab);
    const float coef = clip_coef(clip);
    for (uint32_t c = blockIdx.x; c < tab.nchunk; c += gridDim.x) {
        const int j = find(c);
        const MtJob& jb = tab.job[j];
        const long c0 = (long)(c - tab.first[j]) * MT_CHUNK;
        if (jb.slot_flags & VAE_MT_GRAD_BF16) scale_chunk<true>((void*)jb.g, c0, jb.n, coef);
        else scale_chunk<false>((void*)jb.g, c0, jb.n, coef);
    }
}

__global__ __launch_bounds__(64) void multi_norm_kernel(const MtClip clip) { clip_coef(clip); }

// ---------------------------------------------------------------- 8-bit moments
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
    return v;
}
__device__ __forceinline__ bool finite_bits(uint32_t x) { return x < 0x7F800000u; }     // of a magnitude
__device__ __forceinline__ int level_up(uint32_t x) { return min((int)((x + 0xFFFFFu) >> 20), 0x7F7); }

__device__ __forceinline__ float unpack_m(uint32_t q, int base) {
    const uint32_t c = q & 127u;
    uint32_t x = c ? (uint32_t)(base + (int)c) << 20 : 0u;
    x |= (q & 128u) << 24;
    return __uint_as_float(q == 128u ? 0x7FC00000u : x);
}
__device__ __forceinline__ float unpack_v(uint32_t q, int base) {
    const uint32_t x = q ? (uint32_t)(base + (int)q) << 20 : 0u;
    return __uint_as_float(q == 255u ? 0x7FC00000u : x);
}
// low: level base + 1, the smallest that has a code.  Below it the value becomes 0 or that level, the latter with
// probability |m| / low over the dither (d * low is exact: 20 bits times 4)
__device__ __forceinline__ uint32_t pack_m(float m, int base, float low, uint32_t d) {
    const uint32_t x = __float_as_uint(m) & 0x7FFFFFFFu;
    const float a = __uint_as_float(x);
    const uint32_t big = (uint32_t)min((int)((x + d) >> 20) - base, 127);
    const uint32_t c = a >= low ? big : (a > (float)d * (low * 0x1p-20f) ? 1u : 0u);
    const uint32_t q = c ? c | ((__float_as_uint(m) >> 24) & 128u) : 0u;
    return finite_bits(x) ? q : 128u;
}
__device__ __forceinline__ uint32_t pack_v(float v, int base, uint32_t d) {
    const uint32_t x = __float_as_uint(v) & 0x7FFFFFFFu;
    const int c = min(max((int)((x + d) >> 20) - base, 1), 254);
    return finite_bits(x) ? (x ? (uint32_t)c : 0u) : 255u;
}

// bases of a wave's block from each lane's four values; every lane gets them
__device__ __forceinline__ void block_bases(const float m[4], const float v[4], int& bm, int& bv) {
    uint32_t xm = 0, xv = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t a = __float_as_uint(m[k]) & 0x7FFFFFFFu, b = __float_as_uint(v[k]) & 0x7FFFFFFFu;
        xm = max(xm, finite_bits(a) ? a : 0u);
        xv = max(xv, finite_bits(b) ? b : 0u);
    }
    bm = max(level_up(wave_max_u32(xm)) - 127, 0);
    bv = max(level_up(wave_max_u32(xv)) - 254, 0);
}
__device__ __forceinline__ uint32_t pack_base(int bm, int bv) { return (uint32_t)bm | (uint32_t)bv << 16; }

// ---------------------------------------------------------------- AdamW
// (parameter, remainder) <-> master; a magnitude below zero can only come of a parameter that was written since, and is 0
__device__ __forceinline__ float join_master(bf16_t p, short r) {
    const uint32_t hi = (uint32_t)(p & 0x7FFF) << 16;
    const uint32_t x = hi >= 0x7F800000u && (r > 0 || hi > 0x7F800000u) ? hi : (uint32_t)max((int)hi + (int)r, 0);
    return __uint_as_float(x | (uint32_t)(p & 0x8000) << 16);
}
__device__ __forceinline__ void split_master(float w, bf16_t& p, short& r) {
    const uint32_t x = __float_as_uint(w) & 0x7FFFFFFFu;
    const uint32_t hi = x > 0x7F800000u ? 0x7FC0u : (x + 0x8000u) >> 16;
    r = x > 0x7F800000u ? (short)0 : (short)(int)(x - (hi << 16));
    p = (bf16_t)(hi | ((__float_as_uint(w) >> 16) & 0x8000u));
}

// One block of 256 elements (a wave: 4 per lane) of one tensor.
template <bool PB, bool GB, bool S8>
__device__ __forceinline__ void adamw_block(const MtJob& jb, const MtHyper& h, const MtScal& s, float coef, long i, long blk, int lane) {
    const size_t k0 = (size_t)blk * MT_BLOCK + lane * 4;
    float p[4], g[4], m[4], v[4];
    load4<GB>(jb.g, i, jb.n, g);
    if (PB) {
        u16x4u q = {0, 0, 0, 0};
        if (i + 4 <= jb.n) q = *(const u16x4u*)((const bf16_t*)jb.p + i);
        else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k < jb.n) q[k] = ((const bf16_t*)jb.p)[i + k];
        }
        const short4v r = *(const short4v*)(h.rem + k0);
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] = join_master(q[k], r[k]);
    } else {
        load4<false>(jb.p, i, jb.n, p);
    }
    if (S8) {
        const uint32_t qm = *(const uint32_t*)((const uint8_t*)h.m + k0), qv = *(const uint32_t*)((const uint8_t*)h.v + k0);
        const short2 b = h.base[blk];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            m[k] = unpack_m((qm >> 8 * k) & 255u, b.x);
            v[k] = unpack_v((qv >> 8 * k) & 255u, b.y);
        }
    } else {
        const f32x4 a = *(const f32x4*)((const float*)h.m + k0), b = *(const f32x4*)((const float*)h.v + k0);
#pragma unroll
        for (int k = 0; k < 4; ++k) { m[k] = a[k]; v[k] = b[k]; }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float gk = g[k] * coef;
        m[k] = h.b1 * m[k] + h.omb1 * gk;
        v[k] = h.b2 * v[k] + h.omb2 * gk * gk;
        p[k] = p[k] * s.decay - s.step * m[k] / (sqrtf(v[k]) * s.inv_bc2 + h.eps);
    }
    if (PB) {
        bf16_t q[4];
        short4v r;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            short rk;
            split_master(p[k], q[k], rk);
            r[k] = i + k < jb.n ? rk : (short)0;
        }
        store4((bf16_t*)jb.p, i, jb.n, q);
        *(short4v*)(h.rem + k0) = r;
    } else {
        store4((float*)jb.p, i, jb.n, p);
    }
    if (S8) {
        int bm, bv;
        block_bases(m, v, bm, bv);
        const float low = __uint_as_float((uint32_t)(bm + 1) << 20);
        uint32_t qm = 0, qv = 0, u = (uint32_t)i * DITHER_I;
#pragma unroll
        for (int k = 0; k < 4; ++k, u += DITHER_I) {
            qm |= pack_m(m[k], bm, low, (u + s.phase_m) >> 12) << 8 * k;
            qv |= pack_v(v[k], bv, (u + s.phase_v) >> 12) << 8 * k;
        }
        *(uint32_t*)((uint8_t*)h.m + k0) = qm;
        *(uint32_t*)((uint8_t*)h.v + k0) = qv;
        if (lane == 0) *(uint32_t*)(h.base + blk) = pack_base(bm, bv);
    } else {
        const f32x4 a = {m[0], m[1], m[2], m[3]}, b = {v[0], v[1], v[2], v[3]};
        *(f32x4*)((float*)h.m + k0) = a;
        *(f32x4*)((float*)h.v + k0) = b;
    }
}

template <bool PB, bool GB, bool S8>
__device__ __forceinline__ void adamw_chunk(const MtJob& jb, const MtHyper& h, const MtScal& s, float coef, long c0) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int u = 0; u < MT_CHUNK / MT_BLOCK / 4; ++u) {
        const long b0 = c0 + (u * 4 + wave) * MT_BLOCK;
        if (b0 >= jb.n) break;
        adamw_block<PB, GB, S8>(jb, h, s, coef, b0 + lane * 4, jb.block + b0 / MT_BLOCK, lane);
    }
}

template <bool S8>
__global__ __launch_bounds__(256) void multi_adamw_kernel(const MtTable tab, const MtHyper h, const MtClip clip) {
    const MtFind find(tab);
    const float coef = clip_coef(clip);
    for (uint32_t c = blockIdx.x; c < tab.nchunk; c += gridDim.x) {
        const int j = find(c);
        const MtJob& jb = tab.job[j];
        const long c0 = (long)(c - tab.first[j]) * MT_CHUNK;
        const float* sc = h.scal + 8 * (size_t)(jb.slot_flags >> 2);
        const MtScal s = {sc[0], sc[1], sc[2], __float_as_uint(sc[3]), __float_as_uint(sc[4])};
        switch (jb.slot_flags & 3) {
            case 0: adamw_chunk<false, false, S8>(jb, h, s, coef, c0); break;
            case VAE_MT_GRAD_BF16: adamw_chunk<false, true, S8>(jb, h, s, coef, c0); break;
            case VAE_MT_PARAM_BF16: adamw_chunk<true, false, S8>(jb, h, s, coef, c0); break;
            default: adamw_chunk<true, true, S8>(jb, h, s, coef, c0); break;
        }
    }
}

// masters of the bf16 parameters (and the fp32 parameters themselves) in the state's layout, padding 0
__global__ __launch_bounds__(256) void multi_master_kernel(const MtTable tab, const short* __restrict__ rem, float* __restrict__ out) {
    const MtFind find(tab);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint32_t c = blockIdx.x; c < tab.nchunk; c += gridDim.x) {
        const int j = find(c);
        const MtJob& jb = tab.job[j];
        const long c0 = (long)(c - tab.first[j]) * MT_CHUNK;
        for (int u = 0; u < MT_CHUNK / MT_BLOCK / 4; ++u) {
            const long b0 = c0 + (u * 4 + wave) * MT_BLOCK, i = b0 + lane * 4;
            if (b0 >= jb.n) break;
            const size_t k0 = ((size_t)jb.block + b0 / MT_BLOCK) * MT_BLOCK + lane * 4;
            f32x4 w = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k < jb.n)
                    w[k] = (jb.slot_flags & VAE_MT_PARAM_BF16) ? join_master(((const bf16_t*)jb.p)[i + k], rem[k0 + k]) : ((const float*)jb.p)[i + k];
            *(f32x4*)(out + k0) = w;
        }
    }
}

template <bool BF>
__global__ __launch_bounds__(256) void moments8_unpack_kernel(const uint8_t* __restrict__ qm, const uint8_t* __restrict__ qv,
                                                              const short2* __restrict__ base, void* __restrict__ m, void* __restrict__ v, long nblocks) {
    const int lane = threadIdx.x & 63;
    for (long b = (long)blockIdx.x * 4 + (threadIdx.x >> 6); b < nblocks; b += (long)gridDim.x * 4) {
        const size_t k0 = (size_t)b * MT_BLOCK + lane * 4;
        const uint32_t a = *(const uint32_t*)(qm + k0), c = *(const uint32_t*)(qv + k0);
        const short2 bs = base[b];
        float x[4], y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            x[k] = unpack_m((a >> 8 * k) & 255u, bs.x);
            y[k] = unpack_v((c >> 8 * k) & 255u, bs.y);
        }
        if (BF) {      // 4 significant bits: exact
            *(uint2*)((bf16_t*)m + k0) = make_uint2(pack2bf(x[0], x[1]), pack2bf(x[2], x[3]));
            *(uint2*)((bf16_t*)v + k0) = make_uint2(pack2bf(y[0], y[1]), pack2bf(y[2], y[3]));
        } else {
            *(float4*)((float*)m + k0) = make_float4(x[0], x[1], x[2], x[3]);
            *(float4*)((float*)v + k0) = make_float4(y[0], y[1], y[2], y[3]);
        }
    }
}

// to nearest (half a level up): what is packed here was not rounded the step before, so there is nothing to be unbiased over
__global__ __launch_bounds__(256) void moments8_pack_kernel(const float* __restrict__ m, const float* __restrict__ v, uint8_t* __restrict__ qm,
                                                            uint8_t* __restrict__ qv, short2* __restrict__ base, long nblocks) {
    const int lane = threadIdx.x & 63;
    for (long b = (long)blockIdx.x * 4 + (threadIdx.x >> 6); b < nblocks; b += (long)gridDim.x * 4) {
        const size_t k0 = (size_t)b * MT_BLOCK + lane * 4;
        const float4 a = *(const float4*)(m + k0), c = *(const float4*)(v + k0);
        const float x[4] = {a.x, a.y, a.z, a.w}, y[4] = {c.x, c.y, c.z, c.w};
        int bm, bv;
        block_bases(x, y, bm, bv);
        const float low = __uint_as_float((uint32_t)(bm + 1) << 20);
        uint32_t p = 0, q = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            p |= pack_m(x[k], bm, low, 1u << 19) << 8 * k;
            q |= pack_v(y[k], bv, 1u << 19) << 8 * k;
        }
        *(uint32_t*)(qm + k0) = p;
        *(uint32_t*)(qv + k0) = q;
        if (lane == 0) *(uint32_t*)(base + b) = pack_base(bm, bv);
    }
}

// ---------------------------------------------------------------- host
static int check_tensors(const char* who, const vae_mt_tensor* t, int count, bool params, long nblocks, int nslots, long* chunks) {
    VAE_CHECK(count >= 0 && count <= VAE_MT_MAX_TENSORS && (t || count == 0), "%s: count=%d out of range (0..%d)", who, count, VAE_MT_MAX_TENSORS);
    long total = 0;
    for (int i = 0; i < count; ++i) {
        VAE_CHECK(t[i].n >= 0 && t[i].n < (1L << 40), "%s: tensor %d has n=%ld", who, i, t[i].n);
        VAE_CHECK((t[i].flags & ~3u) == 0, "%s: tensor %d has unknown flags 0x%x", who, i, t[i].flags);
        if (t[i].n == 0) continue;
        VAE_CHECK(t[i].grad && ((uintptr_t)t[i].grad & ((t[i].flags & VAE_MT_GRAD_BF16) ? 1 : 3)) == 0,
                  "%s: tensor %d: gradient is null or not aligned to its type", who, i);
        if (params) {
            VAE_CHECK(t[i].param && ((uintptr_t)t[i].param & ((t[i].flags & VAE_MT_PARAM_BF16) ? 1 : 3)) == 0,
                      "%s: tensor %d: parameter is null or not aligned to its type", who, i);
            VAE_CHECK((long)t[i].block + (t[i].n + MT_BLOCK - 1) / MT_BLOCK <= nblocks, "%s: tensor %d reaches behind the state's %ld blocks", who, i, nblocks);
            VAE_CHECK((long)t[i].slot < nslots, "%s: tensor %d has slot %u of %d", who, i, t[i].slot, nslots);
        }
        total += (t[i].n + MT_CHUNK - 1) / MT_CHUNK;
    }
    VAE_CHECK(total < 0x7FFFFFFFL, "%s: %ld chunks are too many for one call", who, total);
    if (chunks) *chunks = total;
    return 0;
}

// the next launch's table, from tensor `at` on; returns the tensor after its last.  Empty tensors keep their slot (their step counts
// on) but have no chunk: their first chunk is the next tensor's, which find() then prefers.
static int fill_table(const vae_mt_tensor* t, int count, int at, MtTable& tab) {
    tab.count = 0;
    tab.nchunk = 0;
    for (; at < count && tab.count < MT_TENSORS; ++at) {
        const int k = tab.count++;
        tab.first[k] = tab.nchunk;
        tab.job[k] = {t[at].param, t[at].grad, t[at].n, t[at].block, t[at].slot << 2 | t[at].flags};
        tab.nchunk += (uint32_t)((t[at].n + MT_CHUNK - 1) / MT_CHUNK);
    }
    for (int k = tab.count; k < MT_TENSORS; ++k) tab.first[k] = 0xFFFFFFFFu;
    return at;
}
static double elem_bytes(const MtTable& t, int per_grad_f32) {
    double b = 0;
    for (int k = 0; k < t.count; ++k) b += (double)t.job[k].n * ((t.job[k].slot_flags & VAE_MT_GRAD_BF16) ? per_grad_f32 / 2 : per_grad_f32);
    return b;
}
static double elem_count(const MtTable& t) {
    double n = 0;
    for (int k = 0; k < t.count; ++k) n += (double)t.job[k].n;
    return n;
}
static int update_grid(uint32_t nchunk) { return nchunk < 2048u ? (int)nchunk : 2048; }

// sum-of-squares launches over a list (with `prep`: the step is prepared by the same launches); adds their partial sums to *np
static int sumsq_list(const vae_mt_tensor* t, int count, long all_chunks, const MtPrep* prep, bool sums, double* partial, int* np, hipStream_t s) {
    MtTable tab;
    for (int at = 0; at < count;) {
        at = fill_table(t, count, at, tab);
        int n = 0;
        if (sums && tab.nchunk) {
            // of a list longer than one launch each launch gets its share of the partial sums, and at least one
            n = (int)((double)MT_PARTIALS * tab.nchunk / (double)all_chunks);
            if (n < 1) n = 1;
            if ((uint32_t)n > tab.nchunk) n = (int)tab.nchunk;
        }
        if (n == 0 && !prep) continue;
        {
            ProfScope prof("multi_sumsq_kernel", 0.0, n ? elem_bytes(tab, 4) : 0.0, s);
            if (prep) hipLaunchKernelGGL(multi_sumsq_kernel<true>, dim3(n + 1), dim3(256), 0, s, tab, partial + *np, n, *prep);
            else hipLaunchKernelGGL(multi_sumsq_kernel<false>, dim3(n), dim3(256), 0, s, tab, partial + *np, n, MtPrep{});
        }
        VAE_LAUNCH_CHECK("multi_sumsq_kernel");
        *np += n;
    }
    return 0;
}

}  // namespace vae

using namespace vae;

extern "C" int vae_multi_partials(int count) {
    return MT_PARTIALS + (count < 0 ? 0 : count) / MT_TENSORS + 1 + VAE_MT_MAX_GROUPS;
}

extern "C" int vae_multi_grad_norm(const vae_mt_tensor* tensors, int count, double* partial, float grad_mul, float* norm_out, void* stream) {
    long chunks = 0;
    if (check_tensors("vae_multi_grad_norm", tensors, count, false, 0, 0, &chunks)) return 1;
    VAE_CHECK(partial && norm_out, "vae_multi_grad_norm: null pointer");
    hipStream_t s = (hipStream_t)stream;
    int np = 0;
    if (int rc = sumsq_list(tensors, count, chunks, nullptr, true, partial, &np, s)) return rc;
    const MtClip clip = {partial, np ? np : -1, grad_mul, -1.f, norm_out};
    hipLaunchKernelGGL(multi_norm_kernel, dim3(1), dim3(64), 0, s, clip);
    VAE_LAUNCH_CHECK("multi_norm_kernel");
    return 0;
}

extern "C" int vae_multi_clip(const vae_mt_tensor* tensors, int count, double* partial, float grad_mul, float max_norm, float* norm_out, void* stream) {
    long chunks = 0;
    if (check_tensors("vae_multi_clip", tensors, count, false, 0, 0, &chunks)) return 1;
    VAE_CHECK(partial && norm_out, "vae_multi_clip: null pointer");
    VAE_CHECK(max_norm >= 0.f, "vae_multi_clip: max_norm=%g must not be negative or NaN", (double)max_norm);
    if (chunks == 0) return vae_multi_grad_norm(tensors, count, partial, grad_mul, norm_out, stream);
    hipStream_t s = (hipStream_t)stream;
    int np = 0;
    if (int rc = sumsq_list(tensors, count, chunks, nullptr, true, partial, &np, s)) return rc;
    MtTable tab;
    for (int at = 0; at < count;) {
        at = fill_table(tensors, count, at, tab);
        if (!tab.nchunk) continue;
        const MtClip clip = {partial, np, grad_mul, max_norm, norm_out};
        {
            ProfScope prof("multi_scale_kernel", 0.0, elem_bytes(tab, 8), s);
            hipLaunchKernelGGL(multi_scale_kernel, dim3(update_grid(tab.nchunk)), dim3(256), 0, s, tab, clip);
        }
        VAE_LAUNCH_CHECK("multi_scale_kernel");
    }
    return 0;
}

extern "C" int vae_multi_adamw_step(const vae_mt_group* groups, int ngroups, double* partial, float grad_mul, float max_norm, float* norm_out,
                                    void* stream) {
    VAE_CHECK(groups && ngroups >= 1 && ngroups <= VAE_MT_MAX_GROUPS, "vae_multi_adamw_step: ngroups=%d out of range (1..%d)", ngroups, VAE_MT_MAX_GROUPS);
    VAE_CHECK(!(max_norm != max_norm), "vae_multi_adamw_step: max_norm is NaN");
    const bool sums = max_norm >= 0.f || norm_out;
    VAE_CHECK(!sums || partial, "vae_multi_adamw_step: the norm needs its partial sums' buffer");
    long all = 0;
    for (int k = 0; k < ngroups; ++k) {
        const vae_mt_group& q = groups[k];
        VAE_CHECK(q.struct_size == sizeof(vae_mt_group), "vae_multi_adamw_step: vae_mt_group.struct_size is %u, this library's is %zu", q.struct_size,
                  sizeof(vae_mt_group));
        VAE_CHECK(q.state_bits == 32 || q.state_bits == 8, "vae_multi_adamw_step: state_bits=%d must be 32 or 8", q.state_bits);
        VAE_CHECK(q.beta1 >= 0.0 && q.beta1 < 1.0 && q.beta2 >= 0.0 && q.beta2 < 1.0, "vae_multi_adamw_step: betas (%g, %g) must be in [0, 1)", q.beta1, q.beta2);
        VAE_CHECK(q.eps >= 0.0 && q.weight_decay >= 0.0 && (q.lr_dev || q.lr >= 0.0), "vae_multi_adamw_step: lr=%g, eps=%g and weight_decay=%g must not be negative",
                  q.lr, q.eps, q.weight_decay);
        long chunks = 0;
        if (check_tensors("vae_multi_adamw_step", q.tensors, q.count, true, q.nblocks, q.nslots, &chunks)) return 1;
        VAE_CHECK(q.count == 0 || (q.steps && q.scalars), "vae_multi_adamw_step: null step counts or scalars");
        VAE_CHECK(chunks == 0 || (q.exp_avg && q.exp_avg_sq && (q.state_bits == 32 || q.bases)), "vae_multi_adamw_step: null state");
        VAE_CHECK((((uintptr_t)q.exp_avg | (uintptr_t)q.exp_avg_sq | (uintptr_t)q.remainder | (uintptr_t)q.bases | (uintptr_t)q.scalars) & 15) == 0,
                  "vae_multi_adamw_step: state buffers must be 16-byte aligned");
        for (int i = 0; i < q.count; ++i)
            VAE_CHECK(!(q.tensors[i].flags & VAE_MT_PARAM_BF16) || q.tensors[i].n == 0 || q.remainder, "vae_multi_adamw_step: bf16 parameter %d needs the remainder buffer", i);
        all += chunks;
    }
    hipStream_t s = (hipStream_t)stream;
    int np = 0;
    for (int k = 0; k < ngroups; ++k) {
        const vae_mt_group& q = groups[k];
        const MtPrep prep = {q.steps, q.scalars, q.lr_dev, q.lr, q.beta1, q.beta2, q.weight_decay};
        if (int rc = sumsq_list(q.tensors, q.count, all, &prep, sums, partial, &np, s)) return rc;
    }
    if (all == 0 && norm_out) {      // nothing but empty tensors: no launch below writes the norm
        hipLaunchKernelGGL(multi_norm_kernel, dim3(1), dim3(64), 0, s, MtClip{partial, -1, grad_mul, -1.f, norm_out});
        VAE_LAUNCH_CHECK("multi_norm_kernel");
    }
    MtTable tab;
    for (int k = 0; k < ngroups; ++k) {
        const vae_mt_group& q = groups[k];
        const MtHyper h = {q.exp_avg, q.exp_avg_sq, (short2*)q.bases, q.remainder, q.scalars, (float)q.beta1, (float)(1.0 - q.beta1), (float)q.beta2,
                           (float)(1.0 - q.beta2), (float)q.eps};
        for (int at = 0; at < q.count;) {
            at = fill_table(q.tensors, q.count, at, tab);
            if (!tab.nchunk) continue;
            const MtClip clip = {partial, np, grad_mul, max_norm, norm_out};
            const int grid = update_grid(tab.nchunk);
            if (q.state_bits == 8) {
                ProfScope prof("multi_adamw8_kernel", 0.0, elem_bytes(tab, 12) + 4.0 * elem_count(tab), s);
                hipLaunchKernelGGL(multi_adamw_kernel<true>, dim3(grid), dim3(256), 0, s, tab, h, clip);
            } else {
                ProfScope prof("multi_adamw_kernel", 0.0, elem_bytes(tab, 12) + 16.0 * elem_count(tab), s);
                hipLaunchKernelGGL(multi_adamw_kernel<false>, dim3(grid), dim3(256), 0, s, tab, h, clip);
            }
            VAE_LAUNCH_CHECK("multi_adamw_kernel");
        }
    }
    return 0;
}

extern "C" int vae_multi_master(const vae_mt_tensor* tensors, int count, const short* remainder, float* out, long nblocks, void* stream) {
    long chunks = 0;
    VAE_CHECK(out && ((uintptr_t)out & 15) == 0, "vae_multi_master: out is null or not 16-byte aligned");
    VAE_CHECK(count >= 0 && (tensors || count == 0), "vae_multi_master: count=%d", count);
    for (int i = 0; i < count; ++i)
        VAE_CHECK(!(tensors[i].flags & VAE_MT_PARAM_BF16) || tensors[i].n == 0 || remainder, "vae_multi_master: bf16 parameter %d needs the remainder buffer", i);
    if (check_tensors("vae_multi_master", tensors, count, true, nblocks, 0x7FFFFFFF, &chunks)) return 1;
    MtTable tab;
    for (int at = 0; at < count;) {
        at = fill_table(tensors, count, at, tab);
        if (!tab.nchunk) continue;
        {
            ProfScope prof("multi_master_kernel", 0.0, 8.0 * elem_count(tab), (hipStream_t)stream);
            hipLaunchKernelGGL(multi_master_kernel, dim3(update_grid(tab.nchunk)), dim3(256), 0, (hipStream_t)stream, tab, remainder, out);
        }
        VAE_LAUNCH_CHECK("multi_master_kernel");
    }
    return 0;
}

static int blocks_grid(long nblocks) {
    const long g = (nblocks + 3) / 4;
    return (int)(g < 4096 ? g : 4096);
}

extern "C" int vae_moments8_unpack(const void* exp_avg_q, const void* exp_avg_sq_q, const short* bases, void* exp_avg, void* exp_avg_sq, long nblocks,
                                   int bf16_out, void* stream) {
    VAE_CHECK(nblocks >= 0 && nblocks < (1L << 32), "vae_moments8_unpack: nblocks=%ld", nblocks);
    if (nblocks == 0) return 0;
    VAE_CHECK(exp_avg_q && exp_avg_sq_q && bases && exp_avg && exp_avg_sq, "vae_moments8_unpack: null pointer");
    VAE_CHECK((((uintptr_t)exp_avg_q | (uintptr_t)exp_avg_sq_q | (uintptr_t)bases | (uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 15) == 0,
              "vae_moments8_unpack: buffers must be 16-byte aligned");
    {
        ProfScope prof("moments8_unpack_kernel", 0.0, 256.0 * nblocks * (bf16_out ? 6 : 10), (hipStream_t)stream);
        if (bf16_out)
            hipLaunchKernelGGL(moments8_unpack_kernel<true>, dim3(blocks_grid(nblocks)), dim3(256), 0, (hipStream_t)stream, (const uint8_t*)exp_avg_q,
                               (const uint8_t*)exp_avg_sq_q, (const short2*)bases, exp_avg, exp_avg_sq, nblocks);
        else
            hipLaunchKernelGGL(moments8_unpack_kernel<false>, dim3(blocks_grid(nblocks)), dim3(256), 0, (hipStream_t)stream, (const uint8_t*)exp_avg_q,
                               (const uint8_t*)exp_avg_sq_q, (const short2*)bases, exp_avg, exp_avg_sq, nblocks);
    }
    VAE_LAUNCH_CHECK("moments8_unpack_kernel");
    return 0;
}

extern "C" int vae_moments8_pack(const float* exp_avg, const float* exp_avg_sq, void* exp_avg_q, void* exp_avg_sq_q, short* bases, long nblocks, void* stream) {
    VAE_CHECK(nblocks >= 0 && nblocks < (1L << 32), "vae_moments8_pack: nblocks=%ld", nblocks);
    if (nblocks == 0) return 0;
    VAE_CHECK(exp_avg_q && exp_avg_sq_q && bases && exp_avg && exp_avg_sq, "vae_moments8_pack: null pointer");
    VAE_CHECK((((uintptr_t)exp_avg_q | (uintptr_t)exp_avg_sq_q | (uintptr_t)bases | (uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 15) == 0,
              "vae_moments8_pack: buffers must be 16-byte aligned");
    {
        ProfScope prof("moments8_pack_kernel", 0.0, 256.0 * nblocks * 10, (hipStream_t)stream);
        hipLaunchKernelGGL(moments8_pack_kernel, dim3(blocks_grid(nblocks)), dim3(256), 0, (hipStream_t)stream, exp_avg, exp_avg_sq, (uint8_t*)exp_avg_q,
                           (uint8_t*)exp_avg_sq_q, (short2*)bases, nblocks);
    }
    VAE_LAUNCH_CHECK("moments8_pack_kernel");
    return 0;
}
