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
//                that had only been rounded to zero would be a step of size lr * m / eps; 255 = infinite, or beside 0x80 NaN
// A gradient from 5.8e20 on has a square that makes exp_avg_sq infinite.  Its element then takes no more steps, as with moments in 32 bits;
// exp_avg has no further use there and is held as 0, so that its block's base does not see it.
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

#define MT_TENSORS 256           // tensors one launch takes: 32 + 4 bytes of kernel arguments each
#define MT_CHUNK 4096            // elements a workgroup takes at a time
#define AD_DEEP 4                // blocks a wave of the step has in flight
#define MT_BLOCK 256             // elements of one tensor that share a base; a wave's 64 lanes x 4
#define MT_PARTIALS 256          // workgroups (= partial sums) of the norm, one per CU; every launch of a longer list has at least one
#define SQ_THREADS 1024
#define SQ_DEEP 4                // 16-byte loads a thread of the norm has in flight
#define SQ_CHUNK (SQ_THREADS * SQ_DEEP * 4)

// What a call streams through, and holds in memory, above this goes past the caches: fp32 parameters, moments and remainders of a
// step, the gradients a clip rewrites.  The last level holds 256 MB, and a training step touches more than its optimizer does.
// Three models in turn, cached / past the caches, us: step of 4.1 M parameters (65 MB) 22 / 26, 9 M (144 MB) 61 / 53, 20 M 121 / 102,
// 60 M 361 / 297; with 8-bit moments 9 M (90 MB) 51 / 49, 60 M 292 / 269; clip of 20 M gradients (80 MB) 42 / 46, 28 M 62 / 60, 60 M
// 137 / 116.  What stays cached in any case: gradients that the norm has just read and the step reads again, the norm's
// own reads (past the caches: step of 69.8 M 385 against 343), and bf16 parameters, whose accesses are half as wide (151 against 147).
#define MT_STREAM_BYTES 96e6

// Up to this many chunks (four workgroups per CU, all of them running at once) a step without a norm is one launch.  Above, waiting for
// its numbers in every workgroup costs more than the launch that prepares them.  As called from Python, one launch / two, us, 30 tensors of
// together 35 chunks 9.4 / 13.3, 266: 11.4 / 13.9, 996: 21.8 / 23.4, 1970: 41.6 / 42.0, 3921: 75.0 / 72.8; with 8-bit moments 9.3 / 13.5,
// 9.6 / 13.6, 17.0 / 19.6, 28.9 / 27.6, 49.5 / 45.3.
#define MT_OWN_CHUNKS 1024

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
// per-tensor numbers of a step, at scal + 8 * slot
struct MtScal {
    float decay, step, inv_bc2;
    uint32_t phase_m, phase_v;
};

// one chunk's addresses
struct MtChunk {
    void* p;
    const void* g;
    void *m, *v;
    short* rem;
    short2* base;
};

#define DITHER_I 0x9E3779B9u     // 2^32 / golden ratio
#define DITHER_M 0xBB67AE85u     // 2^32 * frac(sqrt 3)
#define DITHER_V 0x6A09E667u     // 2^32 * frac(sqrt 2)

// vectors whose address is only as aligned as one element: the memory system takes any 4-byte (fp32) or 2-byte (bf16) address
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x4u __attribute__((ext_vector_type(4), aligned(2)));

// chunks of a tensor in the step's launch: an empty one has one too, which advances its step count
__host__ __device__ __forceinline__ uint32_t mt_chunks(long n) { return n ? (uint32_t)((n + MT_CHUNK - 1) / MT_CHUNK) : 1u; }

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

// NT: a streaming access, which the caches need not keep
template <bool NT, class T>
__device__ __forceinline__ T ld(const T* p) {
    if (NT) return __builtin_nontemporal_load(p);
    return *p;
}
template <bool NT, class T>
__device__ __forceinline__ void st(T* p, T x) {
    if (NT) __builtin_nontemporal_store(x, p);
    else *p = x;
}

// four consecutive elements at p + o, of which the tensor has `left` (FULL: four); what it has not reads as 0 and is not written
template <bool FULL, bool NT>
__device__ __forceinline__ void load4(const float* p, uint32_t o, int left, float x[4]) {
    if (FULL || left >= 4) {
        const f32x4u q = NT ? __builtin_nontemporal_load((const f32x4u*)(p + o)) : *(const f32x4u*)(p + o);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = q[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = k < left ? p[o + k] : 0.f;
    }
}
template <bool FULL, bool NT>
__device__ __forceinline__ void load4(const bf16_t* p, uint32_t o, int left, u16x4u& x) {
    if (FULL || left >= 4) {
        x = NT ? __builtin_nontemporal_load((const u16x4u*)(p + o)) : *(const u16x4u*)(p + o);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = k < left ? p[o + k] : (bf16_t)0;
    }
}
template <bool BF, bool FULL, bool NT>
__device__ __forceinline__ void load4(const void* p, uint32_t o, int left, float x[4]) {
    if (BF) {
        u16x4u q;
        load4<FULL, NT>((const bf16_t*)p, o, left, q);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = bf2f(q[k]);
    } else {
        load4<FULL, NT>((const float*)p, o, left, x);
    }
}
template <bool FULL, bool NT>
__device__ __forceinline__ void store4(float* p, uint32_t o, int left, const float x[4]) {
    if (FULL || left >= 4) {
        f32x4u q;
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = x[k];
        if (NT) __builtin_nontemporal_store(q, (f32x4u*)(p + o));
        else *(f32x4u*)(p + o) = q;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < left) p[o + k] = x[k];
    }
}
template <bool FULL, bool NT>
__device__ __forceinline__ void store4(bf16_t* p, uint32_t o, int left, const bf16_t x[4]) {
    if (FULL || left >= 4) {
        u16x4u q;
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = x[k];
        if (NT) __builtin_nontemporal_store(q, (u16x4u*)(p + o));
        else *(u16x4u*)(p + o) = q;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < left) p[o + k] = x[k];
    }
}

// ---------------------------------------------------------------- global norm
// Squares and sums in 64 bits: a square of an fp32 gradient can pass fp32's range, and the sum runs over the whole model.
// Bound by HBM, 4 bytes a gradient.  One workgroup of 16 waves per CU, so that every wave of the kernels that read the norm
// folds 256 partial sums (four loads a lane) and needs no launch of its own for that.  279 MB in 88 tensors: 48 us, 5.8 TB/s;
// with 256 threads a workgroup 160 us, with 512 or 1024 workgroups of 256 to 1024 threads and up to 8 loads in flight 47 to 53.
template <bool BF>
__device__ __forceinline__ void sumsq_chunk(const void* g, long c0, long n, double a[4]) {
    const void* p = (const char*)g + c0 * (BF ? 2 : 4);
    const int left = (int)(n - c0 < SQ_CHUNK ? n - c0 : SQ_CHUNK);
    float x[SQ_DEEP][4];
    if (left == SQ_CHUNK) {
#pragma unroll
        for (int u = 0; u < SQ_DEEP; ++u) load4<BF, true, false>(p, (u * SQ_THREADS + threadIdx.x) * 4u, 0, x[u]);
    } else {
#pragma unroll
        for (int u = 0; u < SQ_DEEP; ++u) load4<BF, false, false>(p, (u * SQ_THREADS + threadIdx.x) * 4u, left - (int)((u * SQ_THREADS + threadIdx.x) * 4u), x[u]);
    }
#pragma unroll
    for (int u = 0; u < SQ_DEEP; ++u)
#pragma unroll
        for (int k = 0; k < 4; ++k) a[k] = __builtin_fma((double)x[u][k], (double)x[u][k], a[k]);
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

// What depends on a tensor's step count alone, in 64 bits.  The counts live on the device, so that a captured step counts on when
// it is replayed.
__device__ __forceinline__ MtScal step_numbers(const MtPrep& h, long t) {
    const double lr = h.lr_dev ? (double)*h.lr_dev : h.lr;
    return {(float)(1.0 - lr * h.wd), (float)(lr / (1.0 - int_pow(h.b1, t))), (float)(1.0 / sqrt(1.0 - int_pow(h.b2, t))), (uint32_t)t * DITHER_M,
            (uint32_t)t * DITHER_V};
}
// beside the norm's workgroups: advances the counts and leaves the numbers for the step's launch
__device__ __forceinline__ void prep_tensors(const MtTable& tab, const MtPrep& h) {
    for (int i = threadIdx.x; i < tab.count; i += blockDim.x) {
        const uint32_t slot = tab.job[i].slot_flags >> 2;
        const long t = h.steps[slot] + 1;
        h.steps[slot] = t;
        *(MtScal*)(h.scal + 8 * (size_t)slot) = step_numbers(h, t);
    }
}
// A small step without a norm has no such launch: every workgroup works the numbers out for itself.  The count may advance once all
// of the tensor's workgroups have read it: they are counted (word 7 of the slot's scalars), and the last one writes it.  Called once in a
// workgroup: a list this small has one for every chunk.
__device__ __forceinline__ MtScal own_numbers(const MtPrep& h, uint32_t slot, uint32_t chunks) {
    __shared__ MtScal shared;
    if (threadIdx.x == 0) {
        const long t = h.steps[slot] + 1;
        asm volatile("" ::"v"((uint32_t)t), "v"((uint32_t)(t >> 32)) : "memory");      // the count has arrived
        uint32_t* seen = (uint32_t*)h.scal + 8 * (size_t)slot + 7;
        if (__hip_atomic_fetch_add(seen, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == chunks - 1) {
            h.steps[slot] = t;
            *seen = 0;
        }
        shared = step_numbers(h, t);
    }
    __syncthreads();
    return shared;
}

// workgroups 0..nsum-1: partial sums; with PREP one more, which prepares the step of the same tensors
template <bool PREP>
__global__ __launch_bounds__(SQ_THREADS) void multi_sumsq_kernel(const MtTable tab, double* __restrict__ partial, int nsum, const MtPrep prep) {
    if (PREP && (int)blockIdx.x >= nsum) {
        prep_tensors(tab, prep);
        return;
    }
    __shared__ double red[SQ_THREADS / 64];
    const MtFind find(tab);
    double a4[4] = {0.0, 0.0, 0.0, 0.0};
    for (uint32_t c = blockIdx.x; c < tab.nchunk; c += nsum) {
        const int j = find(c);
        const MtJob& jb = tab.job[j];
        const long c0 = (long)(c - tab.first[j]) * SQ_CHUNK;
        if (jb.slot_flags & VAE_MT_GRAD_BF16) sumsq_chunk<true>(jb.g, c0, jb.n, a4);
        else sumsq_chunk<false>(jb.g, c0, jb.n, a4);
    }
    const double a = wave_sum_d((a4[0] + a4[1]) + (a4[2] + a4[3]));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int w = 0; w < SQ_THREADS / 64; ++w) t += red[w];
        partial[blockIdx.x] = t;
    }
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
    const int lane = threadIdx.x & 63;
    double v[MT_PARTIALS / 64], a = 0.0;
#pragma unroll
    for (int k = 0; k < MT_PARTIALS / 64; ++k) v[k] = lane + k * 64 < c.npartial ? c.partial[lane + k * 64] : 0.0;      // in flight together
#pragma unroll
    for (int k = 0; k < MT_PARTIALS / 64; ++k) a += v[k];
    for (int i = lane + MT_PARTIALS; i < c.npartial; i += 64) a += c.partial[i];      // lists of several launches may have a few more
    a = wave_sum_d(a);
    const double norm = sqrt(a) * fabs((double)c.grad_mul);
    if (blockIdx.x == 0 && threadIdx.x == 0 && c.norm_out) *c.norm_out = (float)norm;
    if (c.max_norm < 0.f) return c.grad_mul;
    const double q = (double)c.max_norm / (norm + 1e-6);
    return (float)(q >= 1.0 ? 1.0 : q) * c.grad_mul;
}

template <bool BF, bool FULL, bool NT>
__device__ __forceinline__ void scale_run(void* g, int left, float coef) {
    float x[4][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) load4<BF, FULL, NT>(g, (u * 256 + threadIdx.x) * 4u, left - (int)((u * 256 + threadIdx.x) * 4u), x[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const uint32_t o = (u * 256 + threadIdx.x) * 4u;
        if (BF) {
            bf16_t y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = f2bf(x[u][k] * coef);
            store4<FULL, NT>((bf16_t*)g, o, left - (int)o, y);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) x[u][k] *= coef;
            store4<FULL, NT>((float*)g, o, left - (int)o, x[u]);
        }
    }
}
template <bool BF, bool NT>
__device__ __forceinline__ void scale_chunk(void* g, long c0, long n, float coef) {
    void* p = (char*)g + c0 * (BF ? 2 : 4);
    if (n - c0 >= MT_CHUNK) scale_run<BF, true, NT>(p, MT_CHUNK, coef);
    else scale_run<BF, false, NT>(p, (int)(n - c0), coef);
}

template <bool NT>
__global__ __launch_bounds__(256) void multi_scale_kernel(const MtTable tab, const MtClip clip) {
    const MtFind find(tab);
    const float coef = clip_coef(clip);
    for (uint32_t w = blockIdx.x; w < tab.nchunk; w += gridDim.x) {
        const uint32_t c = tab.nchunk - 1 - w;      // what the norm has read last is still in the caches
        const int j = find(c);
        const MtJob& jb = tab.job[j];
        const long c0 = (long)(c - tab.first[j]) * MT_CHUNK;
        if (jb.slot_flags & VAE_MT_GRAD_BF16) scale_chunk<true, NT>((void*)jb.g, c0, jb.n, coef);
        else scale_chunk<false, NT>((void*)jb.g, c0, jb.n, coef);
    }
}

__global__ __launch_bounds__(64) void multi_norm_kernel(const MtClip clip) { clip_coef(clip); }

// ---------------------------------------------------------------- 8-bit moments
// maximum over the wave, in a scalar register: within rows of 16 lanes, then across them, towards lane 63
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#define MT_DPP_MAX(ctrl, rows) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xF, false))
    MT_DPP_MAX(0x111, 0xF);      // row_shr:1, 2, 4, 8
    MT_DPP_MAX(0x112, 0xF);
    MT_DPP_MAX(0x114, 0xF);
    MT_DPP_MAX(0x118, 0xF);
    MT_DPP_MAX(0x142, 0xA);      // row_bcast:15, 31
    MT_DPP_MAX(0x143, 0xC);
#undef MT_DPP_MAX
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ bool finite_bits(uint32_t x) { return x < 0x7F800000u; }     // of a magnitude
__device__ __forceinline__ int level_up(uint32_t x) { return min((int)((x + 0xFFFFFu) >> 20), 0x7F7); }

__device__ __forceinline__ float unpack_m(uint32_t q, int base) {
    const uint32_t c = q & 127u;
    uint32_t x = c ? (uint32_t)(base + (int)c) << 20 : 0u;
    x |= (q & 128u) << 24;
    return __uint_as_float(q == 128u ? 0x7FC00000u : x);
}
__device__ __forceinline__ float unpack_v(uint32_t q, int base, bool inf) {
    const uint32_t x = q ? (uint32_t)(base + (int)q) << 20 : 0u;
    return __uint_as_float(q == 255u ? (inf ? 0x7F800000u : 0x7FC00000u) : x);
}
// Does one of the four codes of a word mean "not finite"?  (a byte of x is zero: (x - 01..01) & ~x & 80..80 is not)
__device__ __forceinline__ bool odd_codes(uint32_t qm, uint32_t qv) {
    const uint32_t a = qm ^ 0x80808080u;
    return (((a - 0x01010101u) & ~a) | ((~qv - 0x01010101u) & qv)) & 0x80808080u;
}

// ---------------------------------------------------------------- AdamW
// (parameter, remainder) -> master.  A magnitude below zero can only come of a parameter that was written since, and is 0; so can an
// infinity with a positive remainder, which stays infinite (a master that is rounded to one lies below it).  max(t, inf) lets NaN through.
__device__ __forceinline__ float join_master(bf16_t p, short r) {
    const uint32_t t = (uint32_t)p << 16, mag = t & 0x7FFF0000u;
    uint32_t x;
    asm("v_med3_i32 %0, %1, 0, %2" : "=v"(x) : "v"((int)mag + (int)r), "v"(max(mag, 0x7F800000u)));
    return __uint_as_float(x | (t & 0x80000000u));
}
// master -> (parameter, remainder): adding half a last place rounds the magnitude, and what the upper half is then too
// large or too small by is the lower half, read as a signed number
__device__ __forceinline__ void split_master(float w, bf16_t& p, short& r) {
    const uint32_t x = w != w ? 0x7FC00000u : __float_as_uint(w);
    p = (bf16_t)((x + 0x8000u) >> 16);
    r = (short)(x & 0xFFFFu);
}

// One block of 256 elements of one tensor, a wave's work: 4 elements a lane.  All of a wave's blocks of a chunk are loaded before the
// first is stored: the stores could alias the later loads as far as the compiler knows, and would wait for one another.
// Bound by HBM: 28 bytes a parameter in fp32 with 32-bit moments, 16 with 8-bit ones (26 and 14 in bf16 with remainder).
// 69.8 M fp32 parameters in 88 tensors: 336 us, 5.8 TB/s (295 with the gradients still cached from the norm); 8-bit moments
// 182 us, 6.1 TB/s (a pass over one array in place reaches 5.9).  20 M bf16 parameters in 217 tensors off their alignment: 91 us,
// 5.7 TB/s.
//
// In 8 bits the vector instructions count: 16 bytes a parameter at 5.9 TB/s leave about 100 of them.  The first form took
// 110 a parameter and 240 us, this one 65 (bf16: 78).  So
// - root and reciprocal are the hardware's, 1 ulp each, of a step that is itself a small part of the parameter.  The hardware takes
//   the root of a subnormal for 0, which nobody sees next to an eps of at least 1e-12 (VAE_MT_MIN_EPS8): smaller ones are refused;
// - values that are not finite, their codes, and fp32's last level are looked after in branches that a wave seldom takes;
// - a block's maxima go through the lanes by DPP and end in scalar registers, where the bases are worked out;
// - a full chunk has uniform addresses and no bounds; only a tensor's last chunk looks at its end.
template <bool PB, bool GB, bool S8, bool NT>
struct AdamBlock {
    float p[4], g[4], m[4], v[4];
    uint32_t qm, qv, base;
    short4v r;
    u16x4u pb;

    // o: this lane's first element, counted from the chunk's start; left: elements of the tensor from there on (FULL: at least the
    // whole chunk)
    template <bool FULL>
    __device__ __forceinline__ void load(const MtChunk& c, uint32_t o, int left) {
        load4<GB, FULL, false>(c.g, o, left, g);
        if (PB) {
            load4<FULL, false>((const bf16_t*)c.p, o, left, pb);
            r = ld<NT>((const short4v*)(c.rem + o));
        } else {
            load4<false, FULL, NT>(c.p, o, left, p);
        }
        if (S8) {
            qm = ld<NT>((const uint32_t*)((const uint8_t*)c.m + o));
            qv = ld<NT>((const uint32_t*)((const uint8_t*)c.v + o));
            base = *(const uint32_t*)(c.base + o / MT_BLOCK);
        } else {
            const f32x4 a = ld<NT>((const f32x4*)((const float*)c.m + o)), b = ld<NT>((const f32x4*)((const float*)c.v + o));
#pragma unroll
            for (int k = 0; k < 4; ++k) { m[k] = a[k]; v[k] = b[k]; }
        }
    }

    __device__ __forceinline__ void unpack() {
        const uint32_t b = (uint32_t)__builtin_amdgcn_readfirstlane((int)base), bm = b & 0xFFFFu, bv = b >> 16;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t cm = (qm >> 8 * k) & 127u, cv = (qv >> 8 * k) & 255u;
            m[k] = __uint_as_float((cm ? (cm + bm) << 20 : 0u) | ((qm << (24 - 8 * k)) & 0x80000000u));
            v[k] = __uint_as_float(cv ? (cv + bv) << 20 : 0u);
        }
        if (__any(odd_codes(qm, qv))) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (((qm >> 8 * k) & 255u) == 128u) m[k] = __uint_as_float(0x7FC00000u);
                if (((qv >> 8 * k) & 255u) == 255u) v[k] = __uint_as_float(0x7F800000u);      // NaN only beside one in m, which the step gets from there
            }
        }
    }

    // codes of m and v (which it may change); returns the bases.  i: index of the first element; NEAR: to nearest, without a dither
    template <bool NEAR>
    __device__ __forceinline__ uint32_t pack(uint32_t phase_m, uint32_t phase_v, uint32_t i) {
        uint32_t xm = 0, xv = 0, odd_m = 0, odd_v = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            xm = max(xm, __float_as_uint(m[k]) & 0x7FFFFFFFu);
            xv = max(xv, __float_as_uint(v[k]) & 0x7FFFFFFFu);
        }
        if (__any(max(xm, xv) >= 0x7F700000u)) {
            // not finite: packed as 0 and marked afterwards; fp32's last level: has no level above it to be rounded to
            xm = xv = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t y = __float_as_uint(v[k]) & 0x7FFFFFFFu;
                if (y == 0x7F800000u && finite_bits(__float_as_uint(m[k]) & 0x7FFFFFFFu)) m[k] = 0.f;
                const uint32_t x = __float_as_uint(m[k]) & 0x7FFFFFFFu;
                if (!finite_bits(x)) { odd_m |= 128u << 8 * k; m[k] = 0.f; }
                else if (x > 0x7F700000u) m[k] = copysignf(__uint_as_float(0x7F700000u), m[k]);
                if (!finite_bits(y)) { odd_v |= 255u << 8 * k; v[k] = 0.f; }
                else v[k] = __uint_as_float(min(y, 0x7F700000u));
                xm = max(xm, __float_as_uint(m[k]) & 0x7FFFFFFFu);
                xv = max(xv, __float_as_uint(v[k]));
            }
        }
        const uint32_t bm = (uint32_t)max(level_up(wave_max_u32(xm)) - 127, 0), bv = (uint32_t)max(level_up(wave_max_u32(xv)) - 254, 0);
        const uint32_t low = (bm + 1) << 20, minus_m = 0u - (bm << 20), minus_v = 0u - (bv << 20);
        const float unit = __uint_as_float(low) * 0x1p-20f;
        uint32_t u = i * DITHER_I, cm[4], cv[4];
#pragma unroll
        for (int k = 0; k < 4; ++k, u += DITHER_I) {
            const uint32_t x = __float_as_uint(m[k]) & 0x7FFFFFFFu, y = __float_as_uint(v[k]);
            const uint32_t dm = NEAR ? 1u << 19 : (u + phase_m) >> 12, dv = NEAR ? 1u << 19 : (u + phase_v) >> 12;
            // below the smallest level that has a code: 0 or that level, the latter with probability |m| / low over the
            // dither (d * unit is exact: 20 bits times 4).  Both sides are worked out: a branch would cost more.
            uint32_t small = __uint_as_float(x) > (float)dm * unit ? 1u : 0u, big = (x + dm + minus_m) >> 20;
            asm("" : "+v"(small), "+v"(big));
            cm[k] = x >= low ? big : small;
            cv[k] = (uint32_t)max((int)(y + dv + minus_v) >> 20, (int)min(y, 1u));      // at least 1 unless y is 0
        }
        // the four codes in a word, and the signs of those that are not 0: adding 127 carries into bit 7 of every byte from 1 to 127
        const uint32_t c = cm[0] | cm[1] << 8 | cm[2] << 16 | cm[3] << 24;
        const uint32_t sign = __builtin_amdgcn_perm(__builtin_amdgcn_perm(__float_as_uint(m[3]), __float_as_uint(m[2]), 0x07030C0Cu),
                                                    __builtin_amdgcn_perm(__float_as_uint(m[1]), __float_as_uint(m[0]), 0x0C0C0703u), 0x07060100u);
        qm = c | ((c + 0x7F7F7F7Fu) & sign & 0x80808080u) | odd_m;
        qv = cv[0] | cv[1] << 8 | cv[2] << 16 | cv[3] << 24 | odd_v;
        return bm | bv << 16;
    }

    // i: index of the first element in its tensor
    template <bool FULL>
    __device__ __forceinline__ void step(const MtChunk& c, const MtHyper& h, const MtScal& s, float coef, uint32_t o, int left, uint32_t i) {
        if (PB) {
#pragma unroll
            for (int k = 0; k < 4; ++k) p[k] = join_master(pb[k], r[k]);
        }
        if (S8) unpack();
#pragma unroll
        for (int k = 0; k < 4; ++k) {      // m and v: one rounding per operation, as the plain formula has them
            const float gk = g[k] * coef;
            m[k] = h.b1 * m[k] + h.omb1 * gk;
            v[k] = h.b2 * v[k] + h.omb2 * gk * gk;
            if (!FULL && k >= left) m[k] = v[k] = 0.f;       // the padding stays 0 under a coefficient that is NaN too
        }
        if (S8) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float den = __builtin_fmaf(__builtin_amdgcn_sqrtf(v[k]), s.inv_bc2, h.eps);
                p[k] = __builtin_fmaf(p[k], s.decay, -(s.step * m[k] * __builtin_amdgcn_rcpf(den)));
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) p[k] = p[k] * s.decay - s.step * m[k] / (sqrtf(v[k]) * s.inv_bc2 + h.eps);
        }
        if (PB) {
            bf16_t q[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                short rk;
                split_master(p[k], q[k], rk);
                r[k] = rk;
            }
            store4<FULL, false>((bf16_t*)c.p, o, left, q);
            st<NT>((short4v*)(c.rem + o), r);
        } else {
            store4<FULL, NT>((float*)c.p, o, left, p);
        }
        if (S8) {
            const uint32_t bases = pack<false>(s.phase_m, s.phase_v, i);
            st<NT>((uint32_t*)((uint8_t*)c.m + o), qm);
            st<NT>((uint32_t*)((uint8_t*)c.v + o), qv);
            if ((o & (MT_BLOCK - 1)) == 0) *(uint32_t*)(c.base + o / MT_BLOCK) = bases;
        } else {
            st<NT>((f32x4*)((float*)c.m + o), f32x4{m[0], m[1], m[2], m[3]});
            st<NT>((f32x4*)((float*)c.v + o), f32x4{v[0], v[1], v[2], v[3]});
        }
    }
};

template <bool PB, bool GB, bool S8, bool NT>
__device__ __forceinline__ void adamw_chunk(const MtJob& jb, const MtHyper& h, const MtScal& s, float coef, long c0) {
    const size_t k0 = (size_t)jb.block * MT_BLOCK + c0;
    const MtChunk c = {(char*)jb.p + c0 * (PB ? 2 : 4), (const char*)jb.g + c0 * (GB ? 2 : 4), (char*)h.m + k0 * (S8 ? 1 : 4),
                       (char*)h.v + k0 * (S8 ? 1 : 4), h.rem + k0, h.base + k0 / MT_BLOCK};
    const uint32_t lane4 = (threadIdx.x & 63) * 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i0 = (uint32_t)c0;
    if (jb.n - c0 >= MT_CHUNK) {
#pragma unroll 1
        for (uint32_t b = wave * MT_BLOCK; b < MT_CHUNK; b += 4 * AD_DEEP * MT_BLOCK) {
            AdamBlock<PB, GB, S8, NT> a[AD_DEEP];
#pragma unroll
            for (int u = 0; u < AD_DEEP; ++u) a[u].template load<true>(c, b + u * 4 * MT_BLOCK + lane4, 0);
#pragma unroll
            for (int u = 0; u < AD_DEEP; ++u) {
                const uint32_t o = b + u * 4 * MT_BLOCK + lane4;
                a[u].template step<true>(c, h, s, coef, o, 0, i0 + o);
            }
        }
    } else {
        const int left = (int)(jb.n - c0);
#pragma unroll 1
        for (uint32_t b = wave * MT_BLOCK; (int)b < left; b += 4 * MT_BLOCK) {
            AdamBlock<PB, GB, S8, NT> a;
            const uint32_t o = b + lane4;
            a.template load<false>(c, o, left - (int)o);
            a.template step<false>(c, h, s, coef, o, left - (int)o, i0 + o);
        }
    }
}

template <bool S8, bool NT>
__global__ __launch_bounds__(256) void multi_adamw_kernel(const MtTable tab, const MtHyper h, const MtClip clip, const MtPrep own) {
    const MtFind find(tab);
    const float coef = clip_coef(clip);
    for (uint32_t w = blockIdx.x; w < tab.nchunk; w += gridDim.x) {
        const uint32_t c = tab.nchunk - 1 - w;      // what the norm has read last is still in the caches
        const int j = find(c);
        const MtJob& jb = tab.job[j];
        const long c0 = (long)(c - tab.first[j]) * MT_CHUNK;
        const uint32_t slot = jb.slot_flags >> 2;
        const MtScal s = own.steps ? own_numbers(own, slot, mt_chunks(jb.n)) : *(const MtScal*)(h.scal + 8 * (size_t)slot);
        switch (jb.slot_flags & 3) {
            case 0: adamw_chunk<false, false, S8, NT>(jb, h, s, coef, c0); break;
            case VAE_MT_GRAD_BF16: adamw_chunk<false, true, S8, NT>(jb, h, s, coef, c0); break;
            case VAE_MT_PARAM_BF16: adamw_chunk<true, false, S8, NT>(jb, h, s, coef, c0); break;
            default: adamw_chunk<true, true, S8, NT>(jb, h, s, coef, c0); break;
        }
    }
}

// masters of the bf16 parameters (and the fp32 parameters themselves) in the state's layout, padding 0
template <bool PB, bool FULL, bool NT>
__device__ __forceinline__ void master_chunk(const MtChunk& c, float* out, int left) {
    float w[MT_CHUNK / 1024][4];
    short4v r[MT_CHUNK / 1024];
    u16x4u p[MT_CHUNK / 1024];
#pragma unroll
    for (int u = 0; u < MT_CHUNK / 1024; ++u) {
        const uint32_t o = (u * 256 + threadIdx.x) * 4u;
        if (!FULL && (int)(o & ~(MT_BLOCK - 1u)) >= left) break;       // a block behind the tensor's last is another tensor's
        if (PB) {
            load4<FULL, false>((const bf16_t*)c.p, o, left - (int)o, p[u]);
            r[u] = ld<NT>((const short4v*)(c.rem + o));
        } else {
            load4<FULL, false>((const float*)c.p, o, left - (int)o, w[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < MT_CHUNK / 1024; ++u) {
        const uint32_t o = (u * 256 + threadIdx.x) * 4u;
        if (!FULL && (int)(o & ~(MT_BLOCK - 1u)) >= left) break;
        if (PB) {
#pragma unroll
            for (int k = 0; k < 4; ++k) w[u][k] = FULL || (int)o + k < left ? join_master(p[u][k], r[u][k]) : 0.f;
        }
        st<NT>((f32x4*)(out + o), f32x4{w[u][0], w[u][1], w[u][2], w[u][3]});
    }
}
template <bool NT>
__global__ __launch_bounds__(256) void multi_master_kernel(const MtTable tab, const short* __restrict__ rem, float* __restrict__ out) {
    const MtFind find(tab);
    for (uint32_t c = blockIdx.x; c < tab.nchunk; c += gridDim.x) {
        const int j = find(c);
        const MtJob& jb = tab.job[j];
        const long c0 = (long)(c - tab.first[j]) * MT_CHUNK;
        const size_t k0 = (size_t)jb.block * MT_BLOCK + c0;
        const bool bf = jb.slot_flags & VAE_MT_PARAM_BF16, full = jb.n - c0 >= MT_CHUNK;
        const int left = full ? MT_CHUNK : (int)(jb.n - c0);
        MtChunk k = {(char*)jb.p + c0 * (bf ? 2 : 4), nullptr, nullptr, nullptr, (short*)rem + k0, nullptr};
        if (bf && full) master_chunk<true, true, NT>(k, out + k0, left);
        else if (bf) master_chunk<true, false, NT>(k, out + k0, left);
        else if (full) master_chunk<false, true, NT>(k, out + k0, left);
        else master_chunk<false, false, NT>(k, out + k0, left);
    }
}

// 8 elements a thread: 16-byte stores
template <bool BF, bool NT>
__global__ __launch_bounds__(256) void moments8_unpack_kernel(const uint8_t* __restrict__ qm, const uint8_t* __restrict__ qv,
                                                              const short2* __restrict__ base, void* __restrict__ m, void* __restrict__ v, long n, bool inf) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += (long)gridDim.x * 2048) {
        const u32x2 a = ld<NT>((const u32x2*)(qm + i)), c = ld<NT>((const u32x2*)(qv + i));
        const short2 b = base[i / MT_BLOCK];
        float x[8], y[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t p = (a[k / 4] >> 8 * (k & 3)) & 255u;
            x[k] = unpack_m(p, b.x);
            y[k] = unpack_v((c[k / 4] >> 8 * (k & 3)) & 255u, b.y, inf && p != 128u);
        }
        if (BF) {      // 4 significant bits: exact
            st<NT>((u32x4*)((bf16_t*)m + i), u32x4{pack2bf(x[0], x[1]), pack2bf(x[2], x[3]), pack2bf(x[4], x[5]), pack2bf(x[6], x[7])});
            st<NT>((u32x4*)((bf16_t*)v + i), u32x4{pack2bf(y[0], y[1]), pack2bf(y[2], y[3]), pack2bf(y[4], y[5]), pack2bf(y[6], y[7])});
        } else {
#pragma unroll
            for (int h = 0; h < 8; h += 4) {
                st<NT>((f32x4*)((float*)m + i + h), f32x4{x[h], x[h + 1], x[h + 2], x[h + 3]});
                st<NT>((f32x4*)((float*)v + i + h), f32x4{y[h], y[h + 1], y[h + 2], y[h + 3]});
            }
        }
    }
}

// to nearest (half a level up): what is packed here was not rounded the step before, so there is nothing to be unbiased over
__global__ __launch_bounds__(256) void moments8_pack_kernel(const float* __restrict__ m, const float* __restrict__ v, uint8_t* __restrict__ qm,
                                                            uint8_t* __restrict__ qv, short2* __restrict__ base, long nblocks) {
    const int lane = threadIdx.x & 63;
    for (long b = (long)blockIdx.x * 4 + (threadIdx.x >> 6); b < nblocks; b += (long)gridDim.x * 4) {
        const size_t k0 = (size_t)b * MT_BLOCK + lane * 4;
        const float4 x = *(const float4*)(m + k0), y = *(const float4*)(v + k0);
        AdamBlock<false, false, true, false> a;
        a.m[0] = x.x; a.m[1] = x.y; a.m[2] = x.z; a.m[3] = x.w;
        a.v[0] = y.x; a.v[1] = y.y; a.v[2] = y.z; a.v[3] = y.w;
#pragma unroll
        for (int k = 0; k < 4; ++k) a.v[k] = fabsf(a.v[k]);      // it has no sign bit
        const uint32_t bases = a.template pack<true>(0u, 0u, 0u);
        *(uint32_t*)(qm + k0) = a.qm;
        *(uint32_t*)(qv + k0) = a.qv;
        if (lane == 0) *(uint32_t*)(base + b) = bases;
    }
}

// ---------------------------------------------------------------- host
// *sq_chunks: what the norm's workgroups take in turn, over all tensors
static int check_tensors(const char* who, const vae_mt_tensor* t, int count, bool grads, bool params, long nblocks, long nslots, long* sq_chunks) {
    VAE_CHECK(count >= 0 && count <= VAE_MT_MAX_TENSORS && (t || count == 0), "%s: count=%d out of range (0..%d)", who, count, VAE_MT_MAX_TENSORS);
    long total = 0, sq = 0;
    for (int i = 0; i < count; ++i) {
        VAE_CHECK(t[i].n >= 0 && t[i].n < (1L << 40), "%s: tensor %d has n=%ld", who, i, t[i].n);
        VAE_CHECK((t[i].flags & ~3u) == 0, "%s: tensor %d has unknown flags 0x%x", who, i, t[i].flags);
        VAE_CHECK(!params || (long)t[i].slot < nslots, "%s: tensor %d has slot %u of %ld", who, i, t[i].slot, nslots);      // an empty one counts its steps too
        if (t[i].n == 0) continue;
        VAE_CHECK(!grads || (t[i].grad && ((uintptr_t)t[i].grad & ((t[i].flags & VAE_MT_GRAD_BF16) ? 1 : 3)) == 0),
                  "%s: tensor %d: gradient is null or not aligned to its type", who, i);
        if (params) {
            VAE_CHECK(t[i].param && ((uintptr_t)t[i].param & ((t[i].flags & VAE_MT_PARAM_BF16) ? 1 : 3)) == 0,
                      "%s: tensor %d: parameter is null or not aligned to its type", who, i);
            VAE_CHECK((long)t[i].block + (t[i].n + MT_BLOCK - 1) / MT_BLOCK <= nblocks, "%s: tensor %d reaches behind the state's %ld blocks", who, i, nblocks);
        }
        total += (t[i].n + MT_CHUNK - 1) / MT_CHUNK;
        sq += (t[i].n + SQ_CHUNK - 1) / SQ_CHUNK;
    }
    VAE_CHECK(total < 0x7FFFFFFFL, "%s: %ld chunks are too many for one call", who, total);
    *sq_chunks = sq;
    return 0;
}

// the next launch's table, from tensor `at` on; returns the tensor after its last.  A tensor without a chunk has the next one's as its
// first, and find() takes the last of them.
// chunk: elements, or 0: the step's (mt_chunks)
static int fill_table(const vae_mt_tensor* t, int count, int at, int chunk, MtTable& tab) {
    tab.count = 0;
    tab.nchunk = 0;
    for (; at < count && tab.count < MT_TENSORS; ++at) {
        const int k = tab.count++;
        tab.first[k] = tab.nchunk;
        tab.job[k] = {t[at].param, t[at].grad, t[at].n, t[at].block, t[at].slot << 2 | t[at].flags};
        tab.nchunk += chunk ? (uint32_t)((t[at].n + chunk - 1) / chunk) : mt_chunks(t[at].n);
    }
    for (int k = tab.count; k < MT_TENSORS; ++k) tab.first[k] = 0xFFFFFFFFu;
    return at;
}
// the first tensor of a list's last launch; negative: there is none
static int last_table(int count) { return count > 0 ? (count - 1) / MT_TENSORS * MT_TENSORS : -1; }
static double elem_bytes(const MtTable& t, int per_grad_f32) {
    double b = 0;
    for (int k = 0; k < t.count; ++k) b += (double)t.job[k].n * ((t.job[k].slot_flags & VAE_MT_GRAD_BF16) ? per_grad_f32 / 2 : per_grad_f32);
    return b;
}
static double grad_bytes(const vae_mt_tensor* t, int count) {
    double b = 0;
    for (int k = 0; k < count; ++k) b += (double)t[k].n * ((t[k].flags & VAE_MT_GRAD_BF16) ? 2 : 4);
    return b;
}
static double elem_count(const MtTable& t) {
    double n = 0;
    for (int k = 0; k < t.count; ++k) n += (double)t.job[k].n;
    return n;
}
// bytes a step's launch moves: gradient read, parameter (and remainder) and moments both ways
static double step_bytes(const MtTable& t, bool eight) {
    double b = 0;
    for (int k = 0; k < t.count; ++k)
        b += (double)t.job[k].n * (((t.job[k].slot_flags & VAE_MT_GRAD_BF16) ? 2 : 4) + 8 + (eight ? 4 : 16));
    return b;
}
// a workgroup per chunk; beyond 4.3 G elements they take several
static int update_grid(uint32_t nchunk) { return nchunk < (1u << 20) ? (int)nchunk : 1 << 20; }

// sum-of-squares launches over a list (with `prep`: the step is prepared by the same launches; without `partial`: that alone); adds
// the number of their partial sums to *np
static int sumsq_list(const vae_mt_tensor* t, int count, long all_chunks, const MtPrep* prep, double* partial, int* np, hipStream_t s) {
    MtTable tab;
    for (int at = 0; at < count;) {
        at = fill_table(t, count, at, SQ_CHUNK, tab);
        int n = 0;
        if (partial && tab.nchunk) {
            // of a list longer than one launch each launch gets its share of the partial sums, and at least one
            n = (int)((double)MT_PARTIALS * tab.nchunk / (double)all_chunks);
            if (n < 1) n = 1;
            if ((uint32_t)n > tab.nchunk) n = (int)tab.nchunk;
        }
        if (n == 0 && !prep) continue;
        {
            ProfScope prof("multi_sumsq_kernel", 0.0, n ? elem_bytes(tab, 4) : 0.0, s);
            if (prep) hipLaunchKernelGGL(multi_sumsq_kernel<true>, dim3(n + 1), dim3(SQ_THREADS), 0, s, tab, partial + *np, n, *prep);
            else hipLaunchKernelGGL(multi_sumsq_kernel<false>, dim3(n), dim3(SQ_THREADS), 0, s, tab, partial + *np, n, MtPrep{});
        }
        VAE_LAUNCH_CHECK("multi_sumsq_kernel");
        *np += n;
    }
    return 0;
}

}  // namespace vae

using namespace vae;

extern "C" int vae_multi_partials(int count) {
    return MT_PARTIALS + (count < 0 ? 0 : count) / (MT_TENSORS / 2) + 1 + VAE_MT_MAX_GROUPS;      // more than there are launches
}

extern "C" int vae_multi_grad_norm(const vae_mt_tensor* tensors, int count, double* partial, float grad_mul, float* norm_out, void* stream) {
    long chunks = 0;
    if (check_tensors("vae_multi_grad_norm", tensors, count, true, false, 0, 0, &chunks)) return 1;
    VAE_CHECK(partial && norm_out, "vae_multi_grad_norm: null pointer");
    hipStream_t s = (hipStream_t)stream;
    int np = 0;
    if (int rc = sumsq_list(tensors, count, chunks, nullptr, partial, &np, s)) return rc;
    const MtClip clip = {partial, np ? np : -1, grad_mul, -1.f, norm_out};
    hipLaunchKernelGGL(multi_norm_kernel, dim3(1), dim3(64), 0, s, clip);
    VAE_LAUNCH_CHECK("multi_norm_kernel");
    return 0;
}

extern "C" int vae_multi_clip(const vae_mt_tensor* tensors, int count, double* partial, float grad_mul, float max_norm, float* norm_out, void* stream) {
    long chunks = 0;
    if (check_tensors("vae_multi_clip", tensors, count, true, false, 0, 0, &chunks)) return 1;
    VAE_CHECK(partial && norm_out, "vae_multi_clip: null pointer");
    VAE_CHECK(max_norm >= 0.f, "vae_multi_clip: max_norm=%g must not be negative or NaN", (double)max_norm);
    if (chunks == 0) return vae_multi_grad_norm(tensors, count, partial, grad_mul, norm_out, stream);
    hipStream_t s = (hipStream_t)stream;
    const bool nt = grad_bytes(tensors, count) > MT_STREAM_BYTES;
    int np = 0;
    if (int rc = sumsq_list(tensors, count, chunks, nullptr, partial, &np, s)) return rc;
    MtTable tab;
    for (int at = last_table(count); at >= 0; at -= MT_TENSORS) {
        fill_table(tensors, count, at, MT_CHUNK, tab);
        if (!tab.nchunk) continue;
        const MtClip clip = {partial, np, grad_mul, max_norm, norm_out};
        {
            ProfScope prof("multi_scale_kernel", 0.0, elem_bytes(tab, 8), s);
            if (nt) hipLaunchKernelGGL(multi_scale_kernel<true>, dim3(update_grid(tab.nchunk)), dim3(256), 0, s, tab, clip);
            else hipLaunchKernelGGL(multi_scale_kernel<false>, dim3(update_grid(tab.nchunk)), dim3(256), 0, s, tab, clip);
        }
        VAE_LAUNCH_CHECK("multi_scale_kernel");
    }
    return 0;
}

static MtPrep prep_of(const vae_mt_group& q) { return {q.steps, q.scalars, q.lr_dev, q.lr, q.beta1, q.beta2, q.weight_decay}; }

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
        VAE_CHECK(q.state_bits == 32 || q.eps >= VAE_MT_MIN_EPS8, "vae_multi_adamw_step: eps=%g: 8-bit moments need at least %g", q.eps, VAE_MT_MIN_EPS8);
        VAE_CHECK(q.eps >= 0.0 && q.weight_decay >= 0.0 && (q.lr_dev || q.lr >= 0.0), "vae_multi_adamw_step: lr=%g, eps=%g and weight_decay=%g must not be negative",
                  q.lr, q.eps, q.weight_decay);
        VAE_CHECK(q.nslots >= 0 && q.nslots <= VAE_MT_MAX_TENSORS, "vae_multi_adamw_step: nslots=%d out of range (0..%d)", q.nslots, VAE_MT_MAX_TENSORS);
        long chunks = 0;
        if (check_tensors("vae_multi_adamw_step", q.tensors, q.count, true, true, q.nblocks, q.nslots, &chunks)) return 1;
        VAE_CHECK(((uintptr_t)q.steps & 7) == 0 && ((uintptr_t)q.lr_dev & 3) == 0, "vae_multi_adamw_step: steps or lr_dev not aligned to its type");
        VAE_CHECK(q.count == 0 || (q.steps && q.scalars), "vae_multi_adamw_step: null step counts or scalars");
        VAE_CHECK(chunks == 0 || (q.exp_avg && q.exp_avg_sq && (q.state_bits == 32 || q.bases)), "vae_multi_adamw_step: null state");
        VAE_CHECK((((uintptr_t)q.exp_avg | (uintptr_t)q.exp_avg_sq | (uintptr_t)q.remainder | (uintptr_t)q.bases | (uintptr_t)q.scalars) & 15) == 0,
                  "vae_multi_adamw_step: state buffers must be 16-byte aligned");
        for (int i = 0; i < q.count; ++i)
            VAE_CHECK(!(q.tensors[i].flags & VAE_MT_PARAM_BF16) || q.tensors[i].n == 0 || q.remainder, "vae_multi_adamw_step: bf16 parameter %d needs the remainder buffer", i);
        all += chunks;
    }
    hipStream_t s = (hipStream_t)stream;
    // what the step holds in memory, all groups together
    double bytes = 0.0;
    long step_chunks = 0;
    for (int k = 0; k < ngroups; ++k)
        for (int i = 0; i < groups[k].count; ++i) {
            const vae_mt_tensor& t = groups[k].tensors[i];
            step_chunks += mt_chunks(t.n);
            bytes += (double)t.n * ((t.flags & VAE_MT_GRAD_BF16 ? 2 : 4) + 4 + (groups[k].state_bits == 8 ? 2 : 8));
        }
    const bool nt = bytes > MT_STREAM_BYTES;
    int np = 0;
    const bool norm = sums && all > 0, own = !norm && step_chunks <= MT_OWN_CHUNKS;
    for (int k = 0; k < ngroups && !own; ++k) {
        const MtPrep prep = prep_of(groups[k]);
        if (int rc = sumsq_list(groups[k].tensors, groups[k].count, all, &prep, norm ? partial : nullptr, &np, s)) return rc;
    }
    if (!norm && norm_out) {      // nothing but empty tensors: no launch below writes the norm
        hipLaunchKernelGGL(multi_norm_kernel, dim3(1), dim3(64), 0, s, MtClip{partial, -1, grad_mul, -1.f, norm_out});
        VAE_LAUNCH_CHECK("multi_norm_kernel");
    }
    MtTable tab;
    for (int k = ngroups - 1; k >= 0; --k) {       // from the last launch to the first, as within a launch
        const vae_mt_group& q = groups[k];
        const MtHyper h = {q.exp_avg, q.exp_avg_sq, (short2*)q.bases, q.remainder, q.scalars, (float)q.beta1, (float)(1.0 - q.beta1), (float)q.beta2,
                           (float)(1.0 - q.beta2), (float)q.eps};
        for (int at = last_table(q.count); at >= 0; at -= MT_TENSORS) {
            fill_table(q.tensors, q.count, at, 0, tab);
            if (!tab.nchunk) continue;
            const MtClip clip = {partial, np, grad_mul, max_norm, norm_out};
            const MtPrep numbers = own ? prep_of(q) : MtPrep{};
            const int grid = update_grid(tab.nchunk);
            const bool eight = q.state_bits == 8;
            ProfScope prof(eight ? "multi_adamw8_kernel" : "multi_adamw_kernel", 0.0, step_bytes(tab, eight), s);
            if (eight && nt) hipLaunchKernelGGL((multi_adamw_kernel<true, true>), dim3(grid), dim3(256), 0, s, tab, h, clip, numbers);
            else if (eight) hipLaunchKernelGGL((multi_adamw_kernel<true, false>), dim3(grid), dim3(256), 0, s, tab, h, clip, numbers);
            else if (nt) hipLaunchKernelGGL((multi_adamw_kernel<false, true>), dim3(grid), dim3(256), 0, s, tab, h, clip, numbers);
            else hipLaunchKernelGGL((multi_adamw_kernel<false, false>), dim3(grid), dim3(256), 0, s, tab, h, clip, numbers);
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
    if (check_tensors("vae_multi_master", tensors, count, false, true, nblocks, 1L << 32, &chunks)) return 1;
    MtTable tab;
    for (int at = 0; at < count;) {
        at = fill_table(tensors, count, at, MT_CHUNK, tab);
        if (!tab.nchunk) continue;
        {
            ProfScope prof("multi_master_kernel", 0.0, 8.0 * elem_count(tab), (hipStream_t)stream);
            const auto kernel = 2048.0 * nblocks > MT_STREAM_BYTES ? multi_master_kernel<true> : multi_master_kernel<false>;
            hipLaunchKernelGGL(kernel, dim3(update_grid(tab.nchunk)), dim3(256), 0, (hipStream_t)stream, tab, remainder, out);
        }
        VAE_LAUNCH_CHECK("multi_master_kernel");
    }
    return 0;
}

// workgroups of four blocks (pack) or eight (unpack) each
static int blocks_grid(long nblocks, int per) {
    const long g = (nblocks + per - 1) / per;
    return (int)(g < (1 << 20) ? g : 1 << 20);
}

extern "C" int vae_moments8_unpack(const void* exp_avg_q, const void* exp_avg_sq_q, const short* bases, void* exp_avg, void* exp_avg_sq, long nblocks,
                                   int flags, void* stream) {
    VAE_CHECK((flags & ~(VAE_M8_BF16 | VAE_M8_INF)) == 0, "vae_moments8_unpack: unknown flags 0x%x", flags);
    const bool bf16_out = flags & VAE_M8_BF16;
    VAE_CHECK(nblocks >= 0 && nblocks < (1L << 32), "vae_moments8_unpack: nblocks=%ld", nblocks);
    if (nblocks == 0) return 0;
    VAE_CHECK(exp_avg_q && exp_avg_sq_q && bases && exp_avg && exp_avg_sq, "vae_moments8_unpack: null pointer");
    VAE_CHECK((((uintptr_t)exp_avg_q | (uintptr_t)exp_avg_sq_q | (uintptr_t)bases | (uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 15) == 0,
              "vae_moments8_unpack: buffers must be 16-byte aligned");
    {
        ProfScope prof("moments8_unpack_kernel", 0.0, 256.0 * nblocks * (bf16_out ? 6 : 10), (hipStream_t)stream);
        const bool nt = 256.0 * nblocks * (bf16_out ? 6 : 10) > MT_STREAM_BYTES;
        const auto kernel = bf16_out ? (nt ? moments8_unpack_kernel<true, true> : moments8_unpack_kernel<true, false>)
                                     : (nt ? moments8_unpack_kernel<false, true> : moments8_unpack_kernel<false, false>);
        hipLaunchKernelGGL(kernel, dim3(blocks_grid(nblocks, 8)), dim3(256), 0, (hipStream_t)stream, (const uint8_t*)exp_avg_q,
                           (const uint8_t*)exp_avg_sq_q, (const short2*)bases, exp_avg, exp_avg_sq, nblocks * MT_BLOCK, (flags & VAE_M8_INF) != 0);
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
        hipLaunchKernelGGL(moments8_pack_kernel, dim3(blocks_grid(nblocks, 4)), dim3(256), 0, (hipStream_t)stream, exp_avg, exp_avg_sq, (uint8_t*)exp_avg_q,
                           (uint8_t*)exp_avg_sq_q, (short2*)bases, nblocks);
    }
    VAE_LAUNCH_CHECK("moments8_pack_kernel");
    return 0;
}
