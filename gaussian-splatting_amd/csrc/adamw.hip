// AdamW over many tensors in one launch, with moments in 32 bits or in 8, and what a training loop needs around it: the
// global gradient norm that clips the step, the selection of state rows when rows are pruned or added, and the values
// that packed states stand for.
//
// The update of one element, t = the 1-based count of this update:
//     g  = g * min(1, max_norm / (norm + 1e-6))           with clipping only
//     m  = beta1 m + (1 - beta1) g
//     v  = beta2 v + (1 - beta2) g^2
//     p  = p (1 - lr wd) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
// Everything is fp32 whatever the parameter's type.
//
// 32-bit states: rounding for rounding what torch.optim.AdamW's foreach path computes on the same GPU (the forms at the top of
// optimizer.hip, after p *= fl(1 - lr wd)).
//
// 8-bit states: per element one byte for m and one for u = sqrt(v), interleaved; per block of 64 consecutive elements of
// the flattened tensor two fp32 scales, the block's largest |m| and largest u.  A level is a bit pattern counted down from 1.0f:
//     m: sign, c = 0..127:  c = 0 is 0, else scale * float(0x3F800000 - (127 - c) * 2^20)     8 levels per octave
//     u:       c = 0..255:  c = 0 is 0, else scale * float(0x3F800000 - (255 - c) * 2^19)    16 levels per octave
// Both reach 15.8 octaves below the scale.  u rather than v is kept because it needs half the octaves.  Below its
// lowest level m goes to 0 or to that level; u goes up to it, so that u is 0 only if v is: an element whose u were
// rounded away would divide its m by eps.
// Rounding is stochastic by default: the bit pattern plus 16 random bits, cut (exactly unbiased: within an octave the levels
// are linear in the value).  With beta2 = 0.999 an update moves u by less than 1/60 of a level, which rounding to
// nearest would swallow every time.  The random bits are a hash of (seed, tensor, update, element): no state, and the
// same results whatever the launch looks like.
//
// A NaN makes its whole block NaN (its maximum is), loudly; an infinity leaves nothing of its block's other moments, which start over.
//
// bf16 parameters: p holds the fp32 value rounded to bf16 (halves away from zero), a 16-bit remainder in units of the
// fp32's last place holds the rest, so value = (bits(p) << 16) + remainder.  It costs what an fp32 parameter costs, and a
// parameter that was overwritten from outside with a finite value is off by no more than half a bf16 step.
#include "gsplat_common.h"
#include "../../include/gsplat.h"
#include <math.h>
#pragma clang fp contract(off)

namespace {

constexpr int AW_THREADS = 256;
constexpr int AW_MAX_TENSORS = 32;      // tensors per launch: the table travels in the kernel arguments (4 KB)
constexpr int AW_CHUNK = 2048;          // elements per workgroup, a multiple of AW_THREADS and of GS_ADAMW_BLOCK
// The same for the step.  One group of four elements a lane hides its latency behind other waves where the work is all memory (32 bits,
// 3 M Gaussians: 946 us against 952 with two groups); with codes to compute, two share the workgroup's prologue (533 us
// against 556 with one; with four 532, at 5 waves a SIMD instead of 8).
constexpr int aw_step_chunk(bool q8) { return q8 ? 2048 : 1024; }

// A (rows, row_len) matrix as a chunk of consecutive elements sees it: where the chunk starts (the same for the whole workgroup, so
// scalar arithmetic), and the row of an element `off` further on by one 32-bit multiply-high.  Chunks have at most 8192 elements.
struct AwDivisor { unsigned long long magic; uint32_t len, magic32; };    // floor(2^64 / len) + 1, floor(2^32 / len) + 1; len 0: contiguous
struct AwRows { long long row; uint32_t col, len, magic32; };
struct AwPlace { uint32_t q, col; };                                      // rows after the chunk's first, column
__device__ __forceinline__ AwRows aw_rows(long long base, const AwDivisor& d) {
    const long long row = d.len == 1 ? base : (long long)__umul64hi((unsigned long long)base, d.magic);
    return AwRows{row, (uint32_t)(base - row * d.len), d.len, d.magic32};
}
__device__ __forceinline__ AwPlace aw_place(const AwRows& r, uint32_t off) {
    const uint32_t x = r.col + off;       // < len + 8192
    if (r.len >= 8192u) return x >= r.len ? AwPlace{1u, x - r.len} : AwPlace{0u, x};
    const uint32_t q = r.len == 1 ? x : __umulhi(x, r.magic32);          // exact: x * len < 2^28
    return AwPlace{q, x - __umul24(q, r.len)};
}

struct AwTensor {
    void* p;
    const void* g;
    int16_t* low;
    void* m;                  // fp32 moments, or the code pairs
    float* v;                 // fp32 moments, or the scale pairs
    long long n;
    long long g_row_stride;
    AwDivisor rows;           // of the gradient
    float neg_step, decay, bc2;   // -(lr / (1 - beta1^t)), 1 - lr wd, sqrt(1 - beta2^t) (8 bits: its reciprocal)
    float beta1, beta2, one_minus_beta1, one_minus_beta2, eps;
    uint32_t key;
    int slot;                 // place in `scalars`
    uint32_t blocks, every;   // workgroups; > 0: `every` workgroups of the next tensor follow on each of this one's (see aw_pair)
};

struct AwArgs {
    AwTensor t[AW_MAX_TENSORS];
    uint32_t block_begin[AW_MAX_TENSORS + 1];
    int count;
    int stochastic;
    const float4* scalars;    // (neg_step, decay, bc2, key) per tensor written by adamw_scalars_kernel, or null
    const float* grad_norm;   // or null
    float max_norm;
};

static_assert(sizeof(AwArgs) <= 4096, "kernel arguments");

__host__ __device__ __forceinline__ uint32_t aw_mix(uint32_t x) {
    // two rounds of xor-shift and multiply (odd constants: fractional bits of sqrt(2) and sqrt(3))
    x ^= x >> 16; x *= 0x6A09E667u;
    x ^= x >> 15; x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}

__device__ __forceinline__ float aw_coef(const float* norm, float max_norm) {
    const float c = __fdiv_rn(max_norm, *norm + 1e-6f);
    return c > 1.0f ? 1.0f : c;           // a NaN norm stays NaN
}

// aw_split() gives a zero no negative remainder; one that was left behind when the parameter was set to zero from outside would borrow
// through the sign and make a NaN of it, and is dropped.
__device__ __forceinline__ float aw_join(uint16_t high, int16_t low) {
    const uint32_t h = (uint32_t)high << 16, x = h + (uint32_t)(int32_t)low;
    return __uint_as_float((int32_t)(x ^ h) < 0 ? h : x);
}
__device__ __forceinline__ void aw_split(float x, uint16_t& high, int16_t& low) {
    const uint32_t b = x != x ? 0x7FC00000u : __float_as_uint(x);
    high = (uint16_t)((b + 0x8000u) >> 16);
    low = (int16_t)(b & 0xFFFFu);
}
__device__ __forceinline__ float aw_bf16(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }

__device__ __forceinline__ float aw_level_m(uint32_t code, float scale) {
    const uint32_t c = code & 127u;
    const float f = __uint_as_float((c << 20) + (0x3F800000u - (127u << 20))) * scale;
    return c == 0 ? 0.0f : __uint_as_float(__float_as_uint(f) ^ (code & 128u) << 24);
}
__device__ __forceinline__ float aw_level_u(uint32_t code, float scale) {
    const float f = __uint_as_float((code << 19) + (0x3F800000u - (255u << 19))) * scale;
    return code == 0 ? 0.0f : f;
}
// x = the value over its block's scale, at most 1 (also for NaN); r = 16 random bits, 32768 rounds to nearest
__device__ __forceinline__ uint32_t aw_code_m(float x, uint32_t value_bits, uint32_t r) {
    int c = (int)((r << 4) + __float_as_uint(x) - (0x3F800000u - (127u << 20))) >> 20;
    const int lowest = x * (65536.0f / (1.25f * 0x1p-16f)) > (float)r ? 1 : 0;
    c = c > lowest ? c : lowest;          // below the lowest level c is 0 or negative
    return c == 0 ? 0u : (uint32_t)c | (value_bits >> 24 & 128u);
}
__device__ __forceinline__ uint32_t aw_code_u(float x, uint32_t r) {
    const int c = (int)((r << 3) + __float_as_uint(x) - (0x3F800000u - (255u << 19))) >> 19;
    return x == 0.0f ? 0u : (uint32_t)(c < 1 ? 1 : c);
}
// the scale to keep and the factor that takes values to 0..1 (subnormal maxima count as zero: their reciprocal overflows)
__device__ __forceinline__ float aw_scale(uint32_t max_bits, float& inverse) {
    const float scale = max_bits < 0x00800000u ? 0.0f : __uint_as_float(max_bits);
    const float x = __fdiv_rn(1.0f, scale);
    inverse = max_bits < 0x00800000u ? 0.0f : x;
    return scale;
}
// The largest of x over the 16 lanes of a DPP row, in all of them.
__device__ __forceinline__ uint32_t aw_row_max(uint32_t x) {
    uint32_t y;
    y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, true); x = x > y ? x : y;   // row_ror:8
    y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xf, 0xf, true); x = x > y ? x : y;   // row_ror:4
    y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xf, 0xf, true); x = x > y ? x : y;   // row_ror:2
    y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xf, 0xf, true); x = x > y ? x : y;   // row_ror:1
    return x;
}

// Four consecutive elements belong to a lane and a block of 64 to the 16 lanes of a DPP row: loads and stores are 16 bytes
// wide (8 for 16-bit types and code pairs) and the block's maxima take four DPP steps, no LDS and no barrier.  The hardware
// takes such accesses at any multiple of the element's size, so views need no form of their own.
constexpr int AW_LANE = 4;
constexpr int AW_ITERS = AW_CHUNK / (AW_THREADS * AW_LANE);
static_assert(GS_ADAMW_BLOCK == 16 * AW_LANE && AW_CHUNK % (AW_THREADS * AW_LANE) == 0, "a DPP row holds a block");

typedef float f4v __attribute__((ext_vector_type(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));
typedef float f4m __attribute__((ext_vector_type(4), aligned(4)));        // as they lie in memory
typedef uint32_t u2m __attribute__((ext_vector_type(2), aligned(2)));

// Codes of four elements: m[], u[] in, the pairs and the block's scales out.
__device__ __forceinline__ u2v aw_pack4(const float* m, const float* u, const uint32_t* r, float& sm, float& su) {
    uint32_t mm = 0, mu = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const uint32_t bm = __float_as_uint(m[c]) & 0x7FFFFFFFu, bu = __float_as_uint(u[c]);
        mm = mm > bm ? mm : bm;
        mu = mu > bu ? mu : bu;
    }
    float im, iu;
    sm = aw_scale(aw_row_max(mm), im);
    su = aw_scale(aw_row_max(mu), iu);
    uint32_t pair[4];
#pragma unroll
    for (int c = 0; c < 4; ++c)
        pair[c] = aw_code_m(fminf(fabsf(m[c]) * im, 1.0f), __float_as_uint(m[c]), r[c] & 0xFFFFu) |
                  aw_code_u(fminf(u[c] * iu, 1.0f), r[c] >> 16) << 8;
    return u2v{pair[0] | pair[1] << 16, pair[2] | pair[3] << 16};
}

// how many of the four elements at `off` lie among the `left` ones
__device__ __forceinline__ int aw_count(int off, int left) { return off >= left ? 0 : left - off < 4 ? left - off : 4; }
// elements i .. i + 3 of a tensor, the first `count` of them (zeros for the rest)
__device__ __forceinline__ f4v aw_load4(const float* p, int i, int count) {
    f4v x{0.0f, 0.0f, 0.0f, 0.0f};
    if (count == 4) x = *reinterpret_cast<const f4m*>(p + i);
    else
#pragma unroll
        for (int c = 0; c < 3; ++c)
            if (c < count) x[c] = p[i + c];
    return x;
}
__device__ __forceinline__ u2v aw_load4(const uint16_t* p, int i, int count) {
    u2v x{0, 0};
    if (count == 4) x = *reinterpret_cast<const u2m*>(p + i);
    else
#pragma unroll
        for (int c = 0; c < 3; ++c)
            if (c < count) x[c / 2] |= (uint32_t)p[i + c] << (c % 2 * 16);
    return x;
}
// Streamed once per call and mostly far larger than the caches: non-temporal, out of the way of the reads.
__device__ __forceinline__ void aw_store4(float* p, int i, int count, f4v x) {
    if (count == 4) __builtin_nontemporal_store(x, reinterpret_cast<f4m*>(p + i));
    else
#pragma unroll
        for (int c = 0; c < 3; ++c)
            if (c < count) p[i + c] = x[c];
}
__device__ __forceinline__ void aw_store4(uint16_t* p, int i, int count, u2v x) {
    if (count == 4) __builtin_nontemporal_store(x, reinterpret_cast<u2m*>(p + i));
    else
#pragma unroll
        for (int c = 0; c < 3; ++c)
            if (c < count) p[i + c] = (uint16_t)(x[c / 2] >> (c % 2 * 16));
}
__device__ __forceinline__ uint32_t aw_half(u2v x, int c) { return x[c / 2] >> (c % 2 * 16) & 0xFFFFu; }

// Four elements, `off` after the start of a chunk, of a matrix with a row stride.  Lanes whose elements lie in one row take them at once.
template <class Element>
__device__ __forceinline__ auto aw_load4_rows(const Element* p, long long base, int off, int count, const AwRows& r, long long stride) {
    if (r.len == 0) return aw_load4(p + base, off, count);
    AwPlace at = aw_place(r, (uint32_t)off);
    const Element* row = p + (r.row + at.q) * stride;
    if (at.col + 4 <= r.len) return aw_load4(row, at.col, count);
    decltype(aw_load4(p, 0, count)) x{};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (c < count) {
            const Element y = row[at.col];
            if constexpr (sizeof(Element) == 4) x[c] = y;
            else x[c / 2] |= (uint32_t)y << (c % 2 * 16);
        }
        if (++at.col == r.len) { at.col = 0; row += stride; }
    }
    return x;
}

template <bool BF16> struct AwTypes { typedef f4v vec; typedef float element; };
template <> struct AwTypes<true> { typedef u2v vec; typedef uint16_t element; };

struct AwScalars { float neg_step, decay, bc2, coef; uint32_t key; bool clip; };

// FAST: the whole chunk lies inside the tensor.
template <bool BF16, bool Q8, bool FAST>
__device__ __forceinline__ void adamw_chunk(const AwArgs& a, const AwTensor& T, const AwScalars& S, long long base) {
    constexpr int CHUNK = aw_step_chunk(Q8), ITERS = CHUNK / (AW_THREADS * AW_LANE);
    typedef typename AwTypes<BF16>::vec PVec;
    typedef typename AwTypes<BF16>::element PElement;
    PVec p4[ITERS], g4[ITERS];
    u2v low4[ITERS], codes[ITERS];
    f4v m4[ITERS], v4[ITERS];
    float2 scale[ITERS];
    const AwRows rows = aw_rows(base, T.rows);
    const int left = FAST ? CHUNK : T.n - base < CHUNK ? (int)(T.n - base) : CHUNK;
    PElement* const pp = (PElement*)T.p + base;
    uint16_t* const pl = (uint16_t*)T.low + base;
    uint16_t* const pc = (uint16_t*)T.m + base;           // 8 bits: the code pairs and scale pairs
    float2* const ps = (float2*)T.v + base / GS_ADAMW_BLOCK;
    float* const pm = (float*)T.m + base;                 // 32 bits: the moments
    float* const pv = T.v + base;
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
        const int off = (i * AW_THREADS + (int)threadIdx.x) * AW_LANE;
        const int count = FAST ? 4 : aw_count(off, left);
        p4[i] = aw_load4(pp, off, count);
        if (BF16) low4[i] = aw_load4(pl, off, count);
        if (Q8) {
            codes[i] = aw_load4(pc, off, count);
            scale[i] = count > 0 ? ps[off / GS_ADAMW_BLOCK] : make_float2(0.0f, 0.0f);
        } else {
            m4[i] = aw_load4(pm, off, count);
            v4[i] = aw_load4(pv, off, count);
        }
        g4[i] = aw_load4_rows((const PElement*)T.g, base, off, count, rows, T.g_row_stride);
    }
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
        const int off = (i * AW_THREADS + (int)threadIdx.x) * AW_LANE;
        const int count = FAST ? 4 : aw_count(off, left);
        float p[4], m[4], v[4], u[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            float g;
            if constexpr (BF16) {
                p[c] = aw_join((uint16_t)aw_half(p4[i], c), (int16_t)aw_half(low4[i], c));
                g = aw_bf16((uint16_t)aw_half(g4[i], c));
            } else {
                p[c] = p4[i][c];
                g = g4[i][c];
            }
            if (S.clip) g = g * S.coef;
            p[c] = p[c] * S.decay;
            if (Q8) {
                const uint32_t pair = aw_half(codes[i], c);
                const float x = aw_level_u(pair >> 8, scale[i].y);
                m[c] = aw_level_m(pair & 255u, scale[i].x) * T.beta1 + g * T.one_minus_beta1;
                v[c] = (x * x) * T.beta2 + (g * g) * T.one_minus_beta2;
                u[c] = sqrtf(v[c]);
                // v_rcp_f32 is off by 1 ulp: of the update, not of a state
                p[c] = __fmaf_rn(S.neg_step, m[c] * __builtin_amdgcn_rcpf(u[c] * S.bc2 + T.eps), p[c]);
            } else {
                m[c] = __fmaf_rn(T.one_minus_beta1, g - m4[i][c], m4[i][c]);
                v[c] = __fmaf_rn(T.one_minus_beta2, g * g, v4[i][c] * T.beta2);
                u[c] = sqrtf(v[c]);
                p[c] = __fmaf_rn(S.neg_step, __fdiv_rn(m[c], __fdiv_rn(u[c], S.bc2) + T.eps), p[c]);
            }
        }
        if (Q8) {
            uint32_t r[4];
            // chunks do not cross a multiple of 2^32
            const uint32_t seed = (uint32_t)base + S.key + (uint32_t)((unsigned long long)base >> 32) * 0x3C6EF373u + (uint32_t)off;
#pragma unroll
            for (int c = 0; c < 4; ++c) r[c] = a.stochastic ? aw_mix(seed + c) : 0x80008000u;
            float2 s;
            aw_store4(pc, off, count, aw_pack4(m, u, r, s.x, s.y));      // past the end everything is 0
            if (count > 0 && (threadIdx.x & 15) == 0) ps[off / GS_ADAMW_BLOCK] = s;
        } else {
            aw_store4(pm, off, count, f4v{m[0], m[1], m[2], m[3]});
            aw_store4(pv, off, count, f4v{v[0], v[1], v[2], v[3]});
        }
        if constexpr (BF16) {
            u2v h{0, 0}, l{0, 0};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint16_t high; int16_t low;
                aw_split(p[c], high, low);
                h[c / 2] |= (uint32_t)high << (c % 2 * 16);
                l[c / 2] |= (uint32_t)(uint16_t)low << (c % 2 * 16);
            }
            aw_store4(pp, off, count, h);
            aw_store4(pl, off, count, l);
        } else {
            aw_store4(pp, off, count, f4v{p[0], p[1], p[2], p[3]});
        }
    }
}

// Memory-bound in every form, one pass, everything read and written once (3 M Gaussians = 177 M elements, six tensors, the colour
// gradients strided): fp32 with 32-bit moments 28 B an element, 0.95 ms = 5.2 TB/s; with 8-bit states 16.25 B, 0.53 ms = 5.4 TB/s at 101
// VALU instructions an element, three quarters of the issue slots; a 2 GiB copy reaches 4.9 TB/s.  bf16 parameters (16 M elements):
// 26 B in 64 us, 14.25 B in 46 us.
template <bool BF16, bool Q8>
__global__ __launch_bounds__(AW_THREADS) void adamw_kernel(const AwArgs a) {
    int ti = 0;
    for (int k = 1; k < a.count; ++k) ti += blockIdx.x >= a.block_begin[k] ? 1 : 0;
    uint32_t block = blockIdx.x - a.block_begin[ti];
    if (a.t[ti].every) {
        const uint32_t every = a.t[ti].every, blocks = a.t[ti].blocks, group = block / (every + 1);
        const uint32_t place = block - group * (every + 1);
        if (group >= blocks) { block -= blocks; ++ti; }
        else if (place > 0) { block = group * every + place - 1; ++ti; }
        else block = group;
    }
    const AwTensor& T = a.t[ti];
    constexpr int CHUNK = aw_step_chunk(Q8);
    const long long base = (long long)block * CHUNK;
    AwScalars S{T.neg_step, T.decay, T.bc2, 1.0f, T.key, a.grad_norm != nullptr};
    if (a.scalars) {
        const float4 s = a.scalars[T.slot];
        S.neg_step = s.x; S.decay = s.y; S.bc2 = s.z; S.key = __float_as_uint(s.w);
    }
    if (S.clip) S.coef = aw_coef(a.grad_norm, a.max_norm);
    if (base + CHUNK <= T.n) adamw_chunk<BF16, Q8, true>(a, T, S, base);
    else adamw_chunk<BF16, Q8, false>(a, T, S, base);
}

// ---- counts and learning rates kept on the device (so that a captured step counts on when it is replayed) ----------
struct AwScalarTensor { float* step; const float* lr_dev; double lr, beta1, beta2, weight_decay; uint32_t seed; int pad; };
struct AwScalarArgs { AwScalarTensor t[AW_MAX_TENSORS]; int count; int reciprocal; float4* out; };

__global__ __launch_bounds__(64) void adamw_scalars_kernel(const AwScalarArgs a) {
    const int k = threadIdx.x;
    if (k >= a.count) return;
    const AwScalarTensor& T = a.t[k];
    const float step = *T.step + 1.0f;
    *T.step = step;
    const double lr = T.lr_dev ? (double)*T.lr_dev : T.lr;
    const double root = sqrt(1.0 - pow(T.beta2, (double)step));
    a.out[k] = make_float4((float)(-(lr / (1.0 - pow(T.beta1, (double)step)))), (float)(1.0 - lr * T.weight_decay),
                           (float)(a.reciprocal ? 1.0 / root : root), __uint_as_float(aw_mix(T.seed ^ (uint32_t)step)));
}

// ---- sum of squares over many tensors -------------------------------------------------------------------------------
// The order of the elements is free, so a lane takes a group of four elements of one row (contiguous tensors are one row): group j
// starts at element 4 j, or at the row's fourth from last, and then leaves out what the group before it has.  No load
// crosses a row, none depends on another, and all eight of a lane are under way before the first use.  Bound by reading: 708 MB in
// 0.12 ms = 5.7 TB/s (torch.sum reads at 4.0); doubles cost nothing beside that.
constexpr int NRM_MAX_TENSORS = 48;
constexpr int NRM_GROUPS = 2048;        // groups per workgroup and partial sum
struct NrmTensor {
    const void* g;
    long long groups, row_stride, row_len;
    AwDivisor per_row;                  // groups of a row; len 0: one row
    int bf16;
};
struct NrmArgs { NrmTensor t[NRM_MAX_TENSORS]; uint32_t block_begin[NRM_MAX_TENSORS + 1]; int count; double* partial; };

__device__ __forceinline__ double nrm_block_sum(double s, double* lds) {
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d, 64);
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) lds[wave] = s;
    __syncthreads();
    s = 0.0;
    if (threadIdx.x == 0)
        for (int w = 0; w < (int)blockDim.x >> 6; ++w) s += lds[w];
    return s;
}

template <class Element>
__device__ __forceinline__ double nrm_chunk(const NrmTensor& T, long long base) {
    constexpr int ITERS = NRM_GROUPS / AW_THREADS;
    decltype(aw_load4((const Element*)nullptr, 0, 4)) x[ITERS];
    int skip[ITERS];                    // elements of the group that do not count
    const AwRows rows = aw_rows(base, T.per_row);
    const int last = T.groups - base < NRM_GROUPS ? (int)(T.groups - base) - 1 : NRM_GROUPS - 1;
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
        const int off = i * AW_THREADS + (int)threadIdx.x, o = off < last ? off : last;
        const Element* p;
        if (T.per_row.len == 0) {
            const long long over = 4 * (base + o) - (T.row_len - 4);
            skip[i] = over > 0 ? (int)over : 0;
            p = (const Element*)T.g + 4 * base + (4 * o - skip[i]);
        } else {
            const AwPlace at = aw_place(rows, (uint32_t)o);
            const int over = (int)(4 * at.col) - ((int)T.row_len - 4);
            skip[i] = over > 0 ? over : 0;
            p = (const Element*)T.g + (rows.row + at.q) * T.row_stride + (4 * (int)at.col - skip[i]);
        }
        if (T.row_len >= 4) {
            x[i] = aw_load4(p, 0, 4);
        } else {                        // the row's elements sit in the places that count
            x[i] = {};
#pragma unroll
            for (int c = 1; c < 4; ++c)
                if (c >= 4 - T.row_len) {
                    if constexpr (sizeof(Element) == 4) x[i][c] = p[c];
                    else x[i][c / 2] |= (uint32_t)p[c] << (c % 2 * 16);
                }
        }
        if (off > last) skip[i] = 4;
    }
    double s0 = 0.0, s1 = 0.0;          // two sums, so that the additions of a lane do not wait for each other
#pragma unroll
    for (int i = 0; i < ITERS; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            float y;
            if constexpr (sizeof(Element) == 4) y = x[i][c];
            else y = aw_bf16((uint16_t)aw_half(x[i], c));
            const double z = c < skip[i] ? 0.0f : y;
            if (c & 1) s1 = fma(z, z, s1);
            else s0 = fma(z, z, s0);
        }
    return s0 + s1;
}

__global__ __launch_bounds__(AW_THREADS) void grad_norm_partial_kernel(const NrmArgs a) {
    __shared__ double lds[AW_THREADS / 64];
    int ti = 0;
    for (int k = 1; k < a.count; ++k) ti += blockIdx.x >= a.block_begin[k] ? 1 : 0;
    const NrmTensor& T = a.t[ti];
    const long long base = (long long)(blockIdx.x - a.block_begin[ti]) * NRM_GROUPS;
    double s = T.bf16 ? nrm_chunk<uint16_t>(T, base) : nrm_chunk<float>(T, base);
    s = nrm_block_sum(s, lds);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = s;
}

constexpr int NRM_FINAL_THREADS = 1024;
__global__ __launch_bounds__(NRM_FINAL_THREADS) void grad_norm_final_kernel(long long n, const double* partial, float* out) {
    __shared__ double lds[NRM_FINAL_THREADS / 64];
    // eight loads under way at a time: a lane's sum is a chain of loads otherwise (8.6 us for 21 600 partial sums)
    double s = 0.0;
    for (long long k = threadIdx.x; k < n; k += 8 * NRM_FINAL_THREADS) {
        double x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = k + i * NRM_FINAL_THREADS < n ? partial[k + i * NRM_FINAL_THREADS] : 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += x[i];
    }
    s = nrm_block_sum(s, lds);
    if (threadIdx.x == 0) *out = (float)sqrt(s);
}

// ---- rows of the states ---------------------------------------------------------------------------------------------
struct RowTensor {
    const void* src_m; const float* src_v; const int16_t* src_low;
    void* dst_m; float* dst_v; int16_t* dst_low;
    long long n;                          // elements of the new state
    AwDivisor rows;
};
struct RowArgs { RowTensor t[AW_MAX_TENSORS]; uint32_t block_begin[AW_MAX_TENSORS + 1]; int count; long long src_rows; const int64_t* index; };

__device__ __forceinline__ bool rows_valid(const RowArgs& a, long long row) { return row >= 0 && row < a.src_rows; }

// x[c] = (lo, hi)[c + shift], shift 0..3
__device__ __forceinline__ f4v rows_window(f4v lo, f4v hi, int shift) {
    float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
    for (int c = 0; c < 6; ++c) x[c] = shift & 1 ? x[c + 1] : x[c];
#pragma unroll
    for (int c = 0; c < 4; ++c) x[c] = shift & 2 ? x[c + 2] : x[c];
    return f4v{x[0], x[1], x[2], x[3]};
}
__device__ __forceinline__ u2v rows_window(u2v lo, u2v hi, int shift) {
    const uint64_t l = lo[0] | (uint64_t)lo[1] << 32, h = hi[0] | (uint64_t)hi[1] << 32;
    const uint64_t x = shift ? l >> (16 * shift) | h << (64 - 16 * shift) : l;
    return u2v{(uint32_t)x, (uint32_t)(x >> 32)};
}

template <bool Q8>
__device__ __forceinline__ void rows_store(const RowTensor& T, long long base, int off, int count, f4v m, f4v v, u2v low) {
    if (Q8) {
        const uint32_t r[4] = {0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
        const float mm[4] = {m[0], m[1], m[2], m[3]}, uu[4] = {v[0], v[1], v[2], v[3]};
        float2 s;
        aw_store4((uint16_t*)T.dst_m + base, off, count, aw_pack4(mm, uu, r, s.x, s.y));
        if (count > 0 && (threadIdx.x & 15) == 0) ((float2*)T.dst_v)[base / GS_ADAMW_BLOCK + off / GS_ADAMW_BLOCK] = s;
    } else {
        aw_store4((float*)T.dst_m + base, off, count, m);
        aw_store4(T.dst_v + base, off, count, v);
    }
    if (T.dst_low) aw_store4((uint16_t*)T.dst_low + base, off, count, low);
}

// Rows of four elements and more: a lane's four elements lie in one row or in two.  It loads four elements of the first row (the row's
// last four if they end there) and, if needed, the first four of the second, and shifts them together: no load
// depends on another but on the index.  Every phase runs for all of the lane's groups before the next one, so that the loads overlap.
template <bool Q8>
__device__ __forceinline__ void rows_long(const RowArgs& a, const RowTensor& T, long long base) {
    const AwRows rows = aw_rows(base, T.rows);
    const int left = T.n - base < AW_CHUNK ? (int)(T.n - base) : AW_CHUNK;
    const int64_t* const index = a.index + rows.row;
    long long k0[AW_ITERS], k1[AW_ITERS];     // first the rows, then where the lane's elements of the first and second row start in the source
    int shift[AW_ITERS];
    uint32_t col[AW_ITERS];
#pragma unroll
    for (int i = 0; i < AW_ITERS; ++i) {
        const int off = (i * AW_THREADS + (int)threadIdx.x) * AW_LANE;
        const AwPlace at = aw_place(rows, (uint32_t)off);
        const int over = (int)(at.col + 4 - rows.len);    // elements in the second row
        shift[i] = over > 0 ? over : 0;
        col[i] = at.col - shift[i];
        k0[i] = k1[i] = -1;
        if (off < left) k0[i] = index[at.q];
        if (over > 0 && off + 4 - over < left) k1[i] = index[at.q + 1];
    }
    u2v p0[AW_ITERS], p1[AW_ITERS], l0[AW_ITERS], l1[AW_ITERS];
    f4v m0[AW_ITERS], m1[AW_ITERS], v0[AW_ITERS], v1[AW_ITERS];
    float2 s00[AW_ITERS], s01[AW_ITERS], s10[AW_ITERS], s11[AW_ITERS];
#pragma unroll
    for (int i = 0; i < AW_ITERS; ++i) {
        p0[i] = p1[i] = l0[i] = l1[i] = u2v{0, 0};
        m0[i] = m1[i] = v0[i] = v1[i] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
        s00[i] = s01[i] = s10[i] = s11[i] = make_float2(0.0f, 0.0f);
        if (rows_valid(a, k0[i])) {
            const long long k = k0[i] = k0[i] * rows.len + col[i];
            if (Q8) {
                p0[i] = aw_load4((const uint16_t*)T.src_m + k, 0, 4);
                s00[i] = ((const float2*)T.src_v)[k / GS_ADAMW_BLOCK];
                s01[i] = ((const float2*)T.src_v)[(k + 3) / GS_ADAMW_BLOCK];
            } else {
                m0[i] = aw_load4((const float*)T.src_m + k, 0, 4);
                v0[i] = aw_load4(T.src_v + k, 0, 4);
            }
            if (T.src_low) l0[i] = aw_load4((const uint16_t*)T.src_low + k, 0, 4);
        }
        if (rows_valid(a, k1[i])) {
            const long long k = k1[i] = k1[i] * rows.len;
            if (Q8) {
                p1[i] = aw_load4((const uint16_t*)T.src_m + k, 0, 4);
                s10[i] = ((const float2*)T.src_v)[k / GS_ADAMW_BLOCK];
                s11[i] = ((const float2*)T.src_v)[(k + 3) / GS_ADAMW_BLOCK];
            } else {
                m1[i] = aw_load4((const float*)T.src_m + k, 0, 4);
                v1[i] = aw_load4(T.src_v + k, 0, 4);
            }
            if (T.src_low) l1[i] = aw_load4((const uint16_t*)T.src_low + k, 0, 4);
        }
    }
#pragma unroll
    for (int i = 0; i < AW_ITERS; ++i) {
        const int off = (i * AW_THREADS + (int)threadIdx.x) * AW_LANE;
        f4v m, v;
        if (Q8) {
            const u2v pairs = rows_window(p0[i], p1[i], shift[i]);
            // the place of the first element that belongs to the second of the two blocks, seen from the group's first element
            const int second0 = GS_ADAMW_BLOCK - (int)(k0[i] & (GS_ADAMW_BLOCK - 1)) - shift[i];
            const int first1 = 4 - shift[i], second1 = first1 + GS_ADAMW_BLOCK - (int)(k1[i] & (GS_ADAMW_BLOCK - 1));
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float2 s = c < first1 ? (c < second0 ? s00[i] : s01[i]) : (c < second1 ? s10[i] : s11[i]);
                m[c] = aw_level_m(aw_half(pairs, c) & 255u, s.x);
                v[c] = aw_level_u(aw_half(pairs, c) >> 8, s.y);
            }
        } else {
            m = rows_window(m0[i], m1[i], shift[i]);
            v = rows_window(v0[i], v1[i], shift[i]);
        }
        rows_store<Q8>(T, base, off, aw_count(off, left), m, v, rows_window(l0[i], l1[i], shift[i]));
    }
}

// Rows of one to three elements: one by one, again in phases.
template <bool Q8>
__device__ __forceinline__ void rows_short(const RowArgs& a, const RowTensor& T, long long base) {
    const AwRows rows = aw_rows(base, T.rows);
    const int left = T.n - base < AW_CHUNK ? (int)(T.n - base) : AW_CHUNK;
    const int64_t* const index = a.index + rows.row;
    long long k[AW_ITERS][4];
#pragma unroll
    for (int i = 0; i < AW_ITERS; ++i) {
        const int off = (i * AW_THREADS + (int)threadIdx.x) * AW_LANE;
        AwPlace at = aw_place(rows, (uint32_t)off);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            k[i][c] = off + c < left ? index[at.q] : -1;
            if (++at.col == rows.len) { at.col = 0; ++at.q; }
        }
    }
    uint32_t pair[AW_ITERS][4];
    float2 s[AW_ITERS][4];
    f4v m[AW_ITERS], v[AW_ITERS];
    u2v low[AW_ITERS];
#pragma unroll
    for (int i = 0; i < AW_ITERS; ++i) {
        uint32_t col = aw_place(rows, (uint32_t)((i * AW_THREADS + (int)threadIdx.x) * AW_LANE)).col;
        low[i] = u2v{0, 0};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            pair[i][c] = 0;
            s[i][c] = make_float2(0.0f, 0.0f);
            m[i][c] = v[i][c] = 0.0f;
            if (rows_valid(a, k[i][c])) {
                const long long j = k[i][c] * rows.len + col;
                if (Q8) {
                    pair[i][c] = ((const uint16_t*)T.src_m)[j];
                    s[i][c] = ((const float2*)T.src_v)[j / GS_ADAMW_BLOCK];
                } else {
                    m[i][c] = ((const float*)T.src_m)[j];
                    v[i][c] = T.src_v[j];
                }
                if (T.src_low) low[i][c / 2] |= (uint32_t)(uint16_t)T.src_low[j] << (c % 2 * 16);
            }
            if (++col == rows.len) col = 0;
        }
    }
#pragma unroll
    for (int i = 0; i < AW_ITERS; ++i) {
        const int off = (i * AW_THREADS + (int)threadIdx.x) * AW_LANE;
        if (Q8)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                m[i][c] = aw_level_m(pair[i][c] & 255u, s[i][c].x);
                v[i][c] = aw_level_u(pair[i][c] >> 8, s[i][c].y);
            }
        rows_store<Q8>(T, base, off, aw_count(off, left), m[i], v[i], low[i]);
    }
}

// 3 M rows to 3 M, all six tensors: 32 bits 2.78 GB in 0.53 ms = 5.2 TB/s, memory-bound (one element a lane: 0.63 ms).  8 bits
// 0.75 GB in 0.33 ms = 2.3 TB/s: 78 VALU instructions an element to unpack two codes with up to four scales a group, find the new maxima
// and pack again, behind a chain of three dependent loads (table, index, codes).  Neither alone is the bound: 8 % fewer
// instructions gave 2 %, one or four groups a lane instead of two 360 and 376 us.
template <bool Q8>
__global__ __launch_bounds__(AW_THREADS) void adamw_rows_kernel(const RowArgs a) {
    int ti = 0;
    for (int k = 1; k < a.count; ++k) ti += blockIdx.x >= a.block_begin[k] ? 1 : 0;
    const RowTensor& T = a.t[ti];
    const long long base = (long long)(blockIdx.x - a.block_begin[ti]) * AW_CHUNK;
    if (T.rows.len >= 4) rows_long<Q8>(a, T, base);
    else rows_short<Q8>(a, T, base);
}

// ---- what packed states and split parameters stand for ----------------------------------------------------------------
// 2 B and a share of the scales read, 8 B written: 177 M elements in 0.30 ms = 6.0 TB/s.
struct UnpackTensor { const uint16_t* codes; const float2* scales; const uint16_t* p; const int16_t* low; float* m; float* v; float* x; long long n; };
struct UnpackArgs { UnpackTensor t[AW_MAX_TENSORS]; uint32_t block_begin[AW_MAX_TENSORS + 1]; int count; };

__global__ __launch_bounds__(AW_THREADS) void adamw_unpack_kernel(const UnpackArgs a) {
    int ti = 0;
    for (int k = 1; k < a.count; ++k) ti += blockIdx.x >= a.block_begin[k] ? 1 : 0;
    const UnpackTensor& T = a.t[ti];
    const long long base = (long long)(blockIdx.x - a.block_begin[ti]) * AW_CHUNK;
    const int left = T.n - base < AW_CHUNK ? (int)(T.n - base) : AW_CHUNK;
#pragma unroll
    for (int i = 0; i < AW_ITERS; ++i) {
        const int off = (i * AW_THREADS + (int)threadIdx.x) * AW_LANE;
        if (off >= left) return;
        const int count = aw_count(off, left);
        if (T.codes) {
            const float2 s = T.scales[base / GS_ADAMW_BLOCK + off / GS_ADAMW_BLOCK];
            const u2v pairs = aw_load4(T.codes + base, off, count);
            f4v m, v;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float u = aw_level_u(aw_half(pairs, c) >> 8, s.y);
                m[c] = aw_level_m(aw_half(pairs, c) & 255u, s.x);
                v[c] = u * u;
            }
            aw_store4(T.m + base, off, count, m);
            aw_store4(T.v + base, off, count, v);
        }
        if (T.p) {
            const u2v h = aw_load4(T.p + base, off, count), l = aw_load4((const uint16_t*)T.low + base, off, count);
            f4v x;
#pragma unroll
            for (int c = 0; c < 4; ++c) x[c] = aw_join((uint16_t)aw_half(h, c), (int16_t)aw_half(l, c));
            aw_store4(T.x + base, off, count, x);
        }
    }
}

// At most 2^40 elements, and n * row_len < 2^62 so that one multiply-high finds an element's row.
bool aw_shape(long long rows, int row_len, long long& n) {
    if (rows < 0 || row_len < 1 || rows > (1ll << 40) / row_len || rows > (1ll << 62) / row_len / row_len) return false;
    n = rows * row_len;
    return true;
}
AwDivisor aw_divisor(int len) {
    if (len < 2) return AwDivisor{0, (uint32_t)len, 0};
    return AwDivisor{~0ull / (unsigned long long)len + 1ull, (uint32_t)len, ~0u / (uint32_t)len + 1u};
}

// Gives the tensors of a launch their workgroups; false if the launch would need 2^32 threads (a grid's size is kept in 32 bits).
template <class Args, class Size>
bool aw_plan(Args& a, int count, int chunk, Size elements, uint32_t& blocks) {
    long long b = 0;
    a.count = count;
    for (int k = 0; k < count; ++k) {
        a.block_begin[k] = (uint32_t)b;
        b += (elements(k) + chunk - 1) / chunk;
        if (b * AW_THREADS >= (1ll << 32)) return false;
    }
    a.block_begin[count] = (uint32_t)b;
    blocks = (uint32_t)b;
    return true;
}

// Gradients that are column ranges of one matrix, as the rasterizer's colour gradients are for f_dc and f_rest (3 and 45 of 48
// floats), share cache lines: one after the other, the narrow one would fetch nearly the whole matrix again (192-byte rows, 128-byte
// lines: 384 MB for 36 MB at 3 M Gaussians).  Their workgroups alternate instead, in the ratio of their sizes, so that
// a row's lines are fetched once and found in the cache by the other.
bool aw_siblings(const AwTensor& x, const AwTensor& y, int size) {
    if (!x.n || !x.rows.len || !y.rows.len || x.g_row_stride != y.g_row_stride || x.n / x.rows.len != y.n / y.rows.len) return false;
    const long long apart = ((long long)(uintptr_t)y.g - (long long)(uintptr_t)x.g) / size;
    return apart < x.g_row_stride && -apart < x.g_row_stride;
}
void aw_pair(AwArgs& a, int k, int chunk) {          // tensors k and k + 1: their workgroups become k's
    if (a.t[k].n > a.t[k + 1].n) { const AwTensor t = a.t[k]; a.t[k] = a.t[k + 1]; a.t[k + 1] = t; }
    AwTensor& x = a.t[k];
    x.blocks = (uint32_t)((x.n + chunk - 1) / chunk);
    x.every = (uint32_t)((a.t[k + 1].n + chunk - 1) / chunk) / x.blocks;
    a.block_begin[k + 1] = a.block_begin[k + 2];
}

}  // namespace

extern "C" int gs_adamw_block(void) { return GS_ADAMW_BLOCK; }

extern "C" int gs_adamw_step(int num_tensors, const GsAdamWTensor* tensors, int param_bf16, int state_bits,
                             int stochastic_rounding, const float* grad_norm, double max_norm, float* scalars, void* stream_) {
    GS_REQUIRE(num_tensors >= 0 && (num_tensors == 0 || tensors), "num_tensors %d, tensors %p", num_tensors, (const void*)tensors);
    GS_REQUIRE(state_bits == 8 || state_bits == 32, "state_bits %d is neither 8 nor 32", state_bits);
    GS_REQUIRE(!grad_norm || max_norm >= 0.0, "max_norm must not be negative");
    GS_REQUIRE(((uintptr_t)scalars & 15) == 0, "scalars must be 16-byte aligned");
    const bool q8 = state_bits == 8;
    long long threads = 0;
    for (int k = 0; k < num_tensors; ++k) {
        const GsAdamWTensor& s = tensors[k];
        long long n;
        GS_REQUIRE(aw_shape(s.rows, s.row_len, n), "tensor %d: bad shape %lld x %d", k, s.rows, s.row_len);
        // of the launch that tensor k is in: refused before the first launch, so that a refused call changes nothing
        threads = (k % AW_MAX_TENSORS ? threads : 0) + (n + aw_step_chunk(q8) - 1) / aw_step_chunk(q8) * AW_THREADS;
        GS_REQUIRE(threads < (1ll << 32), "tensor %d: too many workgroups", k);
        GS_REQUIRE(n == 0 || (s.param && s.grad && s.exp_avg && s.exp_avg_sq), "tensor %d: null pointer", k);
        GS_REQUIRE(n == 0 || !param_bf16 || s.param_low, "tensor %d: bf16 parameters need param_low", k);
        GS_REQUIRE(s.grad_row_stride == 0 || s.grad_row_stride >= s.row_len, "tensor %d: grad_row_stride %lld < row_len %d", k,
                   s.grad_row_stride, s.row_len);
        GS_REQUIRE(s.beta1 >= 0.0 && s.beta1 < 1.0 && s.beta2 >= 0.0 && s.beta2 < 1.0, "tensor %d: betas outside [0,1)", k);
        GS_REQUIRE(s.eps >= 0.0, "tensor %d: negative eps", k);
        GS_REQUIRE((s.step_dev != nullptr) == (scalars != nullptr), "tensor %d: a count on the device needs scalars, and all tensors of a call one", k);
        GS_REQUIRE(s.step_dev || s.step >= 1, "tensor %d: step must be >= 1 (the count after this update)", k);
        GS_REQUIRE(s.step_dev || !s.lr_dev, "tensor %d: lr on the device needs its count there too", k);
        const uintptr_t al = q8 ? ((uintptr_t)s.exp_avg & 1) | ((uintptr_t)s.exp_avg_sq & 7) : ((uintptr_t)s.exp_avg | (uintptr_t)s.exp_avg_sq) & 3;
        GS_REQUIRE(al == 0 && (((uintptr_t)s.param | (uintptr_t)s.grad) & (param_bf16 ? 1 : 3)) == 0 && ((uintptr_t)s.param_low & 1) == 0,
                   "tensor %d: misaligned pointer", k);
    }
    for (int first = 0; first < num_tensors; first += AW_MAX_TENSORS) {
        const int count = num_tensors - first < AW_MAX_TENSORS ? num_tensors - first : AW_MAX_TENSORS;
        AwArgs a{};
        AwScalarArgs sc{};
        for (int k = 0; k < count; ++k) {
            const GsAdamWTensor& s = tensors[first + k];
            AwTensor& d = a.t[k];
            d.p = s.param; d.g = s.grad; d.low = param_bf16 ? s.param_low : nullptr; d.m = s.exp_avg; d.v = s.exp_avg_sq;
            d.n = s.rows * s.row_len;
            d.g_row_stride = s.grad_row_stride ? s.grad_row_stride : s.row_len;
            d.rows = aw_divisor(d.g_row_stride == s.row_len ? 0 : s.row_len);
            // torch/optim/adam.py: Python doubles, rounded to fp32 when they meet the tensor
            const double root = sqrt(1.0 - pow(s.beta2, (double)s.step));
            d.neg_step = (float)(-(s.lr / (1.0 - pow(s.beta1, (double)s.step))));
            d.decay = (float)(1.0 - s.lr * s.weight_decay);
            d.bc2 = (float)(q8 ? 1.0 / root : root);
            d.beta1 = (float)s.beta1; d.one_minus_beta1 = (float)(1.0 - s.beta1);
            d.beta2 = (float)s.beta2; d.one_minus_beta2 = (float)(1.0 - s.beta2);
            d.eps = (float)s.eps;
            const uint32_t seed = aw_mix(s.seed + 0x9E3779B9u * (s.index + 1u));
            d.key = aw_mix(seed ^ (uint32_t)s.step);
            d.slot = k;
            sc.t[k] = AwScalarTensor{s.step_dev, s.lr_dev, s.lr, s.beta1, s.beta2, s.weight_decay, seed, 0};
        }
        a.stochastic = stochastic_rounding;
        a.grad_norm = grad_norm;
        a.max_norm = (float)max_norm;
        if (scalars) {
            sc.count = count;
            sc.reciprocal = q8;
            sc.out = (float4*)scalars + first;
            a.scalars = sc.out;
            hipLaunchKernelGGL(adamw_scalars_kernel, dim3(1), dim3(64), 0, (hipStream_t)stream_, sc);
            GS_CHECK_LAUNCH("adamw_scalars");
        }
        uint32_t blocks = 0;
        GS_REQUIRE(aw_plan(a, count, aw_step_chunk(q8), [&](int k) { return a.t[k].n; }, blocks), "too many workgroups");
        if (blocks == 0) continue;
        for (int k = 0; k + 1 < count; ++k)
            if (aw_siblings(a.t[k], a.t[k + 1], param_bf16 ? 2 : 4)) { aw_pair(a, k, aw_step_chunk(q8)); ++k; }
        void (*kernel)(AwArgs) = param_bf16 ? (q8 ? adamw_kernel<true, true> : adamw_kernel<true, false>)
                                            : (q8 ? adamw_kernel<false, true> : adamw_kernel<false, false>);
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(AW_THREADS), 0, (hipStream_t)stream_, a);
        GS_CHECK_LAUNCH("adamw");
    }
    return GS_OK;
}

static_assert(sizeof(NrmArgs) <= 4096, "kernel arguments");

// One row where the rows follow each other without a gap.
static NrmTensor nrm_tensor(const GsGradTensor& s) {
    const bool one = s.row_stride == 0 || s.row_stride == s.row_len;
    const long long row_len = one ? s.rows * s.row_len : s.row_len, per_row = (row_len + 3) / 4;
    return NrmTensor{s.grad, one ? per_row : s.rows * per_row, s.row_stride, row_len, aw_divisor(one ? 0 : (int)per_row), s.bf16};
}
static long long nrm_blocks(const GsGradTensor& s) { return (nrm_tensor(s).groups + NRM_GROUPS - 1) / NRM_GROUPS; }

// Takes tensor k, and with it those after it that continue its rows: neighbouring column ranges of one matrix are read as one (f_dc
// and f_rest of the rasterizer's colour gradient: 3 + 45 of 48 floats, and no line is fetched twice).  Returns how many it took.
static int nrm_take(int num_tensors, const GsGradTensor* tensors, int k, GsGradTensor& out) {
    out = tensors[k];
    int taken = 1;
    for (; k + taken < num_tensors; ++taken) {
        const GsGradTensor& s = tensors[k + taken];
        const long long size = out.bf16 ? 2 : 4;
        if (!out.rows || out.row_stride <= out.row_len || s.rows != out.rows || s.row_stride != out.row_stride || !s.bf16 != !out.bf16 ||
            (uintptr_t)s.grad != (uintptr_t)out.grad + (uintptr_t)(out.row_len * size) || (long long)out.row_len + s.row_len > out.row_stride ||
            (long long)out.row_len + s.row_len > 0x7FFFFFFFll) break;
        out.row_len += s.row_len;
    }
    return taken;
}

extern "C" size_t gs_grad_norm_workspace_bytes(int num_tensors, const GsGradTensor* tensors) {
    size_t blocks = 0;
    for (int k = 0; k < num_tensors; ++k) blocks += (size_t)nrm_blocks(tensors[k]);
    return blocks * sizeof(double);
}

extern "C" int gs_grad_norm(int num_tensors, const GsGradTensor* tensors, float* norm, void* workspace,
                            size_t workspace_bytes, void* stream_) {
    GS_REQUIRE(num_tensors >= 0 && (num_tensors == 0 || tensors) && norm, "bad arguments");
    long long total = 0;
    for (int k = 0; k < num_tensors; ++k) {
        const GsGradTensor& s = tensors[k];
        long long n;
        GS_REQUIRE(aw_shape(s.rows, s.row_len, n), "tensor %d: bad shape %lld x %d", k, s.rows, s.row_len);
        GS_REQUIRE(n == 0 || s.grad, "tensor %d: null pointer", k);
        GS_REQUIRE(s.row_stride == 0 || s.row_stride >= s.row_len, "tensor %d: row_stride %lld < row_len %d", k, s.row_stride, s.row_len);
        GS_REQUIRE(((uintptr_t)s.grad & (s.bf16 ? 1 : 3)) == 0, "tensor %d: misaligned pointer", k);
        total += nrm_blocks(s);
    }
    GS_REQUIRE(workspace_bytes >= (size_t)total * sizeof(double) && (total == 0 || workspace), "workspace too small");
    GS_REQUIRE(((uintptr_t)workspace & 7) == 0, "workspace must be 8-byte aligned");
    long long done = 0;
    for (int next = 0; next < num_tensors;) {
        int count = 0;
        NrmArgs a{};
        for (; next < num_tensors && count < NRM_MAX_TENSORS; ++count) {
            GsGradTensor s;
            next += nrm_take(num_tensors, tensors, next, s);
            a.t[count] = nrm_tensor(s);
        }
        a.partial = (double*)workspace + done;
        uint32_t blocks = 0;
        GS_REQUIRE(aw_plan(a, count, NRM_GROUPS, [&](int k) { return a.t[k].groups; }, blocks), "too many workgroups");
        if (blocks == 0) continue;
        hipLaunchKernelGGL(grad_norm_partial_kernel, dim3(blocks), dim3(AW_THREADS), 0, (hipStream_t)stream_, a);
        GS_CHECK_LAUNCH("grad_norm_partial");
        done += blocks;
    }
    hipLaunchKernelGGL(grad_norm_final_kernel, dim3(1), dim3(NRM_FINAL_THREADS), 0, (hipStream_t)stream_, done,
                       (const double*)workspace, norm);
    GS_CHECK_LAUNCH("grad_norm_final");
    return GS_OK;
}

extern "C" int gs_adamw_gather_rows(int num_tensors, const GsAdamWRows* tensors, int state_bits, long long src_rows,
                                    long long dst_rows, const int64_t* index, void* stream_) {
    GS_REQUIRE(num_tensors >= 0 && (num_tensors == 0 || tensors), "bad arguments");
    GS_REQUIRE(state_bits == 8 || state_bits == 32, "state_bits %d is neither 8 nor 32", state_bits);
    GS_REQUIRE(src_rows >= 0 && dst_rows >= 0 && (dst_rows == 0 || index), "rows %lld -> %lld, index %p", src_rows, dst_rows, (const void*)index);
    GS_REQUIRE(((uintptr_t)index & 7) == 0, "index must be 8-byte aligned");
    const bool q8 = state_bits == 8;
    for (int first = 0; first < num_tensors; first += AW_MAX_TENSORS) {
        const int count = num_tensors - first < AW_MAX_TENSORS ? num_tensors - first : AW_MAX_TENSORS;
        RowArgs a{};
        a.src_rows = src_rows;
        a.index = index;
        for (int k = 0; k < count; ++k) {
            const GsAdamWRows& s = tensors[first + k];
            long long n_src, n_dst;
            GS_REQUIRE(aw_shape(src_rows, s.row_len, n_src) && aw_shape(dst_rows, s.row_len, n_dst), "tensor %d: bad row_len %d", first + k, s.row_len);
            GS_REQUIRE((n_src == 0 || (s.src_exp_avg && s.src_exp_avg_sq)) && (n_dst == 0 || (s.dst_exp_avg && s.dst_exp_avg_sq)),
                       "tensor %d: null pointer", first + k);
            GS_REQUIRE(n_src == 0 || n_dst == 0 || !s.dst_param_low == !s.src_param_low, "tensor %d: param_low of one side only", first + k);
            const uintptr_t am = (uintptr_t)s.src_exp_avg | (uintptr_t)s.dst_exp_avg, av = (uintptr_t)s.src_exp_avg_sq | (uintptr_t)s.dst_exp_avg_sq;
            GS_REQUIRE((am & (q8 ? 1 : 3)) == 0 && (av & (q8 ? 7 : 3)) == 0 && (((uintptr_t)s.src_param_low | (uintptr_t)s.dst_param_low) & 1) == 0,
                       "tensor %d: misaligned pointer", first + k);
            a.t[k] = RowTensor{s.src_exp_avg, s.src_exp_avg_sq, s.src_param_low, s.dst_exp_avg, s.dst_exp_avg_sq, s.dst_param_low,
                               n_dst, aw_divisor(s.row_len)};
        }
        uint32_t blocks = 0;
        GS_REQUIRE(aw_plan(a, count, AW_CHUNK, [&](int k) { return a.t[k].n; }, blocks), "too many workgroups");
        if (blocks == 0) continue;
        if (q8) hipLaunchKernelGGL((adamw_rows_kernel<true>), dim3(blocks), dim3(AW_THREADS), 0, (hipStream_t)stream_, a);
        else hipLaunchKernelGGL((adamw_rows_kernel<false>), dim3(blocks), dim3(AW_THREADS), 0, (hipStream_t)stream_, a);
        GS_CHECK_LAUNCH("adamw_rows");
    }
    return GS_OK;
}

extern "C" int gs_adamw_unpack(int num_tensors, const GsAdamWUnpack* tensors, void* stream_) {
    GS_REQUIRE(num_tensors >= 0 && (num_tensors == 0 || tensors), "bad arguments");
    for (int first = 0; first < num_tensors; first += AW_MAX_TENSORS) {
        const int count = num_tensors - first < AW_MAX_TENSORS ? num_tensors - first : AW_MAX_TENSORS;
        UnpackArgs a{};
        for (int k = 0; k < count; ++k) {
            const GsAdamWUnpack& s = tensors[first + k];
            GS_REQUIRE(s.numel >= 0 && s.numel < (1ll << 40), "tensor %d: bad size %lld", first + k, s.numel);
            GS_REQUIRE(!s.codes || (s.scales && s.exp_avg && s.exp_avg_sq), "tensor %d: codes need scales, exp_avg and exp_avg_sq", first + k);
            GS_REQUIRE(!s.param_bf16 || (s.param_low && s.param), "tensor %d: param_bf16 needs param_low and param", first + k);
            GS_REQUIRE((((uintptr_t)s.codes | (uintptr_t)s.param_bf16 | (uintptr_t)s.param_low) & 1) == 0 && ((uintptr_t)s.scales & 7) == 0 &&
                       (((uintptr_t)s.exp_avg | (uintptr_t)s.exp_avg_sq | (uintptr_t)s.param) & 3) == 0, "tensor %d: misaligned pointer", first + k);
            a.t[k] = UnpackTensor{(const uint16_t*)s.codes, (const float2*)s.scales, (const uint16_t*)s.param_bf16, s.param_low,
                                  s.exp_avg, s.exp_avg_sq, s.param, s.codes || s.param_bf16 ? s.numel : 0};
        }
        uint32_t blocks = 0;
        GS_REQUIRE(aw_plan(a, count, AW_CHUNK, [&](int k) { return a.t[k].n; }, blocks), "too many workgroups");
        if (blocks == 0) continue;
        hipLaunchKernelGGL(adamw_unpack_kernel, dim3(blocks), dim3(AW_THREADS), 0, (hipStream_t)stream_, a);
        GS_CHECK_LAUNCH("adamw_unpack");
    }
    return GS_OK;
}
