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
// bf16 parameters: p holds the fp32 value rounded to bf16 (halves away from zero), a 16-bit remainder in units of the
// fp32's last place holds the rest, so value = (bits(p) << 16) + remainder.  It costs what an fp32 parameter costs, and a
// parameter that was overwritten from outside is off by no more than half a bf16 step.
#include "gsplat_common.h"
#include "../../include/gsplat.h"
#include <math.h>
#pragma clang fp contract(off)

namespace {

constexpr int AW_THREADS = 256;
constexpr int AW_MAX_TENSORS = 32;      // tensors per launch: the table travels in the kernel arguments (4 KB)
constexpr int AW_CHUNK = 2048;          // elements per workgroup, a multiple of AW_THREADS and of GS_ADAMW_BLOCK

struct AwTensor {
    void* p;
    const void* g;
    int16_t* low;
    void* m;                  // fp32 moments, or the code pairs
    float* v;                 // fp32 moments, or the scale pairs
    long long n;
    long long g_row_stride;
    unsigned long long magic; // floor(2^64 / row_len) + 1: e / row_len == umul64hi(e, magic) while n * row_len < 2^64; 0: row_len 1
    int row_len;              // 0: contiguous gradient
    float neg_step, decay, bc2;   // -(lr / (1 - beta1^t)), 1 - lr wd, sqrt(1 - beta2^t) (8 bits: its reciprocal)
    float beta1, beta2, one_minus_beta1, one_minus_beta2, eps;
    uint32_t key;
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

__device__ __forceinline__ float aw_join(uint16_t high, int16_t low) {
    return __uint_as_float(((uint32_t)high << 16) + (uint32_t)(int32_t)low);
}
__device__ __forceinline__ void aw_split(float x, uint16_t& high, int16_t& low) {
    const uint32_t b = x != x ? 0x7FC00000u : __float_as_uint(x);
    high = (uint16_t)((b + 0x8000u) >> 16);
    low = (int16_t)(b & 0xFFFFu);
}
__device__ __forceinline__ float aw_bf16(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }

__device__ __forceinline__ float aw_level_m(uint32_t code, float scale) {
    const uint32_t c = code & 127u;
    const float f = __uint_as_float(0x3F800000u - ((127u - c) << 20)) * scale;
    return c == 0 ? 0.0f : (code & 128u) ? -f : f;
}
__device__ __forceinline__ float aw_level_u(uint32_t code, float scale) {
    const float f = __uint_as_float(0x3F800000u - ((255u - code) << 19)) * scale;
    return code == 0 ? 0.0f : f;
}
// x = the value over its block's scale, at most 1; r = 16 random bits, 32768 rounds to nearest
__device__ __forceinline__ uint32_t aw_code_m(float x, bool negative, uint32_t r) {
    int c = 127 + ((int)(__float_as_uint(x) + r * 16u - 0x3F800000u) >> 20);
    if (c < 1) c = x * (65536.0f / (1.25f * 0x1p-16f)) > (float)r ? 1 : 0;
    return (uint32_t)c + (negative && c > 0 ? 128u : 0u);
}
__device__ __forceinline__ uint32_t aw_code_u(float x, bool zero, uint32_t r) {
    const int c = 255 + ((int)(__float_as_uint(x) + r * 8u - 0x3F800000u) >> 19);
    return zero ? 0u : (uint32_t)(c < 1 ? 1 : c);
}
// the scale to keep and the factor that takes values to 0..1 (subnormal maxima count as zero: their reciprocal overflows)
__device__ __forceinline__ float aw_scale(uint32_t max_bits, float& inverse) {
    if (max_bits < 0x00800000u) { inverse = 0.0f; return 0.0f; }
    inverse = __fdiv_rn(1.0f, __uint_as_float(max_bits));
    return __uint_as_float(max_bits);
}
__device__ __forceinline__ uint32_t aw_wave_max(uint32_t x) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const uint32_t y = (uint32_t)__shfl_xor((int)x, d, 64);
        x = x > y ? x : y;
    }
    return x;
}

template <bool BF16, bool Q8>
__global__ __launch_bounds__(AW_THREADS) void adamw_kernel(const AwArgs a) {
    int ti = 0;
    for (int k = 1; k < a.count; ++k) ti += blockIdx.x >= a.block_begin[k] ? 1 : 0;
    const AwTensor& T = a.t[ti];
    float neg_step = T.neg_step, decay = T.decay, bc2 = T.bc2;
    uint32_t key = T.key;
    if (a.scalars) {
        const float4 s = a.scalars[ti];
        neg_step = s.x; decay = s.y; bc2 = s.z; key = __float_as_uint(s.w);
    }
    for (int i = 0; i < AW_CHUNK; i += AW_THREADS) {
        const long long e = (long long)(blockIdx.x - a.block_begin[ti]) * AW_CHUNK + i + threadIdx.x;
        const bool in = e < T.n;
        float p = 0.0f, g = 0.0f, m = 0.0f, v = 0.0f;
        if (in) {
            long long ge = e;
            if (T.row_len) {
                const long long row = T.magic ? (long long)__umul64hi((unsigned long long)e, T.magic) : e;
                ge = row * T.g_row_stride + (e - row * T.row_len);
            }
            if (BF16) {
                p = aw_join(((const uint16_t*)T.p)[e], T.low[e]);
                g = aw_bf16(((const uint16_t*)T.g)[ge]);
            } else {
                p = ((const float*)T.p)[e];
                g = ((const float*)T.g)[ge];
            }
            if (Q8) {
                const uint32_t codes = ((const uint16_t*)T.m)[e];
                const float2 s = ((const float2*)T.v)[e / GS_ADAMW_BLOCK];
                m = aw_level_m(codes & 255u, s.x);
                const float u = aw_level_u(codes >> 8, s.y);
                v = u * u;
            } else {
                m = ((const float*)T.m)[e];
                v = T.v[e];
            }
            if (a.grad_norm) g = g * aw_coef(a.grad_norm, a.max_norm);
        }
        float u;
        p = p * decay;
        if (Q8) {
            m = m * T.beta1 + g * T.one_minus_beta1;
            v = v * T.beta2 + (g * g) * T.one_minus_beta2;
            u = sqrtf(v);
            p = p + neg_step * __fdiv_rn(m, u * bc2 + T.eps);
        } else {
            m = __fmaf_rn(T.one_minus_beta1, g - m, m);
            v = __fmaf_rn(T.one_minus_beta2, g * g, v * T.beta2);
            u = sqrtf(v);
            p = __fmaf_rn(neg_step, __fdiv_rn(m, __fdiv_rn(u, bc2) + T.eps), p);
        }
        if (Q8) {
            // one wave holds one block of 64; lanes past the end bring zeros
            float im, iu;
            const float sm = aw_scale(aw_wave_max(in ? __float_as_uint(m) & 0x7FFFFFFFu : 0u), im);
            const float su = aw_scale(aw_wave_max(in ? __float_as_uint(u) : 0u), iu);
            uint32_t r = 0x80008000u;
            if (a.stochastic) r = aw_mix((uint32_t)e + key + (uint32_t)((unsigned long long)e >> 32) * 0x3C6EF373u);
            const uint32_t cm = aw_code_m(fminf(fabsf(m) * im, 1.0f), m < 0.0f, r & 0xFFFFu);
            const uint32_t cu = aw_code_u(fminf(u * iu, 1.0f), u == 0.0f || su == 0.0f, r >> 16);
            if (in) {
                ((uint16_t*)T.m)[e] = (uint16_t)(cm | cu << 8);
                if ((threadIdx.x & 63) == 0) ((float2*)T.v)[e / GS_ADAMW_BLOCK] = make_float2(sm, su);
            }
        }
        if (in) {
            if (BF16) {
                uint16_t high; int16_t low;
                aw_split(p, high, low);
                ((uint16_t*)T.p)[e] = high;
                T.low[e] = low;
            } else {
                ((float*)T.p)[e] = p;
            }
            if (!Q8) { ((float*)T.m)[e] = m; T.v[e] = v; }
        }
    }
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
constexpr int NRM_MAX_TENSORS = 64;
constexpr int NRM_CHUNK = 8192;         // elements per workgroup and partial sum
struct NrmTensor { const void* g; long long n, row_stride; unsigned long long magic; int row_len; int bf16; };
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

__global__ __launch_bounds__(AW_THREADS) void grad_norm_partial_kernel(const NrmArgs a) {
    __shared__ double lds[AW_THREADS / 64];
    int ti = 0;
    for (int k = 1; k < a.count; ++k) ti += blockIdx.x >= a.block_begin[k] ? 1 : 0;
    const NrmTensor& T = a.t[ti];
    const long long base = (long long)(blockIdx.x - a.block_begin[ti]) * NRM_CHUNK;
    double s = 0.0;
    for (int k = 0; k < NRM_CHUNK; k += AW_THREADS) {
        const long long e = base + k + threadIdx.x;
        if (e < T.n) {
            long long ge = e;
            if (T.row_len) {
                const long long row = T.magic ? (long long)__umul64hi((unsigned long long)e, T.magic) : e;
                ge = row * T.row_stride + (e - row * T.row_len);
            }
            const double x = T.bf16 ? (double)aw_bf16(((const uint16_t*)T.g)[ge]) : (double)((const float*)T.g)[ge];
            s = fma(x, x, s);
        }
    }
    s = nrm_block_sum(s, lds);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = s;
}

constexpr int NRM_FINAL_THREADS = 1024;
__global__ __launch_bounds__(NRM_FINAL_THREADS) void grad_norm_final_kernel(long long n, const double* partial, float* out) {
    __shared__ double lds[NRM_FINAL_THREADS / 64];
    double s = 0.0;
    for (long long k = threadIdx.x; k < n; k += NRM_FINAL_THREADS) s += partial[k];
    s = nrm_block_sum(s, lds);
    if (threadIdx.x == 0) *out = (float)sqrt(s);
}

// ---- rows of the states ---------------------------------------------------------------------------------------------
struct RowTensor {
    const void* src_m; const float* src_v; const int16_t* src_low;
    void* dst_m; float* dst_v; int16_t* dst_low;
    long long n;                          // elements of the new state
    unsigned long long magic;
    int row_len; int pad;
};
struct RowArgs { RowTensor t[AW_MAX_TENSORS]; uint32_t block_begin[AW_MAX_TENSORS + 1]; int count; long long src_rows; const int64_t* index; };

template <bool Q8>
__global__ __launch_bounds__(AW_THREADS) void adamw_rows_kernel(const RowArgs a) {
    int ti = 0;
    for (int k = 1; k < a.count; ++k) ti += blockIdx.x >= a.block_begin[k] ? 1 : 0;
    const RowTensor& T = a.t[ti];
    for (int i = 0; i < AW_CHUNK; i += AW_THREADS) {
        const long long e = (long long)(blockIdx.x - a.block_begin[ti]) * AW_CHUNK + i + threadIdx.x;
        const bool in = e < T.n;
        float m = 0.0f, v = 0.0f;             // Q8: v holds u
        int16_t low = 0;
        if (in) {
            const long long row = T.magic ? (long long)__umul64hi((unsigned long long)e, T.magic) : e;
            const long long src_row = a.index[row];
            if (src_row >= 0 && src_row < a.src_rows) {
                const long long s = src_row * T.row_len + (e - row * T.row_len);
                if (Q8) {
                    const uint32_t codes = ((const uint16_t*)T.src_m)[s];
                    const float2 sc = ((const float2*)T.src_v)[s / GS_ADAMW_BLOCK];
                    m = aw_level_m(codes & 255u, sc.x);
                    v = aw_level_u(codes >> 8, sc.y);
                } else {
                    m = ((const float*)T.src_m)[s];
                    v = T.src_v[s];
                }
                if (T.src_low) low = T.src_low[s];
            }
        }
        if (Q8) {
            float im, iu;
            const float sm = aw_scale(aw_wave_max(__float_as_uint(m) & 0x7FFFFFFFu), im);
            const float su = aw_scale(aw_wave_max(__float_as_uint(v)), iu);
            const uint32_t cm = aw_code_m(fminf(fabsf(m) * im, 1.0f), m < 0.0f, 32768u);
            const uint32_t cu = aw_code_u(fminf(v * iu, 1.0f), v == 0.0f || su == 0.0f, 32768u);
            if (in) {
                ((uint16_t*)T.dst_m)[e] = (uint16_t)(cm | cu << 8);
                if ((threadIdx.x & 63) == 0) ((float2*)T.dst_v)[e / GS_ADAMW_BLOCK] = make_float2(sm, su);
            }
        } else if (in) {
            ((float*)T.dst_m)[e] = m;
            T.dst_v[e] = v;
        }
        if (in && T.dst_low) T.dst_low[e] = low;
    }
}

// ---- what packed states and split parameters stand for --------------------------------------------------------------
struct UnpackTensor { const uint16_t* codes; const float2* scales; const uint16_t* p; const int16_t* low; float* m; float* v; float* x; long long n; };
struct UnpackArgs { UnpackTensor t[AW_MAX_TENSORS]; uint32_t block_begin[AW_MAX_TENSORS + 1]; int count; };

__global__ __launch_bounds__(AW_THREADS) void adamw_unpack_kernel(const UnpackArgs a) {
    int ti = 0;
    for (int k = 1; k < a.count; ++k) ti += blockIdx.x >= a.block_begin[k] ? 1 : 0;
    const UnpackTensor& T = a.t[ti];
    for (int i = 0; i < AW_CHUNK; i += AW_THREADS) {
        const long long e = (long long)(blockIdx.x - a.block_begin[ti]) * AW_CHUNK + i + threadIdx.x;
        if (e >= T.n) return;
        if (T.codes) {
            const uint32_t codes = T.codes[e];
            const float2 s = T.scales[e / GS_ADAMW_BLOCK];
            const float u = aw_level_u(codes >> 8, s.y);
            T.m[e] = aw_level_m(codes & 255u, s.x);
            T.v[e] = u * u;
        }
        if (T.p) T.x[e] = aw_join(T.p[e], T.low[e]);
    }
}

// At most 2^40 elements, and n * row_len < 2^62 so that one multiply-high finds an element's row.
bool aw_shape(long long rows, int row_len, long long& n) {
    if (rows < 0 || row_len < 1 || rows > (1ll << 40) / row_len || rows > (1ll << 62) / row_len / row_len) return false;
    n = rows * row_len;
    return true;
}
unsigned long long aw_magic(int row_len) { return row_len == 1 ? 0ull : ~0ull / (unsigned long long)row_len + 1ull; }

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

}  // namespace

extern "C" int gs_adamw_block(void) { return GS_ADAMW_BLOCK; }

extern "C" int gs_adamw_step(int num_tensors, const GsAdamWTensor* tensors, int param_bf16, int state_bits,
                             int stochastic_rounding, const float* grad_norm, double max_norm, float* scalars, void* stream_) {
    GS_REQUIRE(num_tensors >= 0 && (num_tensors == 0 || tensors), "num_tensors %d, tensors %p", num_tensors, (const void*)tensors);
    GS_REQUIRE(state_bits == 8 || state_bits == 32, "state_bits %d is neither 8 nor 32", state_bits);
    GS_REQUIRE(!grad_norm || max_norm >= 0.0, "max_norm must not be negative");
    GS_REQUIRE(((uintptr_t)scalars & 15) == 0, "scalars must be 16-byte aligned");
    const bool q8 = state_bits == 8;
    for (int k = 0; k < num_tensors; ++k) {
        const GsAdamWTensor& s = tensors[k];
        long long n;
        GS_REQUIRE(aw_shape(s.rows, s.row_len, n), "tensor %d: bad shape %lld x %d", k, s.rows, s.row_len);
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
            d.row_len = d.g_row_stride == s.row_len ? 0 : s.row_len;
            d.magic = aw_magic(s.row_len);
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
        GS_REQUIRE(aw_plan(a, count, AW_CHUNK, [&](int k) { return a.t[k].n; }, blocks), "too many workgroups");
        if (blocks == 0) continue;
        void (*kernel)(AwArgs) = param_bf16 ? (q8 ? adamw_kernel<true, true> : adamw_kernel<true, false>)
                                            : (q8 ? adamw_kernel<false, true> : adamw_kernel<false, false>);
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(AW_THREADS), 0, (hipStream_t)stream_, a);
        GS_CHECK_LAUNCH("adamw");
    }
    return GS_OK;
}

static long long nrm_blocks(const GsGradTensor& s) { return (s.rows * s.row_len + NRM_CHUNK - 1) / NRM_CHUNK; }

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
    for (int first = 0; first < num_tensors; first += NRM_MAX_TENSORS) {
        const int count = num_tensors - first < NRM_MAX_TENSORS ? num_tensors - first : NRM_MAX_TENSORS;
        NrmArgs a{};
        for (int k = 0; k < count; ++k) {
            const GsGradTensor& s = tensors[first + k];
            const long long stride = s.row_stride ? s.row_stride : s.row_len;
            a.t[k] = NrmTensor{s.grad, s.rows * s.row_len, stride, aw_magic(s.row_len), stride == s.row_len ? 0 : s.row_len, s.bf16};
        }
        a.partial = (double*)workspace + done;
        uint32_t blocks = 0;
        GS_REQUIRE(aw_plan(a, count, NRM_CHUNK, [&](int k) { return a.t[k].n; }, blocks), "too many workgroups");
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
                               n_dst, aw_magic(s.row_len), s.row_len, 0};
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
