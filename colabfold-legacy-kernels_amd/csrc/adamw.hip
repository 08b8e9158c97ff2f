// One AdamW step over many tensors at once for gfx950, with states in 32 or in 8 bits.
//
//   g = grad * grad_scale;  m = b1*m + (1 - b1)*g;  v = b2*v + (1 - b2)*g*g
//   p = p*(1 - lr*decay) - lr/(1 - b1^t) * m / (sqrt(v)/sqrt(1 - b2^t) + eps);  copy = round(p)
//
// p is float32 (the master weights); copy, where given, is the bf16 or f16 working copy that the
// other kernels read, written in the same pass. Every operation on m and v is rounded once, in the
// order above (this file is compiled without contraction), so the states do not depend on how a
// tensor is cut.
//
// 8-bit states: a block of 256 elements of a tensor has two float32 scales, its largest |m| and its
// largest v, and codes relative to them, spaced closer for small values:
//   m = sign(c) * (c/127)^2 * scale_m,  v = (c/255)^4 * scale_v
//   c_m = sign(m) * rint(127 * sqrt(|m| / scale_m)),  c_v = rint(255 * (v / scale_v)^(1/4))
// Rounding to 8 bits is the point of this form (4.06 bytes an element and step instead of 16, at
// relative steps of 1.6% near a block's largest value). Two choices bound what it does to the
// weights: a v above zero keeps a code of at least 1, so no update divides by a v that was rounded
// away, and the scales are exact, so a block whose gradients all shrink follows them exactly. A
// block with an infinite or NaN state gets NaN scales: that cannot be held in codes.
//
// HBM-bound: p, grad, states and copy are read and written once, 28 bytes an element with 32-bit
// states and float32 gradients, 16 with 8-bit ones. A table in device memory lists the chunks of
// all tensors, so a step is one launch however many tensors there are.
#include <cmath>
#include <cstring>
#include <exception>
#include <vector>

#include "rows.hpp"

namespace clk {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 256;  // elements that share two scales: one wave, four elements a lane

// A run of at most one chunk of elements of one tensor; 64 bytes, so a block finds all it needs
// with one scalar load.
struct Chunk {
    float* p;
    const void* g;
    void *m, *v;
    float* scales;
    void* copy;
    int64_t at;  // the chunk's place in the flat buffers of clk_adamw_states
    uint32_t n;
    uint16_t grad_type, copy_type;  // clk_dtype; copy_type 0: none
};
static_assert(sizeof(Chunk) == 64);

struct Step {
    float b1, omb1, b2, omb2, keep, step, inv_bias2, eps, grad_scale;
    float decay;          // weight decay, for `hyper`
    const float* hyper;   // lr, 1 - b1^t, 1 - b2^t, grad_scale in device memory, or null
};
__device__ __forceinline__ void read_hyper(Step& s) {
    if (!s.hyper) return;
    const float lr = s.hyper[0];
    s.keep = 1.f - lr * s.decay;
    s.step = lr / s.hyper[1];
    s.inv_bias2 = 1.f / sqrtf(s.hyper[2]);
    s.grad_scale = s.hyper[3];
}

// Four elements at any element alignment; `cnt` of them exist (the others are zero, and not
// stored).
typedef unsigned int u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));
template <typename TR>
__device__ __forceinline__ void load_half4(const void* p, uint32_t at, int cnt, float (&x)[4]) {
    using E = typename TR::elem;
    const E* e = static_cast<const E*>(p) + at;
    if (cnt >= 4) {
        const u32x2 raw = *reinterpret_cast<const u32x2_a2*>(e);
        E h[4];
        __builtin_memcpy(h, &raw, 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = TR::to_f(h[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = i < cnt ? TR::to_f(e[i]) : 0.f;
    }
}
__device__ __forceinline__ void load_float4(const float* p, uint32_t at, int cnt, float (&x)[4]) {
    if (cnt >= 4) {
        const f32x4 v = ld4f(p + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = v[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = i < cnt ? p[at + i] : 0.f;
    }
}
__device__ __forceinline__ void load_grad4(const Chunk& c, uint32_t at, int cnt, float (&x)[4]) {
    if (c.grad_type == CLK_F32) load_float4(static_cast<const float*>(c.g), at, cnt, x);
    else if (c.grad_type == CLK_BF16) load_half4<BF16>(c.g, at, cnt, x);
    else load_half4<F16>(c.g, at, cnt, x);
}
__device__ __forceinline__ void store_float4(float* p, uint32_t at, int cnt, const float (&x)[4]) {
    if (cnt >= 4) {
        *reinterpret_cast<f32x4_a4*>(p + at) = f32x4{x[0], x[1], x[2], x[3]};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < cnt) p[at + i] = x[i];
    }
}
template <typename TR>
__device__ __forceinline__ void store_half4(void* p, uint32_t at, int cnt, const float (&x)[4]) {
    using E = typename TR::elem;
    E* e = static_cast<E*>(p) + at;
    E h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = TR::from_f(x[i]);
    if (cnt >= 4) {
        u32x2 raw;
        __builtin_memcpy(&raw, h, 8);
        *reinterpret_cast<u32x2_a2*>(e) = raw;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < cnt) e[i] = h[i];
    }
}
__device__ __forceinline__ void store_copy4(const Chunk& c, uint32_t at, int cnt,
                                            const float (&x)[4]) {
    if (c.copy_type == CLK_BF16) store_half4<BF16>(c.copy, at, cnt, x);
    else if (c.copy_type == CLK_F16) store_half4<F16>(c.copy, at, cnt, x);
}
__device__ __forceinline__ uint32_t load_codes4(const void* p, uint32_t at, int cnt) {
    const uint8_t* e = static_cast<const uint8_t*>(p) + at;
    if (cnt >= 4) return *reinterpret_cast<const uint32_t*>(e);
    uint32_t q = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < cnt) q |= (uint32_t)e[i] << (8 * i);
    return q;
}
__device__ __forceinline__ void store_codes4(void* p, uint32_t at, int cnt, uint32_t q) {
    uint8_t* e = static_cast<uint8_t*>(p) + at;
    if (cnt >= 4) {
        *reinterpret_cast<uint32_t*>(e) = q;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < cnt) e[i] = (uint8_t)(q >> (8 * i));
    }
}

__device__ __forceinline__ void update(const Step& s, float grad, float& p, float& m, float& v) {
    const float g = grad * s.grad_scale;
    m = m * s.b1 + g * s.omb1;
    v = v * s.b2 + (g * s.omb2) * g;
    p = p * s.keep - m / (sqrtf(v) * s.inv_bias2 + s.eps) * s.step;
}

__device__ __forceinline__ int left(uint32_t n, uint32_t at) {
    return at < n ? (n - at < 4 ? (int)(n - at) : 4) : 0;
}

__global__ __launch_bounds__(kThreads) void adamw32_kernel(const Chunk* __restrict__ table,
                                                           Step s) {
    const Chunk c = table[blockIdx.x];
    read_hyper(s);
    float *m = static_cast<float*>(c.m), *v = static_cast<float*>(c.v);
    for (uint32_t at = 4 * threadIdx.x; at < c.n; at += 4 * kThreads) {
        const int cnt = left(c.n, at);
        float ps[4], gs[4], ms[4], vs[4];
        load_float4(c.p, at, cnt, ps);
        load_grad4(c, at, cnt, gs);
        load_float4(m, at, cnt, ms);
        load_float4(v, at, cnt, vs);
#pragma unroll
        for (int i = 0; i < 4; ++i) update(s, gs[i], ps[i], ms[i], vs[i]);
        store_float4(c.p, at, cnt, ps);
        store_float4(m, at, cnt, ms);
        store_float4(v, at, cnt, vs);
        if (c.copy_type) store_copy4(c, at, cnt, ps);
    }
}

// Largest of the 64 lanes' values, as whole numbers: those of non-negative floats are in the order
// of the floats, with infinity and then NaN above all.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    const auto step = [](u32x2 p) { return p[0] > p[1] ? p[0] : p[1]; };
    x = step(lane_pair<1>(__uint_as_float(x)));
    x = step(lane_pair<2>(__uint_as_float(x)));
    x = step(lane_pair<4>(__uint_as_float(x)));
    x = step(lane_pair<8>(__uint_as_float(x)));
    x = step(lane_pair<16>(__uint_as_float(x)));
    return step(lane_pair<32>(__uint_as_float(x)));
}

__device__ __forceinline__ void decode(uint32_t qm, uint32_t qv, float sm, float sv, float (&m)[4],
                                       float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float rm = (float)(int8_t)(qm >> (8 * i)) * (1.f / 127.f);
        const float rv = (float)((qv >> (8 * i)) & 255u) * (1.f / 255.f);
        m[i] = (rm * fabsf(rm)) * sm;
        v[i] = ((rv * rv) * (rv * rv)) * sv;
    }
}

constexpr uint32_t kInfBits = 0x7F800000u;

__global__ __launch_bounds__(kThreads) void adamw8_kernel(const Chunk* __restrict__ table,
                                                          Step s) {
    const Chunk c = table[blockIdx.x];
    read_hyper(s);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint32_t b = wave; b * kBlock < c.n; b += kThreads / 64) {
        const uint32_t at = b * kBlock + 4 * lane;
        const int cnt = left(c.n, at);
        float ps[4], gs[4], ms[4], vs[4];
        load_float4(c.p, at, cnt, ps);
        load_grad4(c, at, cnt, gs);
        decode(load_codes4(c.m, at, cnt), load_codes4(c.v, at, cnt), c.scales[2 * b],
               c.scales[2 * b + 1], ms, vs);
        uint32_t am = 0, av = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            update(s, gs[i], ps[i], ms[i], vs[i]);
            if (i < cnt) {
                am = max(am, __float_as_uint(fabsf(ms[i])));
                av = max(av, __float_as_uint(fabsf(vs[i])));
            }
        }
        am = wave_max(am);
        av = wave_max(av);
        const float sm = __uint_as_float(am), sv = __uint_as_float(av);
        const float om = am ? sm : 1.f, ov = av ? sv : 1.f;
        uint32_t qm = 0, qv = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = rintf(sqrtf(fabsf(ms[i]) / om) * 127.f);
            float q = rintf(sqrtf(sqrtf(vs[i] / ov)) * 255.f);
            if (vs[i] > 0.f) q = fmaxf(q, 1.f);
            qm |= ((uint32_t)(int)(ms[i] < 0.f ? -a : a) & 255u) << (8 * i);
            qv |= ((uint32_t)(int)q & 255u) << (8 * i);
        }
        if (am >= kInfBits) qm = 0;
        if (av >= kInfBits) qv = 0;
        store_float4(c.p, at, cnt, ps);
        store_codes4(c.m, at, cnt, qm);
        store_codes4(c.v, at, cnt, qv);
        if (lane == 0) {
            c.scales[2 * b] = am >= kInfBits ? __builtin_nanf("") : sm;
            c.scales[2 * b + 1] = av >= kInfBits ? __builtin_nanf("") : sv;
        }
        if (c.copy_type) store_copy4(c, at, cnt, ps);
    }
}

// The float32 states in flat buffers where every tensor begins at a multiple of 256 elements, with
// zeros up to the next one.
template <int BITS>
__global__ __launch_bounds__(kThreads) void adamw_states_kernel(const Chunk* __restrict__ table,
                                                                float* __restrict__ m,
                                                                float* __restrict__ v) {
    const Chunk c = table[blockIdx.x];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint32_t b = wave; b * kBlock < c.n; b += kThreads / 64) {
        const uint32_t at = b * kBlock + 4 * lane;
        const int cnt = left(c.n, at);
        float ms[4], vs[4];
        if (BITS == 8) {
            decode(load_codes4(c.m, at, cnt), load_codes4(c.v, at, cnt), c.scales[2 * b],
                   c.scales[2 * b + 1], ms, vs);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i >= cnt) ms[i] = vs[i] = 0.f;  // a NaN scale's as well
        } else {
            load_float4(static_cast<const float*>(c.m), at, cnt, ms);
            load_float4(static_cast<const float*>(c.v), at, cnt, vs);
        }
        *reinterpret_cast<f32x4*>(m + c.at + at) = f32x4{ms[0], ms[1], ms[2], ms[3]};
        *reinterpret_cast<f32x4*>(v + c.at + at) = f32x4{vs[0], vs[1], vs[2], vs[3]};
    }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------

// Elements a chunk: few enough that a small parameter set still fills the chip.
constexpr int64_t kSmallChunk = 1024, kLargeChunk = 4096;

struct Span {
    uintptr_t beg, end;
    bool written;
};

bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

clk_status check_tensor(const char* who, const clk_adamw_tensor& t, int64_t i, int bits) {
    if (t.numel < 0 || t.numel > ((int64_t)1 << 40))
        return fail(CLK_INVALID_ARGUMENT, "%s: tensor %lld has %lld elements", who, (long long)i,
                    (long long)t.numel);
    if (t.grad_dtype != CLK_F32 && t.grad_dtype != CLK_BF16 && t.grad_dtype != CLK_F16)
        return fail(CLK_INVALID_ARGUMENT, "%s: gradient %lld of type %s (f16, bf16, f32)", who,
                    (long long)i, dtype_name(t.grad_dtype));
    if (t.numel == 0) return CLK_OK;
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || (bits == 8 && !t.scales))
        return fail(CLK_INVALID_ARGUMENT, "%s: null pointer in tensor %lld", who, (long long)i);
    if (t.copy && t.copy_dtype != CLK_BF16 && t.copy_dtype != CLK_F16)
        return fail(CLK_INVALID_ARGUMENT, "%s: copy %lld of type %s (f16, bf16)", who,
                    (long long)i, dtype_name(t.copy_dtype));
    if (!aligned_to(t.param, 4) || !aligned_to(t.grad, elem_size(t.grad_dtype)) ||
        !aligned_to(t.exp_avg, 4) || !aligned_to(t.exp_avg_sq, 4) || !aligned_to(t.scales, 4) ||
        !aligned_to(t.copy, 2))
        return fail(CLK_INVALID_ARGUMENT,
                    "%s: tensor %lld is misaligned (elements; 4 bytes for 8-bit states)", who,
                    (long long)i);
    return CLK_OK;
}

// Every buffer that a step writes has to be apart from all others; gradients may be shared.
bool overlapping(std::vector<Span>& spans) {
    std::sort(spans.begin(), spans.end(),
              [](const Span& a, const Span& b) { return a.beg < b.beg; });
    uintptr_t any = 0, written = 0;
    for (const Span& s : spans) {
        if (s.beg < (s.written ? any : written)) return true;
        any = std::max(any, s.end);
        if (s.written) written = std::max(written, s.end);
    }
    return false;
}

clk_status build_table(const char* who, const clk_adamw_tensor* tensors, int64_t n, int bits,
                       void* table, size_t table_bytes, int64_t* chunks) {
    int64_t total = 0, large = 0, small = 0;
    std::vector<Span> spans;
    for (int64_t i = 0; i < n; ++i) {
        const clk_adamw_tensor& t = tensors[i];
        const clk_status s = check_tensor(who, t, i, bits);
        if (s != CLK_OK) return s;
        total += t.numel;
        large += up(t.numel, kLargeChunk);
        small += up(t.numel, kSmallChunk);
        const auto span = [&](const void* p, int64_t bytes, bool written) {
            const uintptr_t b = reinterpret_cast<uintptr_t>(p);
            if (p && bytes > 0) spans.push_back({b, b + (uintptr_t)bytes, written});
        };
        const int64_t state = t.numel * (bits / 8);
        span(t.param, t.numel * 4, true);
        span(t.grad, t.numel * (int64_t)elem_size(t.grad_dtype), false);
        span(t.exp_avg, state, true);
        span(t.exp_avg_sq, state, true);
        if (bits == 8) span(t.scales, up(t.numel, kBlock) * 8, true);
        span(t.copy, t.numel * 2, true);
    }
    if (overlapping(spans))
        return fail(CLK_INVALID_ARGUMENT,
                    "%s: tensors overlap (parameters, states, scales and copies are written)", who);
    const int64_t chunk = large < 2048 ? kSmallChunk : kLargeChunk;
    const int64_t count = chunk == kSmallChunk ? small : large;
    if (count >= (1 << 24))
        return fail(CLK_INVALID_ARGUMENT, "%s: %lld elements are too many", who, (long long)total);
    *chunks = count;
    if (!table) return ok();
    if (table_bytes < (size_t)count * sizeof(Chunk))
        return fail(CLK_INVALID_ARGUMENT, "%s: table %zu bytes, needs %zu", who, table_bytes,
                    (size_t)count * sizeof(Chunk));
    char* to = static_cast<char*>(table);
    int64_t base = 0;
    for (int64_t i = 0; i < n; ++i) {
        const clk_adamw_tensor& t = tensors[i];
        for (int64_t o = 0; o < t.numel; o += chunk) {
            Chunk c;
            c.p = t.param + o;
            c.g = static_cast<const char*>(t.grad) + o * (int64_t)elem_size(t.grad_dtype);
            c.m = static_cast<char*>(t.exp_avg) + o * (bits / 8);
            c.v = static_cast<char*>(t.exp_avg_sq) + o * (bits / 8);
            c.scales = bits == 8 ? t.scales + 2 * (o / kBlock) : nullptr;
            c.copy = t.copy ? static_cast<char*>(t.copy) + 2 * o : nullptr;
            c.at = base + o;
            c.n = (uint32_t)std::min(chunk, t.numel - o);
            c.grad_type = (uint16_t)t.grad_dtype;
            c.copy_type = t.copy ? (uint16_t)t.copy_dtype : 0;
            std::memcpy(to, &c, sizeof(c));
            to += sizeof(c);
        }
        base += up(t.numel, kBlock) * kBlock;
    }
    return ok();
}

clk_status check_call(const char* who, const void* table, int64_t chunks, int bits) {
    if (bits != 8 && bits != 32)
        return fail(CLK_INVALID_ARGUMENT, "%s: states of %d bits (8, 32)", who, bits);
    if (chunks < 0 || chunks >= (1 << 24))
        return fail(CLK_INVALID_ARGUMENT, "%s: %lld chunks", who, (long long)chunks);
    if (chunks > 0 && (!table || !aligned16(table)))
        return fail(CLK_INVALID_ARGUMENT, "%s: the table must be a 16-byte aligned device pointer",
                    who);
    return CLK_OK;
}

}  // namespace
}  // namespace clk

using namespace clk;

extern "C" clk_status clk_adamw_table(const clk_adamw_tensor* tensors, int64_t n, int state_bits,
                                      void* table, size_t table_bytes, int64_t* chunks) {
    const char* who = "adamw_table";
    if (state_bits != 8 && state_bits != 32)
        return fail(CLK_INVALID_ARGUMENT, "%s: states of %d bits (8, 32)", who, state_bits);
    if (n < 0 || (n > 0 && !tensors) || !chunks)
        return fail(CLK_INVALID_ARGUMENT, "%s: null pointer or negative count", who);
    try {
        return build_table(who, tensors, n, state_bits, table, table_bytes, chunks);
    } catch (const std::exception&) {
        return fail(CLK_INTERNAL, "%s: out of host memory", who);
    }
}

extern "C" clk_status clk_adamw_step(hipStream_t stream, const void* table, int64_t chunks,
                                     int state_bits, int64_t step, double lr, double beta1,
                                     double beta2, double eps, double weight_decay,
                                     double grad_scale, const float* hyper) {
    const char* who = "adamw";
    const clk_status s = check_call(who, table, chunks, state_bits);
    if (s != CLK_OK) return s;
    if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0))
        return fail(CLK_INVALID_ARGUMENT, "%s: betas must lie in [0, 1)", who);
    if (!((float)eps > 0.f) || !std::isfinite(eps))
        return fail(CLK_INVALID_ARGUMENT, "%s: eps must be positive and finite", who);
    if (!std::isfinite(weight_decay))
        return fail(CLK_INVALID_ARGUMENT, "%s: weight_decay must be finite", who);
    if (hyper) {
        if (!aligned_to(hyper, 4))
            return fail(CLK_INVALID_ARGUMENT, "%s: hyper is misaligned", who);
    } else {
        if (step < 1) return fail(CLK_INVALID_ARGUMENT, "%s: step counts from 1", who);
        if (!std::isfinite(lr) || !std::isfinite(grad_scale))
            return fail(CLK_INVALID_ARGUMENT, "%s: lr and grad_scale must be finite", who);
    }
    if (chunks == 0) return ok();
    const double bias1 = 1.0 - std::pow(beta1, (double)step);
    const double bias2 = 1.0 - std::pow(beta2, (double)step);
    Step k = {};
    k.b1 = (float)beta1;
    k.omb1 = (float)(1.0 - beta1);
    k.b2 = (float)beta2;
    k.omb2 = (float)(1.0 - beta2);
    k.eps = (float)eps;
    k.decay = (float)weight_decay;
    k.hyper = hyper;
    if (!hyper) {
        k.keep = (float)(1.0 - lr * weight_decay);
        k.step = (float)(lr / bias1);
        k.inv_bias2 = (float)(1.0 / std::sqrt(bias2));
        k.grad_scale = (float)grad_scale;
    }
    const Chunk* t = static_cast<const Chunk*>(table);
    KernelTimer timer("adamw", stream);
    if (state_bits == 8) adamw8_kernel<<<(int)chunks, kThreads, 0, stream>>>(t, k);
    else adamw32_kernel<<<(int)chunks, kThreads, 0, stream>>>(t, k);
    return check_launch(who);
}

extern "C" clk_status clk_adamw_states(hipStream_t stream, const void* table, int64_t chunks,
                                       int state_bits, float* exp_avg, float* exp_avg_sq) {
    const char* who = "adamw_states";
    const clk_status s = check_call(who, table, chunks, state_bits);
    if (s != CLK_OK) return s;
    if (chunks == 0) return ok();
    if (!exp_avg || !exp_avg_sq || !aligned16(exp_avg) || !aligned16(exp_avg_sq))
        return fail(CLK_INVALID_ARGUMENT, "%s: outputs must be 16-byte aligned", who);
    const Chunk* t = static_cast<const Chunk*>(table);
    KernelTimer timer("adamw_states", stream);
    if (state_bits == 8)
        adamw_states_kernel<8><<<(int)chunks, kThreads, 0, stream>>>(t, exp_avg, exp_avg_sq);
    else
        adamw_states_kernel<32><<<(int)chunks, kThreads, 0, stream>>>(t, exp_avg, exp_avg_sq);
    return check_launch(who);
}
