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
// states and float32 gradients, 16 with 8-bit ones, 2 more with a copy. 14.6 M weights in 32 bits
// with copies take 82.8 us (5.3 TB/s), 87.8 M in 8 bits with bf16 gradients and copies 240 to 260
// (5.4 to 5.9 TB/s). A table in device memory lists the chunks of all tensors, so a step is one
// launch however many tensors there are.
#include <cmath>
#include <cstring>
#include <exception>
#include <vector>

#include "rows.hpp"

namespace clk {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 256;  // elements that share two scales: one wave, four elements a lane

// A run of at most one chunk of elements of one tensor.
struct alignas(16) Chunk {
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

// The block's chunk, all 64 bytes in one round of scalar loads (field by field the compiler loads
// each where it is first needed, one wait after the other).
__device__ __forceinline__ Chunk load_chunk(const Chunk* table) {
    typedef unsigned int u32x16 __attribute__((ext_vector_type(16), aligned(16)));
    const u32x16 raw = *reinterpret_cast<const u32x16*>(table + blockIdx.x);
    return __builtin_bit_cast(Chunk, raw);
}

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

// The pointers of a table come out of memory: said to be global, their accesses need no check for
// LDS (flat accesses also wait for one another).
template <typename T>
using Global = __attribute__((address_space(1))) T*;
template <typename T>
__device__ __forceinline__ Global<T> global(const void* p) {
    return (Global<T>)p;
}

// Four elements from `at` on of a chunk of n, at any element alignment. FULL: all four exist.
// Otherwise the missing ones are loaded as the chunk's last and become zero, so that no lane
// branches around a load (each branch would wait for the loads in it), and are not stored.
__device__ __forceinline__ uint32_t inside(uint32_t at, uint32_t n) { return at < n ? at : n - 1; }
typedef unsigned int u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));
template <typename TR, bool FULL>
__device__ __forceinline__ void load_half4(const void* p, uint32_t at, uint32_t n, float (&x)[4]) {
    using E = typename TR::elem;
    const auto e = global<const E>(p);
    if (FULL) {
        const u32x2 raw = __builtin_nontemporal_load((Global<const u32x2_a2>)(e + at));
        E h[4];
        __builtin_memcpy(h, &raw, 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = TR::to_f(h[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = TR::to_f(e[inside(at + i, n)]);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = at + i < n ? x[i] : 0.f;
    }
}
template <bool FULL>
__device__ __forceinline__ void load_float4(const void* p, uint32_t at, uint32_t n, float (&x)[4]) {
    const auto e = global<const float>(p);
    if (FULL) {
        const f32x4 v = __builtin_nontemporal_load((Global<const f32x4_a4>)(e + at));
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = v[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = e[inside(at + i, n)];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = at + i < n ? x[i] : 0.f;
    }
}
template <bool FULL>
__device__ __forceinline__ void load_grad4(const Chunk& c, uint32_t at, uint32_t n, float (&x)[4]) {
    if (c.grad_type == CLK_F32) load_float4<FULL>(c.g, at, n, x);
    else if (c.grad_type == CLK_BF16) load_half4<BF16, FULL>(c.g, at, n, x);
    else load_half4<F16, FULL>(c.g, at, n, x);
}
template <bool FULL>
__device__ __forceinline__ void store_float4(void* p, uint32_t at, uint32_t n, const float (&x)[4]) {
    const auto e = global<float>(p) + at;
    if (FULL) {
        *(Global<f32x4_a4>)e = f32x4{x[0], x[1], x[2], x[3]};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i < n) e[i] = x[i];
    }
}
template <typename TR, bool FULL>
__device__ __forceinline__ void store_half4(void* p, uint32_t at, uint32_t n, const float (&x)[4]) {
    using E = typename TR::elem;
    const auto e = global<E>(p) + at;
    E h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = TR::from_f(x[i]);
    if (FULL) {
        u32x2 raw;
        __builtin_memcpy(&raw, h, 8);
        *(Global<u32x2_a2>)e = raw;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i < n) e[i] = h[i];
    }
}
template <bool FULL>
__device__ __forceinline__ void store_copy4(const Chunk& c, uint32_t at, uint32_t n,
                                            const float (&x)[4]) {
    if (c.copy_type == CLK_BF16) store_half4<BF16, FULL>(c.copy, at, n, x);
    else if (c.copy_type == CLK_F16) store_half4<F16, FULL>(c.copy, at, n, x);
}
template <bool FULL>
__device__ __forceinline__ uint32_t load_codes4(const void* p, uint32_t at, uint32_t n) {
    const auto e = global<const uint8_t>(p);
    if (FULL) return *(Global<const uint32_t>)(e + at);
    uint32_t q = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        q |= (at + i < n ? (uint32_t)e[inside(at + i, n)] : 0u) << (8 * i);
    return q;
}
template <bool FULL>
__device__ __forceinline__ void store_codes4(void* p, uint32_t at, uint32_t n, uint32_t q) {
    const auto e = global<uint8_t>(p) + at;
    if (FULL) {
        *(Global<uint32_t>)e = q;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i < n) e[i] = (uint8_t)(q >> (8 * i));
    }
}

// sqrt(x) within 2 ulp: the hardware's root, of a scaled argument where that is too small for it.
__device__ __forceinline__ float near_sqrt(float x) {
    const bool small = x < 0x1p-96f;
    return __builtin_amdgcn_sqrtf(x * (small ? 0x1p64f : 1.f)) * (small ? 0x1p-32f : 1.f);
}
// The moments are rounded operation by operation; the weight's step takes the hardware's root and
// reciprocal (1 ulp each, of a step that is itself a small part of the weight).
__device__ __forceinline__ void update(const Step& s, float grad, float& p, float& m, float& v) {
    const float g = grad * s.grad_scale;
    m = m * s.b1 + g * s.omb1;
    v = v * s.b2 + (g * s.omb2) * g;
    const float denom = near_sqrt(v) * s.inv_bias2 + s.eps;
    p = p * s.keep - m * fast_rcp(denom) * s.step;
}

// A block takes a chunk, a thread four elements of it: all of a chunk's loads are in flight at once
// (chunks of 4096 elements in four rounds took 94 us instead of 84 for eight blocks' parameters).
constexpr int kChunk = 4 * kThreads;

template <bool FULL>
__device__ __forceinline__ void step32(const Chunk& c, const Step& s) {
    const uint32_t at = 4 * threadIdx.x;
    float ps[4], gs[4], ms[4], vs[4];
    load_float4<FULL>(c.p, at, c.n, ps);
    load_float4<FULL>(c.m, at, c.n, ms);
    load_float4<FULL>(c.v, at, c.n, vs);
    load_grad4<FULL>(c, at, c.n, gs);
#pragma unroll
    for (int i = 0; i < 4; ++i) update(s, gs[i], ps[i], ms[i], vs[i]);
    store_float4<FULL>(c.p, at, c.n, ps);
    store_float4<FULL>(c.m, at, c.n, ms);
    store_float4<FULL>(c.v, at, c.n, vs);
    if (c.copy_type) store_copy4<FULL>(c, at, c.n, ps);
}

__global__ __launch_bounds__(kThreads) void adamw32_kernel(const Chunk* __restrict__ table,
                                                           Step s) {
    const Chunk c = load_chunk(table);
    read_hyper(s);
    if (c.n == kChunk) step32<true>(c, s);
    else step32<false>(c, s);
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

constexpr uint32_t kInfBits = 0x7F800000u, kNanBits = 0x7FC00000u;

// The codes of four elements, as the rounded operations of their definition give them. Those cost
// some 30 instructions an element for the correctly rounded quotients and roots, more than the
// memory leaves time for, and matter only where 127*sqrt(.) or 255*sqrt(sqrt(.)) lies next to a
// half. So the hardware's reciprocal and roots (1 ulp) come first: with them a value is off by at
// most 4 * 2^-23 of itself from the defined one (reciprocal and product under the root, root, last
// product, on both sides): 127 * 2^-21 < 2^-14 and 255 * 2^-21 < 2^-13. Lanes that come within twice
// that of a half take the definition, and so does a block whose scale's reciprocal is not a normal
// number. Quotients below 2^-96 give 0 either way.
__device__ __forceinline__ void encode(const float (&m)[4], const float (&v)[4], float sm,
                                       float sv, uint32_t& qm, uint32_t& qv) {
    const float om = sm > 0.f ? sm : 1.f, ov = sv > 0.f ? sv : 1.f;
    const float im = fast_rcp(om), iv = fast_rcp(ov);
    float tm[4], tv[4];
    constexpr float kLow = 0x1p-120f, kHigh = 0x1p120f;
    bool exact = om < kLow || om > kHigh || ov < kLow || ov > kHigh;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = __builtin_amdgcn_sqrtf(fabsf(m[i]) * im) * 127.f;
        const float b = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(v[i] * iv)) * 255.f;
        tm[i] = rintf(a);
        tv[i] = rintf(b);
        exact |= fabsf(a - tm[i]) > 0.5f - 0x1p-13f || fabsf(b - tv[i]) > 0.5f - 0x1p-12f;
    }
    if (exact) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            tm[i] = rintf(sqrtf(fabsf(m[i]) / om) * 127.f);
            tv[i] = rintf(sqrtf(sqrtf(v[i] / ov)) * 255.f);
        }
    }
    qm = qv = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = v[i] > 0.f ? fmaxf(tv[i], 1.f) : tv[i];
        qm |= ((uint32_t)(int)(m[i] < 0.f ? -tm[i] : tm[i]) & 255u) << (8 * i);
        qv |= ((uint32_t)(int)q & 255u) << (8 * i);
    }
}

// A wave takes a block of 256 elements, four a lane.
template <bool FULL>
__device__ __forceinline__ void step8(const Chunk& c, const Step& s) {
    const int lane = threadIdx.x & 63;
    const uint32_t b = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (!FULL && b * kBlock >= c.n) return;
    const uint32_t at = b * kBlock + 4 * lane;
    const auto scales = global<float>(c.scales) + 2 * b;
    float ps[4], gs[4], ms[4], vs[4];
    const uint32_t qm0 = load_codes4<FULL>(c.m, at, c.n), qv0 = load_codes4<FULL>(c.v, at, c.n);
    const float sm0 = scales[0], sv0 = scales[1];
    load_float4<FULL>(c.p, at, c.n, ps);
    load_grad4<FULL>(c, at, c.n, gs);
    decode(qm0, qv0, sm0, sv0, ms, vs);
    uint32_t am = 0, av = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        update(s, gs[i], ps[i], ms[i], vs[i]);
        if (FULL || at + i < c.n) {
            am = max(am, __float_as_uint(fabsf(ms[i])));
            av = max(av, __float_as_uint(fabsf(vs[i])));
        }
    }
    am = wave_max(am);
    av = wave_max(av);
    uint32_t qm, qv;
    encode(ms, vs, __uint_as_float(am), __uint_as_float(av), qm, qv);
    if (am >= kInfBits) qm = 0, am = kNanBits;
    if (av >= kInfBits) qv = 0, av = kNanBits;
    store_float4<FULL>(c.p, at, c.n, ps);
    store_codes4<FULL>(c.m, at, c.n, qm);
    store_codes4<FULL>(c.v, at, c.n, qv);
    if (lane == 0) {
        scales[0] = __uint_as_float(am);
        scales[1] = __uint_as_float(av);
    }
    if (c.copy_type) store_copy4<FULL>(c, at, c.n, ps);
}

__global__ __launch_bounds__(kThreads) void adamw8_kernel(const Chunk* __restrict__ table,
                                                          Step s) {
    const Chunk c = load_chunk(table);
    read_hyper(s);
    if (c.n == kChunk) step8<true>(c, s);
    else step8<false>(c, s);
}

// The float32 states in flat buffers where every tensor begins at a multiple of 256 elements, with
// zeros up to the next one: a wave takes two of a chunk's blocks of 256 elements (48 Evoformer
// blocks' step and states: 410 us, with one or four blocks a wave 417 and 421).
constexpr int WB = 2;
template <int BITS, bool FULL>
__device__ __forceinline__ void states(const Chunk& c, float* m, float* v) {
    const int lane = threadIdx.x & 63;
    const uint32_t b0 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * WB;
    float ms[WB][4], vs[WB][4], sm[WB], sv[WB];
    uint32_t qm[WB], qv[WB];
#pragma unroll
    for (int k = 0; k < WB; ++k) {
        const uint32_t b = b0 + k, at = b * kBlock + 4 * lane;
        if (BITS == 8) {
            const auto scales = global<const float>(c.scales);
            const bool there = FULL || b * kBlock < c.n;
            qm[k] = load_codes4<FULL>(c.m, at, c.n);
            qv[k] = load_codes4<FULL>(c.v, at, c.n);
            sm[k] = there ? scales[2 * b] : 0.f;
            sv[k] = there ? scales[2 * b + 1] : 0.f;
        } else {
            load_float4<FULL>(c.m, at, c.n, ms[k]);
            load_float4<FULL>(c.v, at, c.n, vs[k]);
        }
    }
#pragma unroll
    for (int k = 0; k < WB; ++k) {
        const uint32_t b = b0 + k, at = b * kBlock + 4 * lane;
        if (!FULL && b * kBlock >= c.n) break;
        if (BITS == 8) {
            decode(qm[k], qv[k], sm[k], sv[k], ms[k], vs[k]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!FULL && at + i >= c.n) ms[k][i] = vs[k][i] = 0.f;  // a NaN scale's as well
        }
        __builtin_nontemporal_store(f32x4{ms[k][0], ms[k][1], ms[k][2], ms[k][3]},
                                    reinterpret_cast<f32x4*>(m + c.at + at));
        __builtin_nontemporal_store(f32x4{vs[k][0], vs[k][1], vs[k][2], vs[k][3]},
                                    reinterpret_cast<f32x4*>(v + c.at + at));
    }
}
constexpr int kStatesThreads = kChunk / 4 / WB;
template <int BITS>
__global__ __launch_bounds__(kStatesThreads) void adamw_states_kernel(
    const Chunk* __restrict__ table, float* __restrict__ m, float* __restrict__ v) {
    const Chunk c = load_chunk(table);
    if (c.n == kChunk) states<BITS, true>(c, m, v);
    else states<BITS, false>(c, m, v);
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------

// A launch holds fewer than 2^32 threads.
constexpr int64_t kMaxChunks = (1 << 24) - 1;

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
    int64_t total = 0, count = 0;
    std::vector<Span> spans;
    for (int64_t i = 0; i < n; ++i) {
        const clk_adamw_tensor& t = tensors[i];
        const clk_status s = check_tensor(who, t, i, bits);
        if (s != CLK_OK) return s;
        total += t.numel;
        count += up(t.numel, kChunk);
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
    if (count > kMaxChunks)
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
        for (int64_t o = 0; o < t.numel; o += kChunk) {
            Chunk c;
            c.p = t.param + o;
            c.g = static_cast<const char*>(t.grad) + o * (int64_t)elem_size(t.grad_dtype);
            c.m = static_cast<char*>(t.exp_avg) + o * (bits / 8);
            c.v = static_cast<char*>(t.exp_avg_sq) + o * (bits / 8);
            c.scales = bits == 8 ? t.scales + 2 * (o / kBlock) : nullptr;
            c.copy = t.copy ? static_cast<char*>(t.copy) + 2 * o : nullptr;
            c.at = base + o;
            c.n = (uint32_t)std::min<int64_t>(kChunk, t.numel - o);
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
    if (chunks < 0 || chunks > kMaxChunks)
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
    if (!((float)eps >= 0x1p-126f) || !std::isfinite((float)eps))
        return fail(CLK_INVALID_ARGUMENT, "%s: eps must be positive (a normal float32) and finite",
                    who);
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
        adamw_states_kernel<8><<<(int)chunks, kStatesThreads, 0, stream>>>(t, exp_avg, exp_avg_sq);
    else
        adamw_states_kernel<32><<<(int)chunks, kStatesThreads, 0, stream>>>(t, exp_avg, exp_avg_sq);
    return check_launch(who);
}
