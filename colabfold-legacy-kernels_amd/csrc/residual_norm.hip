// The join of a block's output o with its residual stream x, and the norm in front of the next
// block, for gfx950: forward and backward.
//
//   u = N_post(o);  t = sigmoid(gate) * u;  r = round(x + a * t);  h = N_pre(r)
//
// with N a LayerNorm or an RMS norm over the last axis (float32 scale, and offset where given) and
// a [C] float32. The norm after the block, the gate, a and the norm before the next block may each
// be absent. r is rounded to its type before it is normed, so h is what a norm of the stored
// stream gives and the backward pass, which reads r, sees the same numbers.
//
// Backward, with the gradients dr of r (from the stream's other readers) and dh of h:
//   D = dr + N_pre'(dh; r);  dx = D;  du = a * D * s (s = sigmoid(gate));
//   dgate = a * D * u * s * (1 - s);  do = N_post'(du; o)
//   N'(dy; v) = rstd * (g - mean(g) - vhat * mean(g * vhat)), g = scale * dy (no mean(g): RMS)
// and the column sums over the rows: dh * rhat, dh, D * t, du * ohat, du.
//
// HBM-bound: a team of lanes holds its row in registers from the loads to the stores, so the
// forward moves 3 reads and 2 writes of [M, C], the backward 5 reads and 3 writes; all statistics,
// sums and intermediate values are float32. Rows are read once: non-temporal loads take the forward
// of [512*512, 128] bf16 from 60.4 to 58.7 us (5.7 TB/s) and the backward of [384*384, 128] from
// 68.3 to 65; there plain stores in place of non-temporal ones make it 57.6 (5.2 TB/s), while they
// cost the forward 2.
#include "rows.hpp"

namespace clk {
namespace {

constexpr int kThreads = 256;
constexpr int kSums = 5;  // column sums: dpre_scale, dpre_offset, dres_scale, dpost_scale, dpost_offset

struct Params {
    const float *post_scale, *post_offset, *res_scale, *pre_scale, *pre_offset;
    int64_t M;
    int C;
    int rms;
    float eps;
};

// K sums over the lanes of a team of T lanes (a part of a wave, a wave, or a whole block), the
// same bits in every lane. `lds` holds two sets of one slot a wave, used in turn (`turn`), so one
// barrier a call is enough: a set is written again only after the barrier of the other.
template <int T, int K>
__device__ __forceinline__ void team_sums(float (&v)[K], float* lds, int& turn) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = group_sum<(T < 64 ? T : 64)>(v[k]);
    if constexpr (T > 64) {
        constexpr int W = T / 64;
        float* set = lds + turn * (2 * W);
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) set[k * W + (threadIdx.x >> 6)] = v[k];
        }
        lds_barrier();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float s = set[k * W];
#pragma unroll
            for (int w = 1; w < W; ++w) s += set[k * W + w];
            v[k] = s;
        }
    }
}

__device__ __forceinline__ float sigmoid(float x) {
    return fast_rcp(1.f + fast_exp2(-kLog2e * x));
}

// How a row fills its team: its last vector may be partial; whole vectors; as many columns as the
// team holds (no element needs a test: 10% fewer instructions in the backward).
enum Fill { kPartial, kWhole, kExact };

// The elements that a lane holds: NV vectors, at columns (v * T + s) * N.
template <typename TR, int T, int NV, Fill FILL>
struct Lane {
    static constexpr int N = Vec<TR>::N;
    static constexpr bool WHOLE = FILL != kPartial;
    using E = typename TR::elem;
    int s;
    int C;
    __device__ __forceinline__ int col(int v) const { return (v * T + s) * N; }
    __device__ __forceinline__ bool has(int v, int i) const {
        return FILL == kExact || (WHOLE ? col(v) < C : col(v) + i < C);
    }
    __device__ __forceinline__ bool has(int v) const { return FILL == kExact || col(v) < C; }
    // The loads of a row take no branch (a branch would wait for the loads in it before the next:
    // 21.8 against 15.6 us in the backward of [2053, 449] float32). Vectors that do not exist are
    // loaded from elsewhere in the row, and unpack makes them zeros. `row` has to exist.
    __device__ __forceinline__ int from(int v) const {
        return FILL == kPartial ? min(col(v), max(C - N, 0)) : has(v) ? col(v) : 0;
    }
    __device__ __forceinline__ void load(const E* p, int64_t row, u32x4 (&raw)[NV]) const {
        if (FILL == kPartial && C < N) {  // the same for all rows
#pragma unroll
            for (int v = 0; v < NV; ++v)
                raw[v] = has(v) ? load_vec<TR, false>(p + (size_t)row * C, col(v), C) : u32x4{};
            return;
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const E* e = p + (size_t)row * C + from(v);
            raw[v] = WHOLE ? __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(e))
                           : ld16_a2(e);
        }
    }
    __device__ __forceinline__ void unpack(u32x4 raw, int v, bool there, float (&x)[N]) const {
        if (FILL == kPartial && C >= N) raw = move_to<TR>(raw, min(from(v), col(v)), col(v));
        if (!there || !has(v)) raw = u32x4{0u, 0u, 0u, 0u};
        unpack_vec<TR>(raw, x);
    }
    // The forward's stores are non-temporal, the backward's are not: its three results then stay
    // in the caches beside the loads that pass them by.
    template <bool NT>
    __device__ __forceinline__ void store(E* p, int64_t row, int v, const float (&x)[N]) const {
        if (has(v)) store_vec<TR, WHOLE, NT>(p + (size_t)row * C, col(v), C, pack_vec<TR>(x));
    }
    __device__ __forceinline__ void floats(const float* p, float none,
                                           float (&out)[NV][N]) const {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (p && has(v)) {
                load_floats<N, WHOLE>(p, col(v), C, none, out[v]);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) out[v][i] = none;
            }
        }
    }
};

// Statistics of one row: mean (0 for an RMS norm) and 1 / sqrt(variance + eps), in two passes over
// the registers.
template <int T, typename L, int NV, int N>
__device__ __forceinline__ void row_stats(const L& lane, const float (&x)[NV][N],
                                          const Params& p, float* lds, int& turn, float& mean,
                                          float& rstd) {
    const float inv = 1.f / (float)p.C;
    mean = 0.f;
    float sum[1] = {0.f};
    if (!p.rms) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < N; ++i) sum[0] += x[v][i];  // zeros past the row's end
        team_sums<T>(sum, lds, turn);
        mean = sum[0] * inv;
    }
    sum[0] = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float d = lane.has(v, i) ? x[v][i] - mean : 0.f;
            sum[0] += d * d;
        }
    team_sums<T>(sum, lds, turn);
    rstd = rsqrtf(sum[0] * inv + p.eps);
}

// Threads of a block: a team that spans waves is the block.
template <int T>
constexpr int block_threads() {
    return T > 64 ? T : kThreads;
}

template <typename TR, int T, int NV, Fill FILL>
__global__ __launch_bounds__(block_threads<T>()) void join_fwd_kernel(
    const typename TR::elem* __restrict__ x, const typename TR::elem* __restrict__ o,
    const typename TR::elem* __restrict__ gate, typename TR::elem* __restrict__ r,
    typename TR::elem* __restrict__ h, Params p) {
    using L = Lane<TR, T, NV, FILL>;
    constexpr int N = L::N, ROWS = block_threads<T>() / T;
    __shared__ float lds[4 * (T > 64 ? T / 64 : 1)];
    int turn = 0;
    const L lane{(int)(threadIdx.x % T), p.C};
    const int slot = threadIdx.x / T;
    for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < p.M; row0 += (int64_t)gridDim.x * ROWS) {
        const int64_t row = row0 + slot;
        const bool there = row < p.M;
        u32x4 ro[NV], rx[NV], rg[NV];
        const int64_t in = there ? row : p.M - 1;
        lane.load(o, in, ro);
        lane.load(x, in, rx);
        if (gate) lane.load(gate, in, rg);
        float t[NV][N], w[NV][N];
#pragma unroll
        for (int v = 0; v < NV; ++v) lane.unpack(ro[v], v, there, t[v]);
        if (p.post_scale) {
            float mean, rstd, b[NV][N];
            row_stats<T>(lane, t, p, lds, turn, mean, rstd);
            lane.floats(p.post_scale, 0.f, w);
            lane.floats(p.post_offset, 0.f, b);
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < N; ++i) t[v][i] = (t[v][i] - mean) * rstd * w[v][i] + b[v][i];
        }
        if (gate) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                float g[N];
                lane.unpack(rg[v], v, there, g);
#pragma unroll
                for (int i = 0; i < N; ++i) t[v][i] *= sigmoid(g[i]);
            }
        }
        lane.floats(p.res_scale, 1.f, w);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float xs[N];
            lane.unpack(rx[v], v, there, xs);
#pragma unroll
            for (int i = 0; i < N; ++i) xs[i] += w[v][i] * t[v][i];
            if (there) lane.template store<true>(r, row, v, xs);
#pragma unroll
            for (int i = 0; i < N; ++i)
                t[v][i] = lane.has(v, i) ? TR::to_f(TR::from_f(xs[i])) : 0.f;
        }
        if (p.pre_scale) {
            float mean, rstd, b[NV][N];
            row_stats<T>(lane, t, p, lds, turn, mean, rstd);
            lane.floats(p.pre_scale, 0.f, w);
            lane.floats(p.pre_offset, 0.f, b);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                float y[N];
#pragma unroll
                for (int i = 0; i < N; ++i) y[i] = (t[v][i] - mean) * rstd * w[v][i] + b[v][i];
                if (there) lane.template store<true>(h, row, v, y);
            }
        }
    }
}

// Rows of any length: a block takes a row and passes over it again for each statistic; a thread
// always meets the same columns, so it reads back only what it wrote.
template <typename TR>
__global__ __launch_bounds__(kThreads) void join_fwd_long(
    const typename TR::elem* __restrict__ x, const typename TR::elem* __restrict__ o,
    const typename TR::elem* __restrict__ gate, typename TR::elem* r, typename TR::elem* h,
    Params p) {
    __shared__ float lds[4 * (kThreads / 64)];
    int turn = 0;
    const float inv = 1.f / (float)p.C;
    const auto stats = [&](const typename TR::elem* v, float& mean, float& rstd) {
        float sum[1] = {0.f};
        mean = 0.f;
        if (!p.rms) {
            for (int c = threadIdx.x; c < p.C; c += kThreads) sum[0] += TR::to_f(v[c]);
            team_sums<kThreads>(sum, lds, turn);
            mean = sum[0] * inv;
        }
        sum[0] = 0.f;
        for (int c = threadIdx.x; c < p.C; c += kThreads) {
            const float d = TR::to_f(v[c]) - mean;
            sum[0] += d * d;
        }
        team_sums<kThreads>(sum, lds, turn);
        rstd = rsqrtf(sum[0] * inv + p.eps);
    };
    for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
        const size_t base = (size_t)row * p.C;
        float mean = 0.f, rstd = 1.f;
        if (p.post_scale) stats(o + base, mean, rstd);
        for (int c = threadIdx.x; c < p.C; c += kThreads) {
            float t = TR::to_f(o[base + c]);
            if (p.post_scale)
                t = (t - mean) * rstd * p.post_scale[c] + (p.post_offset ? p.post_offset[c] : 0.f);
            if (gate) t *= sigmoid(TR::to_f(gate[base + c]));
            r[base + c] =
                TR::from_f(TR::to_f(x[base + c]) + (p.res_scale ? p.res_scale[c] : 1.f) * t);
        }
        if (p.pre_scale) {
            stats(r + base, mean, rstd);
            for (int c = threadIdx.x; c < p.C; c += kThreads)
                h[base + c] = TR::from_f((TR::to_f(r[base + c]) - mean) * rstd * p.pre_scale[c] +
                                         (p.pre_offset ? p.pre_offset[c] : 0.f));
        }
    }
}

struct SumsOut {
    float* to[kSums];
};

// Backward. A block walks its contiguous rows, ROWS at a time; each lane sums its columns over the
// rows it meets, the block joins its row slots in order, and join_colsum adds the blocks' partial
// rows part[block][sum][C4] in a fixed order; a block that is alone writes the results itself.
template <typename E>
struct BwdRows {
    const E *r, *o, *gate, *dr, *dh;
    E *dx, *d_o, *dgate;
};

template <typename TR, int T, int NV, Fill FILL>
__global__ __launch_bounds__(block_threads<T>()) void join_bwd_kernel(
    BwdRows<typename TR::elem> a, float* __restrict__ part, int C4, int rows_per_block, Params p,
    SumsOut result) {
    using L = Lane<TR, T, NV, FILL>;
    constexpr int N = L::N, ROWS = block_threads<T>() / T;
    __shared__ float lds[4 * (T > 64 ? T / 64 : 1)];
    int turn = 0;
    const L lane{(int)(threadIdx.x % T), p.C};
    const int slot = threadIdx.x / T;
    const float inv = 1.f / (float)p.C;
    // The parameters stay in LDS: in registers they would cost a wave a SIMD's worth of them.
    constexpr int PW = T * NV * N;  // columns that a team holds, at least C
    __shared__ __attribute__((aligned(16))) float prm[4][PW];
    for (int c = threadIdx.x; c < PW; c += block_threads<T>()) {
        const int in = min(c, p.C - 1);
        const float w0 = p.pre_scale ? p.pre_scale[in] : 0.f;
        const float w1 = p.post_scale ? p.post_scale[in] : 0.f;
        const float w2 = p.post_offset ? p.post_offset[in] : 0.f;
        const float w3 = p.res_scale ? p.res_scale[in] : 1.f;
        prm[0][c] = c < p.C ? w0 : 0.f;
        prm[1][c] = c < p.C ? w1 : 0.f;
        prm[2][c] = c < p.C ? w2 : 0.f;
        prm[3][c] = w3;
    }
    __syncthreads();
    const auto from_lds = [&](int k, float (&w)[NV][N]) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int q = 0; q < N; q += 4) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(&prm[k][lane.col(v) + q]);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[v][q + i] = x[i];
            }
    };
    float acc[kSums][NV][N];
#pragma unroll
    for (int k = 0; k < kSums; ++k)
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < N; ++i) acc[k][v][i] = 0.f;
    const int64_t beg = (int64_t)blockIdx.x * rows_per_block;
    const int64_t end = p.M - beg < rows_per_block ? p.M : beg + rows_per_block;
    // The next rows' loads are issued before the current rows' arithmetic.
    u32x4 nr[NV], no[NV], ng[NV], nd[NV], nh[NV];
    const auto fetch = [&](int64_t row) {
        const int64_t in = row < end ? row : end - 1;
        if (p.pre_scale) {
            lane.load(a.r, in, nr);
            lane.load(a.dh, in, nh);
        }
        lane.load(a.o, in, no);
        if (a.gate) lane.load(a.gate, in, ng);
        if (a.dr) lane.load(a.dr, in, nd);
    };
    fetch(beg + slot);
    for (int64_t row0 = beg; row0 < end; row0 += ROWS) {
        const int64_t row = row0 + slot;
        const bool there = row < end;
        u32x4 rr[NV], ro[NV], rg[NV], rd[NV], rh[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            rr[v] = nr[v];
            ro[v] = no[v];
            rg[v] = ng[v];
            rd[v] = nd[v];
            rh[v] = nh[v];
        }
        if (row0 + ROWS < end) fetch(row + ROWS);
        __atomic_signal_fence(__ATOMIC_SEQ_CST);  // keeps the parameters in LDS, not in registers

        float d[NV][N], w[NV][N];  // D
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (a.dr) {
                lane.unpack(rd[v], v, there, d[v]);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) d[v][i] = 0.f;
            }
        }
        if (p.pre_scale) {
            float y[NV][N], mean, rstd, s[2] = {0.f, 0.f};
#pragma unroll
            for (int v = 0; v < NV; ++v) lane.unpack(rr[v], v, there, y[v]);
            row_stats<T>(lane, y, p, lds, turn, mean, rstd);
            if (!there) rstd = 0.f;  // eps = 0: a row of zeros has none
            from_lds(0, w);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                float g[N];
                lane.unpack(rh[v], v, there, g);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float hat = (y[v][i] - mean) * rstd;
                    acc[0][v][i] += g[i] * hat;
                    acc[1][v][i] += g[i];
                    y[v][i] = hat;
                    w[v][i] *= g[i];
                    s[0] += w[v][i];
                    s[1] += w[v][i] * hat;
                }
            }
            team_sums<T>(s, lds, turn);
            const float m0 = p.rms ? 0.f : s[0] * inv, m1 = s[1] * inv;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < N; ++i) d[v][i] += rstd * (w[v][i] - m0 - y[v][i] * m1);
        }
        // Columns that do not exist, and rows that do not, have D = 0 and add nothing below.
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < N; ++i) d[v][i] = lane.has(v, i) ? d[v][i] : 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (there) lane.template store<false>(a.dx, row, v, d[v]);

        float u[NV][N], hat[NV][N], rstd = 1.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) lane.unpack(ro[v], v, there, u[v]);
        if (p.post_scale) {
            float mean, b[NV][N];
            row_stats<T>(lane, u, p, lds, turn, mean, rstd);
            if (!there) rstd = 0.f;
            from_lds(1, w);
            from_lds(2, b);
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    hat[v][i] = (u[v][i] - mean) * rstd;
                    u[v][i] = hat[v][i] * w[v][i] + b[v][i];
                }
        }
        {
            float as[NV][N];
            from_lds(3, as);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                float g[N], dg[N];
                if (a.gate) lane.unpack(rg[v], v, there, g);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float sig = a.gate ? sigmoid(g[i]) : 1.f;
                    acc[2][v][i] += d[v][i] * (sig * u[v][i]);
                    const float dt = as[v][i] * d[v][i];
                    dg[i] = dt * u[v][i] * (sig * (1.f - sig));
                    d[v][i] = dt * sig;  // du
                }
                if (a.gate && there) lane.template store<false>(a.dgate, row, v, dg);
            }
        }
        if (p.post_scale) {
            float s[2] = {0.f, 0.f};
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float du = d[v][i];
                    acc[3][v][i] += du * hat[v][i];
                    acc[4][v][i] += du;
                    d[v][i] = du * w[v][i];
                    s[0] += d[v][i];
                    s[1] += d[v][i] * hat[v][i];
                }
            team_sums<T>(s, lds, turn);
            const float m0 = p.rms ? 0.f : s[0] * inv, m1 = s[1] * inv;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < N; ++i)
                    d[v][i] = rstd * (d[v][i] - m0 - hat[v][i] * m1);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (there) lane.template store<false>(a.d_o, row, v, d[v]);
    }

    // Join the block's row slots, one sum at a time, in the order of the slots.
    const bool alone = gridDim.x == 1;
    const auto sums_to = [&](int k) {
        return alone ? result.to[k] : part + ((size_t)blockIdx.x * kSums + k) * C4;
    };
    if constexpr (ROWS == 1) {
#pragma unroll
        for (int k = 0; k < kSums; ++k)
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (lane.has(v) && sums_to(k))
                    store_floats<N>(sums_to(k), lane.col(v), alone ? p.C : C4, acc[k][v]);
    } else {
        __shared__ __attribute__((aligned(16))) float red[ROWS][PW];
#pragma unroll
        for (int k = 0; k < kSums; ++k) {
            if (k > 0) __syncthreads();
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < N; ++i) red[slot][lane.col(v) + i] = acc[k][v][i];
            __syncthreads();
            for (int c = threadIdx.x; c < p.C; c += kThreads) {
                float s = red[0][c];
                for (int j = 1; j < ROWS; ++j) s += red[j][c];
                if (sums_to(k)) sums_to(k)[c] = s;
            }
        }
    }
}

// Rows of any length: a block takes rows in turn and adds their column sums to its own partial row
// in memory; a thread always meets the same columns.
template <typename TR>
__global__ __launch_bounds__(kThreads) void join_bwd_long(BwdRows<typename TR::elem> a,
                                                          float* part, int C4, Params p) {
    __shared__ float lds[4 * (kThreads / 64)];
    int turn = 0;
    const float inv = 1.f / (float)p.C;
    float* out = part + (size_t)blockIdx.x * kSums * C4;
    for (int k = 0; k < kSums; ++k)
        for (int c = threadIdx.x; c < p.C; c += kThreads) out[(size_t)k * C4 + c] = 0.f;
    const auto stats = [&](const typename TR::elem* v, float& mean, float& rstd) {
        float sum[1] = {0.f};
        mean = 0.f;
        if (!p.rms) {
            for (int c = threadIdx.x; c < p.C; c += kThreads) sum[0] += TR::to_f(v[c]);
            team_sums<kThreads>(sum, lds, turn);
            mean = sum[0] * inv;
        }
        sum[0] = 0.f;
        for (int c = threadIdx.x; c < p.C; c += kThreads) {
            const float d = TR::to_f(v[c]) - mean;
            sum[0] += d * d;
        }
        team_sums<kThreads>(sum, lds, turn);
        rstd = rsqrtf(sum[0] * inv + p.eps);
    };
    for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
        const size_t base = (size_t)row * p.C;
        float mr = 0.f, sr = 1.f, mo = 0.f, so = 1.f, q[2] = {0.f, 0.f};
        if (p.pre_scale) {
            stats(a.r + base, mr, sr);
            for (int c = threadIdx.x; c < p.C; c += kThreads) {
                const float hat = (TR::to_f(a.r[base + c]) - mr) * sr;
                const float dy = TR::to_f(a.dh[base + c]), g = p.pre_scale[c] * dy;
                q[0] += g;
                q[1] += g * hat;
                out[c] += dy * hat;
                out[C4 + c] += dy;
            }
            team_sums<kThreads>(q, lds, turn);
        }
        const float q0 = p.rms ? 0.f : q[0] * inv, q1 = q[1] * inv;
        if (p.post_scale) stats(a.o + base, mo, so);
        // D of a column, and what its gate and u give.
        const auto column = [&](int c, float& d, float& u, float& hat, float& sig) {
            d = a.dr ? TR::to_f(a.dr[base + c]) : 0.f;
            if (p.pre_scale) {
                const float rhat = (TR::to_f(a.r[base + c]) - mr) * sr;
                d += sr * (p.pre_scale[c] * TR::to_f(a.dh[base + c]) - q0 - rhat * q1);
            }
            u = hat = TR::to_f(a.o[base + c]);
            if (p.post_scale) {
                hat = (u - mo) * so;
                u = hat * p.post_scale[c] + (p.post_offset ? p.post_offset[c] : 0.f);
            }
            sig = a.gate ? sigmoid(TR::to_f(a.gate[base + c])) : 1.f;
        };
        float s[2] = {0.f, 0.f};
        for (int c = threadIdx.x; c < p.C; c += kThreads) {
            float d, u, hat, sig;
            column(c, d, u, hat, sig);
            a.dx[base + c] = TR::from_f(d);
            out[2 * (size_t)C4 + c] += d * (sig * u);
            const float dt = (p.res_scale ? p.res_scale[c] : 1.f) * d, du = dt * sig;
            if (a.gate) a.dgate[base + c] = TR::from_f(dt * u * (sig * (1.f - sig)));
            if (p.post_scale) {
                out[3 * (size_t)C4 + c] += du * hat;
                out[4 * (size_t)C4 + c] += du;
                const float g = du * p.post_scale[c];
                s[0] += g;
                s[1] += g * hat;
            } else {
                a.d_o[base + c] = TR::from_f(du);
            }
        }
        if (p.post_scale) {
            team_sums<kThreads>(s, lds, turn);
            const float s0 = p.rms ? 0.f : s[0] * inv, s1 = s[1] * inv;
            for (int c = threadIdx.x; c < p.C; c += kThreads) {
                float d, u, hat, sig;
                column(c, d, u, hat, sig);
                const float du = (p.res_scale ? p.res_scale[c] : 1.f) * d * sig;
                a.d_o[base + c] = TR::from_f(so * (du * p.post_scale[c] - s0 - hat * s1));
            }
        }
    }
}

// out.to[k][c] = sum over the blocks' partial rows, in a fixed order: thread i adds rows i, i+256,
// ..., a wave joins its lanes by a fixed butterfly and the four waves are added in order. Four
// columns a block.
__global__ __launch_bounds__(256) void join_colsum(const float* __restrict__ part, int nblocks,
                                                   int C, int C4, SumsOut out) {
    constexpr int U = 4;
    const int u = xcd_contiguous(blockIdx.x, gridDim.x);
    const int k = u / (C4 / 4), c = 4 * (u - k * (C4 / 4));
    float* to = out.to[k];
    if (!to) return;
    const f32x4* p4 = reinterpret_cast<const f32x4*>(part) + u;
    const size_t stride = (size_t)kSums * C4 / 4;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    for (int b0 = threadIdx.x; b0 < nblocks; b0 += 256 * U) {
        f32x4 v[U];
#pragma unroll
        for (int i = 0; i < U; ++i)
            v[i] = b0 + 256 * i < nblocks ? p4[(size_t)(b0 + 256 * i) * stride]
                                          : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < U; ++i) a += v[i];
    }
    __shared__ f32x4 wsum[4];
    f32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = group_sum<64>(a[j]);
    if ((threadIdx.x & 63) == 0) wsum[threadIdx.x >> 6] = w;
    __syncthreads();
    if (threadIdx.x < 4 && c + (int)threadIdx.x < C)
        to[c + threadIdx.x] = ((wsum[0][threadIdx.x] + wsum[1][threadIdx.x]) +
                               wsum[2][threadIdx.x]) + wsum[3][threadIdx.x];
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------

// Lanes and vectors a lane for a row: a team of a power of two of lanes, two vectors a lane where
// a row has eight or more (as the LayerNorm kernels), up to 512 vectors; {0, 0}: the long form.
struct Team {
    int t, nv;
};
Team team_of(int64_t nvec, int want) {
    if (nvec > 512) return {0, 0};
    if (nvec > 64 * want) return {256, nvec > 256 ? 2 : 1};
    int t = 4;
    while (t < 64 && t * want < nvec) t *= 2;
    return {t, nvec > t ? 2 : 1};
}

// Blocks of the backward: the three a CU that its registers allow, so that all run at once (with
// 1024 the last quarter ran alone: 81 us against 72 at [384*384, 128] bf16); one for long rows, so
// that the partial sums stay small.
int64_t bwd_blocks(int64_t C) { return C <= 4096 ? 768 : 256; }
int64_t bwd_rows_per_block(int64_t M, int64_t C, int t) {
    const int64_t slots = t > 64 ? 1 : kThreads / t;
    // Up to four rounds of rows go to one block, which then needs no second launch.
    if (M <= 4 * slots) return 4 * slots;
    return slots * up(up(M, slots), bwd_blocks(C));
}

// Calls f(T, NV, FILL) as integral constants for the team of a row of C elements, N a vector.
template <typename F>
bool with_team(Team k, int64_t C, int N, F f) {
    const Fill fill = C % N ? kPartial : C == (int64_t)k.t * k.nv * N ? kExact : kWhole;
#define CLK_JOIN_FILL(T, NV, FILL)                                                  \
    f(std::integral_constant<int, T>(), std::integral_constant<int, NV>(),          \
      std::integral_constant<Fill, FILL>())
#define CLK_JOIN_CASE(T, NV)                                                        \
    if (k.t == (T) && k.nv == (NV)) {                                               \
        if (fill == kExact) CLK_JOIN_FILL(T, NV, kExact);                           \
        else if (fill == kWhole) CLK_JOIN_FILL(T, NV, kWhole);                      \
        else CLK_JOIN_FILL(T, NV, kPartial);                                        \
        return true;                                                                \
    }
#define CLK_JOIN_TEAM(T) CLK_JOIN_CASE(T, 1) CLK_JOIN_CASE(T, 2)
    CLK_JOIN_TEAM(4) CLK_JOIN_TEAM(8) CLK_JOIN_TEAM(16) CLK_JOIN_TEAM(32) CLK_JOIN_TEAM(64)
    CLK_JOIN_TEAM(256)
#undef CLK_JOIN_TEAM
#undef CLK_JOIN_CASE
#undef CLK_JOIN_FILL
    return false;
}

template <typename TR>
void launch_fwd(hipStream_t st, const void* x, const void* o, const void* gate, void* r, void* h,
                const Params& p) {
    using E = typename TR::elem;
    constexpr int N = Vec<TR>::N;
    const E *xe = static_cast<const E*>(x), *oe = static_cast<const E*>(o),
            *ge = static_cast<const E*>(gate);
    E *re = static_cast<E*>(r), *he = static_cast<E*>(h);
    KernelTimer timer("residual_norm", st);
    const bool done = with_team(team_of(up(p.C, N), 2), p.C, N, [&](auto t, auto nv, auto w) {
        constexpr int T = decltype(t)::value;
        const int64_t blocks = up(p.M, T > 64 ? 1 : kThreads / T);
        join_fwd_kernel<TR, T, decltype(nv)::value, decltype(w)::value>
            <<<(int)std::min<int64_t>(blocks, 1 << 22), block_threads<T>(), 0, st>>>(xe, oe, ge,
                                                                                     re, he, p);
    });
    if (!done)
        join_fwd_long<TR><<<(int)std::min<int64_t>(p.M, 4096), kThreads, 0, st>>>(xe, oe, ge, re,
                                                                                  he, p);
}

template <typename TR>
void launch_bwd(hipStream_t st, const void* r, const void* o, const void* gate, const void* dr,
                const void* dh, void* dx, void* d_o, void* dgate, float* part, const SumsOut& out,
                const Params& p) {
    using E = typename TR::elem;
    constexpr int N = Vec<TR>::N;
    const BwdRows<E> a = {static_cast<const E*>(r),  static_cast<const E*>(o),
                          static_cast<const E*>(gate), static_cast<const E*>(dr),
                          static_cast<const E*>(dh), static_cast<E*>(dx),
                          static_cast<E*>(d_o),      static_cast<E*>(dgate)};
    const int C4 = (int)up(p.C, 4) * 4;
    int nblocks = 0;
    {
        KernelTimer timer("residual_norm_bwd", st);
        const bool done =
            with_team(team_of(up(p.C, N), 8 / N), p.C, N, [&](auto t, auto nv, auto w) {
                constexpr int T = decltype(t)::value;
                const int64_t rows = bwd_rows_per_block(p.M, p.C, T);
                nblocks = (int)up(p.M, rows);
                join_bwd_kernel<TR, T, decltype(nv)::value, decltype(w)::value>
                    <<<nblocks, block_threads<T>(), 0, st>>>(a, part, C4, (int)rows, p, out);
            });
        if (done && nblocks == 1) return;
        if (!done) {
            nblocks = (int)std::min<int64_t>(p.M, bwd_blocks(p.C));
            join_bwd_long<TR><<<nblocks, kThreads, 0, st>>>(a, part, C4, p);
        }
    }
    KernelTimer timer("residual_norm_bwd_colsum", st);
    join_colsum<<<kSums * (C4 / 4), 256, 0, st>>>(part, nblocks, p.C, C4, out);
}

clk_status validate(const char* who, clk_dtype dtype, int64_t M, int64_t C) {
    if (dtype != CLK_F16 && dtype != CLK_BF16 && dtype != CLK_F32)
        return fail(CLK_INVALID_ARGUMENT, "%s: dtype %s not supported (f16, bf16, f32)", who,
                    dtype_name(dtype));
    if (M < 0 || C <= 0)
        return fail(CLK_INVALID_ARGUMENT, "%s: rows must be [M,C] with C > 0", who);
    if (M > INT32_MAX || C > (1 << 20) || M * C > ((int64_t)1 << 40))
        return fail(CLK_INVALID_ARGUMENT, "%s: [M,C] = [%lld,%lld] too large", who, (long long)M,
                    (long long)C);
    return CLK_OK;
}

// Results may not lie over operands or each other: rows are written while others are read.
template <size_t NIN, size_t NOUT>
bool rows_overlap(const void* const (&in)[NIN], const void* const (&out)[NOUT], clk_dtype dtype,
                  int64_t M, int64_t C) {
    const size_t bytes = (size_t)M * C * (dtype == CLK_F32 ? 4 : 2);
    for (size_t i = 0; i < NOUT; ++i) {
        for (const void* p : in)
            if (overlap(out[i], bytes, p, bytes)) return true;
        for (size_t j = 0; j < i; ++j)
            if (overlap(out[i], bytes, out[j], bytes)) return true;
    }
    return false;
}

clk_status validate_norms(const char* who, clk_norm norm, const float* post_scale,
                          const float* post_offset, const float* pre_scale,
                          const float* pre_offset) {
    if (norm != CLK_NORM_LAYER && norm != CLK_NORM_RMS)
        return fail(CLK_INVALID_ARGUMENT, "%s: norm %d not supported (layer, rms)", who, (int)norm);
    if ((!post_scale && post_offset) || (!pre_scale && pre_offset))
        return fail(CLK_INVALID_ARGUMENT, "%s: a norm's offset without its scale", who);
    return CLK_OK;
}

}  // namespace
}  // namespace clk

using namespace clk;

extern "C" clk_status clk_residual_norm_fwd(hipStream_t stream, clk_dtype dtype, clk_norm norm,
                                            const void* x, const void* o, const void* gate,
                                            const float* post_scale, const float* post_offset,
                                            const float* res_scale, const float* pre_scale,
                                            const float* pre_offset, void* r, void* h, int64_t M,
                                            int64_t C, float eps) {
    const char* who = "residual_norm";
    clk_status s = validate(who, dtype, M, C);
    if (s != CLK_OK) return s;
    s = validate_norms(who, norm, post_scale, post_offset, pre_scale, pre_offset);
    if (s != CLK_OK) return s;
    if ((pre_scale != nullptr) != (h != nullptr) && M > 0)
        return fail(CLK_INVALID_ARGUMENT, "%s: h is given with pre_scale, and only with it", who);
    if (M == 0) return ok();
    if (!x || !o || !r) return fail(CLK_INVALID_ARGUMENT, "%s: null pointer", who);
    if (!aligned16(x) || !aligned16(o) || !aligned16(gate) || !aligned16(r) || !aligned16(h))
        return fail(CLK_INVALID_ARGUMENT, "%s: x, o, gate, r and h must be 16-byte aligned", who);
    if (rows_overlap({x, o, gate}, {r, h}, dtype, M, C))
        return fail(CLK_INVALID_ARGUMENT, "%s: r and h may not overlap x, o, gate or each other",
                    who);
    const Params p = {post_scale, post_offset, res_scale, pre_scale,
                      pre_offset, M,           (int)C,    norm == CLK_NORM_RMS, eps};
    switch (dtype) {
        case CLK_BF16: launch_fwd<BF16>(stream, x, o, gate, r, h, p); break;
        case CLK_F16: launch_fwd<F16>(stream, x, o, gate, r, h, p); break;
        default: launch_fwd<F32>(stream, x, o, gate, r, h, p); break;
    }
    return check_launch(who);
}

extern "C" size_t clk_residual_norm_bwd_workspace_size(int64_t M, int64_t C) {
    if (M <= 0 || C <= 0) return 0;
    return (size_t)std::min<int64_t>(M, bwd_blocks(C)) * kSums * (size_t)up(C, 4) * 4 * sizeof(float);
}

extern "C" clk_status clk_residual_norm_bwd(
    hipStream_t stream, clk_dtype dtype, clk_norm norm, const void* r, const void* o,
    const void* gate, const float* post_scale, const float* post_offset, const float* res_scale,
    const float* pre_scale, const void* dr, const void* dh, void* dx, void* d_o, void* dgate,
    float* dpost_scale, float* dpost_offset, float* dres_scale, float* dpre_scale,
    float* dpre_offset, void* workspace, size_t workspace_bytes, int64_t M, int64_t C,
    float eps) {
    const char* who = "residual_norm_bwd";
    clk_status s = validate(who, dtype, M, C);
    if (s != CLK_OK) return s;
    s = validate_norms(who, norm, post_scale, post_offset, pre_scale, nullptr);
    if (s != CLK_OK) return s;
    if ((!post_scale && (dpost_scale || dpost_offset)) || (!res_scale && dres_scale) ||
        (!pre_scale && (dpre_scale || dpre_offset)))
        return fail(CLK_INVALID_ARGUMENT, "%s: gradient of a parameter that is not there", who);
    const SumsOut out = {{dpre_scale, dpre_offset, dres_scale, dpost_scale, dpost_offset}};
    if (M == 0) {  // no rows: the column sums are zero
        const int C4 = (int)up(C, 4) * 4;
        join_colsum<<<kSums * (C4 / 4), 256, 0, stream>>>(nullptr, 0, (int)C, C4, out);
        return check_launch(who);
    }
    if (!o || !dx || !d_o || !workspace || (!dr && !dh))
        return fail(CLK_INVALID_ARGUMENT, "%s: null pointer", who);
    if ((pre_scale != nullptr) != (dh != nullptr) || (pre_scale && !r))
        return fail(CLK_INVALID_ARGUMENT, "%s: r and dh are needed with pre_scale, dh only with it",
                    who);
    if ((gate != nullptr) != (dgate != nullptr))
        return fail(CLK_INVALID_ARGUMENT, "%s: dgate is given with gate, and only with it", who);
    if (!aligned16(r) || !aligned16(o) || !aligned16(gate) || !aligned16(dr) || !aligned16(dh) ||
        !aligned16(dx) || !aligned16(d_o) || !aligned16(dgate) || !aligned16(workspace))
        return fail(CLK_INVALID_ARGUMENT, "%s: rows and workspace must be 16-byte aligned", who);
    const size_t need = clk_residual_norm_bwd_workspace_size(M, C);
    if (workspace_bytes < need)
        return fail(CLK_INVALID_ARGUMENT, "%s: workspace %zu bytes, needs %zu", who,
                    workspace_bytes, need);
    if (rows_overlap({r, o, gate, dr, dh}, {dx, d_o, dgate}, dtype, M, C))
        return fail(CLK_INVALID_ARGUMENT,
                    "%s: dx, d_o and dgate may not overlap the operands or each other", who);
    const Params p = {post_scale, post_offset, res_scale, pre_scale,
                      nullptr,    M,           (int)C,    norm == CLK_NORM_RMS, eps};
    float* part = static_cast<float*>(workspace);
    switch (dtype) {
        case CLK_BF16:
            launch_bwd<BF16>(stream, r, o, gate, dr, dh, dx, d_o, dgate, part, out, p);
            break;
        case CLK_F16:
            launch_bwd<F16>(stream, r, o, gate, dr, dh, dx, d_o, dgate, part, out, p);
            break;
        default:
            launch_bwd<F32>(stream, r, o, gate, dr, dh, dx, d_o, dgate, part, out, p);
            break;
    }
    return check_launch(who);
}
