// Token embedding for gfx950: rows of a table, scaled, and the table's gradient.
//
//   out[i]    = scale * table[ids[i]]                       ids in [0, V); any other id is an
//   dtable[v] = scale * sum of dout[i] over ids[i] = v      absent token: a zero row, no gradient
//
// The forward is one pass that writes M*C*b bytes (the rows of a table that is used often stay in
// the L2s): 262144 tokens of 128 bf16 columns in 11.8 us, 5.7 TB/s.
//
// The gradient of a table of few rows is a product on the matrix cores that reads dout once, in
// order (147456 tokens, 65 rows of 128 bf16 columns: 17 us, of which the bytes need 7; sorting took
// 76). Others sort the tokens by row (stably, so that the order of every sum is fixed), sum runs of
// equal rows over the sorted order and join the runs that were cut; dout is read once, in whole
// rows of at least 256 bytes where a row has them (16411 tokens, 30011 rows of 640 float16 columns:
// 44 us, of which the bytes need 17 and the sort's four launches, with the zeros they write, 27).
#include "rows.hpp"

namespace clk {
namespace {

constexpr int kThreads = 256;
// ---------------------------------------------------------------------------------------------
// Forward: a block takes `rows` whole rows; thread t takes vectors t, t + 256, ... of them, four
// in flight, so that every wave writes consecutive vectors whatever C is.
// ---------------------------------------------------------------------------------------------
template <typename TR, typename ID, bool WHOLE>
__global__ __launch_bounds__(kThreads) void embed_kernel(
    const typename TR::elem* __restrict__ table, const ID* __restrict__ ids,
    typename TR::elem* __restrict__ out, int64_t M, int64_t V, int C, int rows, FastDiv nvec,
    float scale) {
    constexpr int N = Vec<TR>::N, U = 4;
    for (int64_t row0 = (int64_t)blockIdx.x * rows; row0 < M; row0 += (int64_t)gridDim.x * rows) {
        const int here = (int)(M - row0 < rows ? M - row0 : rows);
        const uint32_t total = (uint32_t)here * nvec.d;
        for (uint32_t f0 = threadIdx.x; f0 < total; f0 += U * kThreads) {
            int64_t id[U];
            uint32_t r[U];
            int col[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t f = f0 + u * kThreads < total ? f0 + u * kThreads : f0;
                r[u] = div_by(f, nvec);
                col[u] = (int)(f - r[u] * nvec.d) * N;
                id[u] = (int64_t)ids[row0 + r[u]];
            }
            u32x4 raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                raw[u] = id[u] >= 0 && id[u] < V
                             ? load_vec<TR, WHOLE>(table + (size_t)id[u] * C, col[u], C)
                             : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (f0 + u * kThreads >= total) break;
                // Absent rows are +0 whatever the scale is (a zero times infinity is NaN).
                if (id[u] >= 0 && id[u] < V) {
                    float v[N];
                    unpack_vec<TR>(raw[u], v);
#pragma unroll
                    for (int i = 0; i < N; ++i) v[i] *= scale;
                    raw[u] = pack_vec<TR>(v);
                }
                store_vec<TR, WHOLE, true>(out + (size_t)(row0 + r[u]) * C, col[u], C, raw[u]);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Sorting the tokens: keys are rows of the table, V for an absent token (they come last). These
// kernels wait for memory more than they use it: blocks behind the ones that sort set the gradient
// to zero meanwhile, a part in each kernel, so that the sums write only the rows that tokens name
// (16,411 tokens of 30,011 rows of 640 columns: all of it in the first kernel 48 us, in parts 43).
// ---------------------------------------------------------------------------------------------
template <typename ID>
__device__ __forceinline__ uint32_t token_key(const ID* ids, int64_t i, uint32_t V) {
    const int64_t id = (int64_t)ids[i];
    return id >= 0 && id < (int64_t)V ? (uint32_t)id : V;
}

// Keeps a wave's LDS operations in the order of the program (the hardware does not reorder them).
__device__ __forceinline__ void wave_order() {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_wave_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// A part of the gradient, floats [beg, end) with beg a multiple of four, that blocks first ..
// first + blocks - 1 of a grid fill.
struct Zero {
    float* p;
    size_t beg, end;
    int first, blocks;
};
// True for a block that fills (and has filled).
__device__ __forceinline__ bool zero_block(const Zero& z) {
    if ((int)blockIdx.x < z.first) return false;
    const size_t end4 = z.end / 4, step = (size_t)z.blocks * kThreads;
    const size_t b = (size_t)((int)blockIdx.x - z.first);
    f32x4* p4 = reinterpret_cast<f32x4*>(z.p);
    for (size_t i = z.beg / 4 + b * kThreads + threadIdx.x; i < end4; i += step)
        __builtin_nontemporal_store(f32x4{0.f, 0.f, 0.f, 0.f}, p4 + i);
    if (b == 0 && threadIdx.x < z.end % 4) z.p[4 * end4 + threadIdx.x] = 0.f;
    return true;
}

// Up to kRankMax tokens: each one's place is the number of tokens before it, counted over all of
// them. M^2 comparisons over the whole chip, in one launch: 16 tokens a block, 16 threads a token.
constexpr int kRankMax = 4096;  // 12 us, as two digits' passes; 8192 tokens 21 us against 16
constexpr int kRankTokens = 16, kRankSlices = kThreads / kRankTokens;
template <typename ID>
__global__ __launch_bounds__(kThreads) void embed_rank_kernel(const ID* __restrict__ ids, int M,
                                                              uint32_t V,
                                                              uint32_t* __restrict__ keys,
                                                              uint32_t* __restrict__ order,
                                                              Zero zero) {
    __shared__ __attribute__((aligned(16))) uint32_t k[kRankMax];
    if (zero_block(zero)) return;
    const int padded = (M + 3) & ~3;
    for (int i = threadIdx.x; i < padded; i += kThreads)
        k[i] = i < M ? token_key(ids, i, V) : ~0u;  // past every token
    __syncthreads();
    const int slice = threadIdx.x % kRankSlices;
    const int i = blockIdx.x * kRankTokens + threadIdx.x / kRankSlices;
    const uint32_t mine = i < M ? k[i] : 0;
    int before = 0;
    for (int j = 4 * slice; j < padded; j += 4 * kRankSlices) {
        const u32x4 o = *reinterpret_cast<const u32x4*>(k + j);
#pragma unroll
        for (int t = 0; t < 4; ++t) before += o[t] < mine + (j + t < i ? 1u : 0u);
    }
#pragma unroll
    for (int s = kRankSlices / 2; s > 0; s >>= 1) before += __shfl_xor(before, s);
    if (slice == 0 && i < M) {
        keys[before] = mine;
        order[before] = (uint32_t)i;
    }
}

// More tokens: a stable least-significant-digit radix sort, 8 bits a pass: the digits of each tile of
// tokens are counted, the counts summed over the tiles before, and the tokens moved. Up to
// kFewTiles tiles the moving blocks sum the counts themselves; more are summed by a kernel of its
// own, a block a digit. Count (digit, tile) is at digit * by_digit + tile * by_tile.
constexpr int kTile = 1024, kDigits = 256;
constexpr int64_t kFewTiles = 32;  // at 128 tiles the move takes 12 us, after a scan 8 + 2
struct Counts {
    uint32_t* n;
    int64_t tiles;
    size_t by_digit, by_tile;
    __device__ __forceinline__ uint32_t& at(int digit, int64_t tile) const {
        return n[digit * by_digit + tile * by_tile];
    }
};

template <typename ID>
struct FirstKeys {  // the first pass reads the ids themselves
    const ID* ids;
    uint32_t V;
    __device__ __forceinline__ uint32_t key(int64_t i) const { return token_key(ids, i, V); }
    __device__ __forceinline__ uint32_t value(int64_t i) const { return (uint32_t)i; }
};
struct NextKeys {
    const uint32_t *keys, *order;
    __device__ __forceinline__ uint32_t key(int64_t i) const { return keys[i]; }
    __device__ __forceinline__ uint32_t value(int64_t i) const { return order[i]; }
};

template <typename SRC>
__global__ __launch_bounds__(kThreads) void embed_count_kernel(SRC src, int64_t M, int shift,
                                                               Counts counts, Zero zero) {
    __shared__ uint32_t n[kDigits];
    if (zero_block(zero)) return;
    n[threadIdx.x] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * kTile;
#pragma unroll
    for (int u = 0; u < kTile / kThreads; ++u) {
        const int64_t i = base + u * kThreads + threadIdx.x;
        if (i < M) atomicAdd(&n[(src.key(i) >> shift) & 255u], 1u);  // whole numbers: any order
    }
    __syncthreads();
    counts.at(threadIdx.x, blockIdx.x) = n[threadIdx.x];
}

// Exclusive sums of one digit's counts over the tiles, in place, and its total.
__global__ __launch_bounds__(kThreads) void embed_scan_kernel(Counts counts,
                                                              uint32_t* __restrict__ totals) {
    __shared__ uint32_t wave_sum[kThreads / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t carry = 0;
    for (int64_t t0 = 0; t0 < counts.tiles; t0 += kThreads) {
        const int64_t t = t0 + threadIdx.x;
        const uint32_t own = t < counts.tiles ? counts.at(blockIdx.x, t) : 0;
        uint32_t sum = own;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const uint32_t o = __shfl_up(sum, s);
            if (lane >= s) sum += o;
        }
        if (lane == 63) wave_sum[wave] = sum;
        __syncthreads();
        uint32_t before = carry, all = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) {
            if (w < wave) before += wave_sum[w];
            all += wave_sum[w];
        }
        if (t < counts.tiles) counts.at(blockIdx.x, t) = before + sum - own;
        carry += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// Moves a tile's tokens to their places. Wave w takes the tile's w-th quarter, 64 consecutive
// tokens a round; lanes with equal digits find each other by eight ballots, so a token's rank
// follows the order of the tokens. `totals`: the scan kernel's, or null.
template <typename SRC>
__global__ __launch_bounds__(kThreads) void embed_scatter_kernel(
    SRC src, int64_t M, int shift, Counts counts, const uint32_t* __restrict__ totals,
    uint32_t* __restrict__ keys, uint32_t* __restrict__ order, Zero zero) {
    constexpr int kWaves = kThreads / 64, kRounds = kTile / kThreads;
    __shared__ uint32_t n[kWaves][kDigits];
    __shared__ uint32_t wave_sum[kWaves];
    if (zero_block(zero)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) n[w][threadIdx.x] = 0;
    // One thread a digit: its tokens in the tiles before this one, and in all.
    uint32_t earlier = 0, own = 0;
    if (totals) {
        earlier = counts.at(threadIdx.x, blockIdx.x);
        own = totals[threadIdx.x];
    } else {
        constexpr int U = 16;
        for (int t0 = 0; t0 < (int)counts.tiles; t0 += U) {
            uint32_t k[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                k[u] = t0 + u < (int)counts.tiles ? counts.at(threadIdx.x, t0 + u) : 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                own += k[u];
                earlier += t0 + u < (int)blockIdx.x ? k[u] : 0;
            }
        }
    }
    // Exclusive sum of the digits' totals.
    uint32_t sum = own;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const uint32_t o = __shfl_up(sum, s);
        if (lane >= s) sum += o;
    }
    if (lane == 63) wave_sum[wave] = sum;
    __syncthreads();
    uint32_t first = sum - own + earlier;
    for (int w = 0; w < wave; ++w) first += wave_sum[w];

    const int64_t base = (int64_t)blockIdx.x * kTile + wave * (kTile / kWaves);
    uint32_t key[kRounds], rank[kRounds];
#pragma unroll
    for (int u = 0; u < kRounds; ++u) {
        const int64_t i = base + u * 64 + lane;
        key[u] = i < M ? src.key(i) : 0;
    }
#pragma unroll
    for (int u = 0; u < kRounds; ++u) {
        const bool there = base + u * 64 + lane < M;
        const uint32_t digit = (key[u] >> shift) & 255u;
        uint64_t same = __ballot(there);
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const uint64_t set = __ballot((digit >> b) & 1u);
            same &= (digit >> b) & 1u ? set : ~set;
        }
        const uint64_t below = same & ((1ull << lane) - 1ull);
        if (there) {
            // LDS operations of a wave are in order: all its lanes read before the first lane of
            // each digit writes the new count.
            const uint32_t had = n[wave][digit];
            rank[u] = had + (uint32_t)__popcll(below);
            wave_order();
            if (below == 0) n[wave][digit] = had + (uint32_t)__popcll(same);
        }
        wave_order();
    }
    __syncthreads();
    // Where each wave's tokens of a digit begin.
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const uint32_t had = n[w][threadIdx.x];
        n[w][threadIdx.x] = first;
        first += had;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kRounds; ++u) {
        const int64_t i = base + u * 64 + lane;
        if (i < M) {
            const uint32_t to = n[wave][(key[u] >> shift) & 255u] + rank[u];
            keys[to] = key[u];
            order[to] = src.value(i);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Sums of the sorted tokens. A group of LPR lanes takes kRun tokens of the sorted order and one
// slice of LPR vectors of the columns; it keeps the running sum in registers and stores it where
// the row ends: into the table if the run also began in the group, else in LDS, as the group's
// `head` (of a run that began before it). A group whose last run goes on then adds the heads of the
// groups that it goes on into; what the block's ends cut leaves as a head or a tail of the block's
// chunk of tokens, and embed_join_kernel joins those.
// ---------------------------------------------------------------------------------------------
constexpr int kRun = 16;
template <int LPR>
constexpr int chunk_tokens() {
    return kThreads / LPR * kRun;
}

template <typename TR, int LPR, bool WHOLE>
__global__ __launch_bounds__(kThreads) void embed_sum_kernel(
    const typename TR::elem* __restrict__ dout, const uint32_t* __restrict__ keys,
    const uint32_t* __restrict__ order, float* __restrict__ dtable, float* __restrict__ head,
    float* __restrict__ tail, uint32_t M, uint32_t V, int C, FastDiv slices, float scale) {
    constexpr int N = Vec<TR>::N, U = 8, G = kThreads / LPR, W = LPR * N;
    static_assert(kRun % U == 0);
    __shared__ __attribute__((aligned(16))) float heads[G][W];
    __shared__ uint32_t first_key[G];
    const uint32_t chunk = div_by(blockIdx.x, slices), slice = blockIdx.x - chunk * slices.d;
    const int g = threadIdx.x / LPR, s = threadIdx.x % LPR;
    const int col = (int)(slice * LPR + s) * N;
    const bool cols = col < C;
    const uint32_t beg = chunk * chunk_tokens<LPR>() + g * kRun;
    const uint32_t end = beg >= M ? beg : M - beg < kRun ? M : beg + kRun;
    // The keys around the group, loaded at once.
    const uint32_t before = keys[beg > 0 && beg < M ? beg - 1 : 0], after = keys[min(end, M - 1)];
    uint32_t cur = beg < M ? keys[min(beg, M - 1)] : V;
    if (s == 0) first_key[g] = cur;
    // A head run began before the group; the last run goes on behind it.
    const bool has_head = beg > 0 && cur < V && before == cur;
    bool began = !has_head, has_tail = false;
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    const auto keep = [&](float (&piece)[W]) {
#pragma unroll
        for (int i = 0; i < N; ++i) piece[s * N + i] = acc[i];
    };
    const auto finish = [&](uint32_t row) {
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] *= scale;
        if (cols) store_floats(dtable + (size_t)row * C, col, C, acc);
    };
    for (uint32_t i0 = beg; i0 < end && cur < V; i0 += U) {
        uint32_t k[U], at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            k[u] = i0 + u < end ? keys[i0 + u] : V;
            at[u] = i0 + u < end ? order[i0 + u] : 0;
        }
        u32x4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            raw[u] = k[u] < V && cols ? load_vec<TR, WHOLE>(dout + (size_t)at[u] * C, col, C)
                                      : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + u >= end) break;
            if (k[u] != cur) {
                if (began) finish(cur);
                else keep(heads[g]);
#pragma unroll
                for (int i = 0; i < N; ++i) acc[i] = 0.f;
                cur = k[u];
                began = true;
                if (cur >= V) break;
            }
            float v[N];
            unpack_vec<TR>(raw[u], v);
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] += v[i];
        }
    }
    if (cur < V) {
        if (!began) {
            keep(heads[g]);
        } else if (end < M && after == cur) {
            has_tail = true;
        } else {
            finish(cur);
        }
    }
    __syncthreads();
    // The run of a tail goes on through the groups that begin with its key; the first group's head
    // is the block's.
    if (!has_tail && !(g == 0 && has_head)) return;
    for (int own = 0; own < 2; ++own) {
        if (own == 0 ? !(g == 0 && has_head) : !has_tail) continue;
        const uint32_t key = own == 0 ? first_key[0] : cur;
        int j = g + own;
        float sum[N];
#pragma unroll
        for (int i = 0; i < N; ++i) sum[i] = own == 0 ? 0.f : acc[i];
        for (; j < G && first_key[j] == key; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] += heads[j][s * N + i];
        const uint32_t next = (chunk + 1) * chunk_tokens<LPR>();
        float* to = head + (size_t)chunk * C;
        if (own == 1) {
            const bool goes_on = j == G && next < M && keys[next] == key;
            to = goes_on ? tail + (size_t)chunk * C : dtable + (size_t)key * C;
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] *= goes_on ? 1.f : scale;
        }
        if (cols) store_floats(to, col, C, sum);
    }
}

// Runs cut by the ends of chunks: the tail of the chunk they begin in plus the heads of the chunks
// they go on into, whose first keys are theirs. A block looks at one chunk and 256 columns, its
// waves take the heads in turn.
__global__ __launch_bounds__(kThreads) void embed_join_kernel(
    const uint32_t* __restrict__ keys, const float* __restrict__ head,
    const float* __restrict__ tail, float* __restrict__ dtable, uint32_t V, int C,
    uint32_t chunks, int tokens, FastDiv slices, float scale) {
    constexpr int kWaves = kThreads / 64, U = 16;
    __shared__ f32x4 part[kWaves][64];
    const uint32_t c = div_by(blockIdx.x, slices);  // not the last chunk
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = (int)((blockIdx.x - c * slices.d) * 64 + lane) * 4;
    const size_t beg = (size_t)c * tokens;
    const uint32_t before = keys[c > 0 ? beg - 1 : 0], begins = keys[beg],
                   ends = keys[beg + tokens - 1], key = keys[beg + tokens];
    // The run that the next chunk begins with began in this one, and is no absent tokens'.
    if (key >= V || ends != key || (c > 0 && begins == key && before == key)) return;
    const auto load = [&](const float* p, uint32_t chunk) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (col < C) load_floats<4, false>(p + (size_t)chunk * C, col, C, 0.f, v);
        return f32x4{v[0], v[1], v[2], v[3]};
    };
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (wave == 0) sum = load(tail, c);
    // The heads are loaded along with the keys that say whether they are this run's.
    for (uint32_t c0 = c + 1 + wave;; c0 += U * kWaves) {
        f32x4 p[U];
        uint32_t k[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t at = c0 + u * kWaves, in = min(at, chunks - 1);
            k[u] = at < chunks ? keys[(size_t)in * tokens] : V;
            p[u] = load(head, in);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) sum += k[u] == key ? p[u] : f32x4{0.f, 0.f, 0.f, 0.f};
        if (k[U - 1] != key) break;
    }
    part[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && col < C) {
#pragma unroll
        for (int w = 1; w < kWaves; ++w) sum += part[w][lane];
        const float v4[4] = {sum[0] * scale, sum[1] * scale, sum[2] * scale, sum[3] * scale};
        store_floats(dtable + (size_t)key * C, col, C, v4);
    }
}

// ---------------------------------------------------------------------------------------------
// Tables of few rows: the gradient is the product onehot(ids)^T . dout on the matrix cores, with
// float32 sums. No token is sorted and dout is read once, in order. A wave keeps every row of its
// 64 columns in registers (VT tiles of 16 rows x 4 tiles of 16 columns). A block's 8 waves take WC
// groups of columns and, 8/WC at a time, steps of 32 tokens; their sums are joined in LDS in the
// order of the waves and leave as one partial [V, C] a block, which embed_parts_kernel adds up.
//
// Neither operand goes through LDS. Lane (r16, g) of an MFMA holds eight tokens (8g + j) of row r16
// of A and of column r16 of B. As A it compares the ids of its tokens with its row; as B it loads
// columns 4*r16 .. +3 of each of its tokens, which are the four column tiles' operands once the
// token pairs are interleaved: tile ct then stands for the columns 4*r16 + ct.
//
// 0 * NaN and 0 * infinity would reach other rows: a wave whose sums are not all finite at the end
// adds its tokens up one by one instead.
// ---------------------------------------------------------------------------------------------
constexpr int kStep = 32, kHotWaves = 8, kHotCols = 64;
constexpr int kHotRows = 144;  // rows of a block; a table of more takes a block for each so many
// Tables of up to kHotRows rows take this path, and larger ones where reading dout once for every
// kHotRows rows costs less than the sort's launches: 4332 tokens of 496 rows of 256 columns 20.5 us
// instead of 29.2.
constexpr int64_t kHotSlices = 8, kHotWork = 1 << 23;
inline bool hot_table(int64_t M, int64_t V, int64_t C) {
    const int64_t slices = up(V, kHotRows);
    return slices <= 1 ||
           (slices <= kHotSlices && M * up(C, kHotCols) * kHotCols <= kHotWork / slices);
}

// A token's row counted from v0, -1 if it is not among the kHotRows rows from there on.
template <typename ID>
__device__ __forceinline__ int hot_id(ID id, int v0) {
    return id >= (ID)v0 && id < (ID)(v0 + kHotRows) ? (int)(id - (ID)v0) : -1;
}

// Tokens t .. t + 7 of a lane.
template <typename ID>
__device__ __forceinline__ void load_ids8(const ID* ids, int64_t t, int64_t end, int v0,
                                          int (&id)[8]) {
    typedef ID ID4 __attribute__((ext_vector_type(4), aligned(sizeof(ID))));
    if (t + 8 <= end) {
        const ID4 a = *reinterpret_cast<const ID4*>(ids + t);
        const ID4 b = *reinterpret_cast<const ID4*>(ids + t + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) id[j] = hot_id(a[j], v0), id[4 + j] = hot_id(b[j], v0);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) id[j] = t + j < end ? hot_id(ids[t + j], v0) : -1;
    }
}

// Four columns of a row, zero past its end.
template <typename TR>
struct Four {
    typename TR::elem e[4];
};
template <typename TR, bool WHOLE>
__device__ __forceinline__ Four<TR> load_four(const typename TR::elem* row, int col, int C) {
    using E = typename TR::elem;
    constexpr int R = sizeof(E);  // 4-byte words
    typedef unsigned int raw_t
        __attribute__((ext_vector_type(R), aligned(WHOLE ? 4 * sizeof(E) : sizeof(E))));
    Four<TR> f;
    if (WHOLE || C >= 4) {
        // A partial vector as load_vec takes it.
        const int at = WHOLE || col < C - 4 ? col : C - 4, s = col - at;
        const raw_t raw = *reinterpret_cast<const raw_t*>(row + at);
        u32x4 r = {raw[0], raw[1], 0u, 0u};
        if (R == 4) r = u32x4{raw[0], raw[1], raw[R - 2], raw[R - 1]};
        if (!WHOLE) r = R == 4 ? move_down4(r, s) : move_down2(r, s);
        __builtin_memcpy(&f, &r, sizeof(f));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) f.e[i] = col + i < C ? row[col + i] : TR::from_f(0.f);
    }
    return f;
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// The A operand of 16 rows: 1 - |id ^ row|, saturated at 0, is whether they are equal; times the
// bits of 1.
template <typename TR>
__device__ __forceinline__ typename TR::vec8 onehot(const u16x2 (&ids)[4], unsigned short row) {
    const unsigned short one = (unsigned short)kOnePair<TR>;
    u16x2 a[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
        a[q] = __builtin_elementwise_sub_sat(u16x2{1, 1}, ids[q] ^ u16x2{row, row}) *
               u16x2{one, one};
    typename TR::vec8 av;
    __builtin_memcpy(&av, a, 16);
    return av;
}

// One step of 32 tokens: acc[v][ct] += onehot . columns.
//
// A float32 column is the sum of three bf16 ones, its bits cut after 8, 16 and 24 (exactly, but for
// what lies below 2^-133), and three products of bf16 take a fifth of the matrix cores' time of one
// of float32: 147456 tokens of 65 rows of 128 columns 22 us instead of 36, 131072 of 23 rows of 256
// columns 30.4 instead of 33.4 (24 by their bytes).
template <typename TR, int VT>
__device__ __forceinline__ void hot_step(const int (&id)[8], const Four<TR> (&x)[8], int r16,
                                         f32x4 (&acc)[VT][4]) {
    u16x2 ids[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
        ids[q] = u16x2{(unsigned short)id[2 * q], (unsigned short)id[2 * q + 1]};
    if constexpr (sizeof(typename TR::elem) == 2) {
        using V8 = typename TR::vec8;
        V8 b[4];
#pragma unroll
        for (int ct = 0; ct < 4; ++ct)
#pragma unroll
            for (int j = 0; j < 8; ++j) b[ct][j] = x[j].e[ct];
#pragma unroll
        for (int v = 0; v < VT; ++v) {
            const V8 av = onehot<TR>(ids, (unsigned short)(16 * v + r16));
#pragma unroll
            for (int ct = 0; ct < 4; ++ct) acc[v][ct] = TR::mfma(av, b[ct], acc[v][ct]);
        }
    } else {
        using V8 = BF16::vec8;
#pragma unroll
        for (int ct = 0; ct < 4; ++ct) {
            // Many rows' A operands are made again for each column: kept, they would spill.
            if constexpr (VT > 5)
                asm volatile("" : "+v"(ids[0]), "+v"(ids[1]), "+v"(ids[2]), "+v"(ids[3]));
            uint32_t w[3][4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float f0 = x[2 * q].e[ct], f1 = x[2 * q + 1].e[ct];
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    const uint32_t u0 = __float_as_uint(f0), u1 = __float_as_uint(f1);
                    w[k][q] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
                    f0 -= __uint_as_float(u0 & 0xFFFF0000u);
                    f1 -= __uint_as_float(u1 & 0xFFFF0000u);
                }
            }
            V8 b[3];
            __builtin_memcpy(&b, w, sizeof(w));
#pragma unroll
            for (int v = 0; v < VT; ++v) {
                const V8 av = onehot<BF16>(ids, (unsigned short)(16 * v + r16));
#pragma unroll
                for (int k = 2; k >= 0; --k)  // the smallest first
                    acc[v][ct] = BF16::mfma(av, b[k], acc[v][ct]);
            }
            __builtin_amdgcn_sched_barrier(0);  // one column's operands at a time
        }
    }
}

template <typename TR, typename ID, int VT, int WC, bool WHOLE>
__global__ __launch_bounds__(64 * kHotWaves) void embed_hot_kernel(
    const typename TR::elem* __restrict__ dout, const ID* __restrict__ ids,
    float* __restrict__ out, size_t part_stride, int64_t M, int V, int C, int64_t tokens,
    float scale) {
    constexpr int WT = kHotWaves / WC;
    constexpr int LD = kHotCols + 4;
    __shared__ __attribute__((aligned(16))) float red[kHotWaves][16][LD];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const int cbase = (int)blockIdx.y * kHotCols * WC;
    const int col = cbase + (wave % WC) * kHotCols + 4 * r16;
    const int64_t beg = (int64_t)blockIdx.x * tokens;
    const int64_t end = M - beg < tokens ? M : beg + tokens;
    const int64_t first = beg + (wave / WC) * kStep;
    const int v0 = (int)blockIdx.z * kHotRows;

    f32x4 acc[VT][4];
#pragma unroll
    for (int v = 0; v < VT; ++v)
#pragma unroll
        for (int ct = 0; ct < 4; ++ct) acc[v][ct] = f32x4{0.f, 0.f, 0.f, 0.f};

    // Steps are wave-uniform, so a step's rows are at a scalar base and 32-bit lane offsets. Lanes
    // past the last column load the first ones; their sums are not stored.
    const int lcol = col < C ? col : 0;
    const auto load = [&](int64_t t0, int(&id)[8], Four<TR>(&x)[8]) {
        load_ids8(ids, t0 + 8 * g, end, v0, id);
        const typename TR::elem* base = dout + (size_t)t0 * C;
        const uint32_t off = (uint32_t)(8 * g * C);
        if (t0 + kStep <= end) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                x[j] = load_four<TR, WHOLE>(base + (off + (uint32_t)(j * C)), lcol, C);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (t0 + 8 * g + j < end) {
                    x[j] = load_four<TR, WHOLE>(base + (off + (uint32_t)(j * C)), lcol, C);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[j].e[i] = TR::from_f(0.f);
                }
            }
        }
    };
    constexpr int64_t kNext = WT * kStep;
    // Two steps in flight where there are registers for them.
    if constexpr (VT <= 2 || (VT <= 5 && (WHOLE || sizeof(typename TR::elem) == 2))) {
        int id0[8], id1[8];
        Four<TR> x0[8], x1[8];
        if (first < end) load(first, id0, x0);
        for (int64_t t0 = first; t0 < end; t0 += 2 * kNext) {
            if (t0 + kNext < end) load(t0 + kNext, id1, x1);
            hot_step<TR, VT>(id0, x0, r16, acc);
            if (t0 + kNext < end) {
                if (t0 + 2 * kNext < end) load(t0 + 2 * kNext, id0, x0);
                hot_step<TR, VT>(id1, x1, r16, acc);
            }
        }
    } else {
        for (int64_t t0 = first; t0 < end; t0 += kNext) {
            int id[8];
            Four<TR> x[8];
            load(t0, id, x);
            hot_step<TR, VT>(id, x, r16, acc);
        }
    }

    bool finite = true;
#pragma unroll
    for (int v = 0; v < VT; ++v)
#pragma unroll
        for (int ct = 0; ct < 4; ++ct)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                finite = finite && __builtin_fabsf(acc[v][ct][i]) < __builtin_inff();
    if (__any(!finite)) {
#pragma unroll
        for (int v = 0; v < VT; ++v)
#pragma unroll
            for (int ct = 0; ct < 4; ++ct) acc[v][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int64_t t0 = first; t0 < end; t0 += WT * kStep)
            for (int64_t t = t0; t < end && t < t0 + kStep; ++t) {
                const int id = hot_id(ids[t], v0);
                if (id < 0 || col >= C || ((id >> 2) & 3) != g) continue;
                const Four<TR> x = load_four<TR, WHOLE>(dout + (size_t)t * C, col, C);
#pragma unroll
                for (int v = 0; v < VT; ++v)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (id >> 4 == v && (id & 3) == i) {
#pragma unroll
                            for (int ct = 0; ct < 4; ++ct) acc[v][ct][i] += TR::to_f(x.e[ct]);
                        }
            }
    }

    // Join the waves of each column group, a tile of 16 rows at a time.
    float* to = out + (size_t)blockIdx.x * part_stride;
#pragma unroll
    for (int v = 0; v < VT; ++v) {
        if (v > 0) lds_barrier();
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<f32x4*>(&red[wave][4 * g + i][4 * r16]) =
                f32x4{acc[v][0][i], acc[v][1][i], acc[v][2][i], acc[v][3][i]};
        lds_barrier();
        constexpr int Q = kHotCols / 4 * WC;  // vectors of four columns in a row of the block
        for (int e = threadIdx.x; e < 16 * Q; e += 64 * kHotWaves) {
            const int row = e / Q, q = e % Q;
            const int wc = q / (kHotCols / 4), c4 = q % (kHotCols / 4) * 4;
            f32x4 sum = *reinterpret_cast<const f32x4*>(&red[wc][row][c4]);
#pragma unroll
            for (int w = 1; w < WT; ++w)
                sum += *reinterpret_cast<const f32x4*>(&red[w * WC + wc][row][c4]);
            if (v0 + 16 * v + row < V) {
                const float s4[4] = {sum[0] * scale, sum[1] * scale, sum[2] * scale,
                                     sum[3] * scale};
                store_floats<4>(to + (size_t)(v0 + 16 * v + row) * C, cbase + 4 * q, C, s4);
            }
        }
    }
}

// dtable = scale * the sum of the partials, n floats each, `stride` apart (a multiple of 4): a
// block takes 32 of them (one 128-byte line of every partial), 32 groups of 8 lanes the partials in
// turn.
__global__ __launch_bounds__(kThreads) void embed_parts_kernel(const float* __restrict__ parts,
                                                               size_t stride, int nparts,
                                                               float* __restrict__ dtable,
                                                               size_t n, float scale) {
    constexpr int U = 8, G = kThreads / 8;
    __shared__ __attribute__((aligned(16))) float red[G][36];
    const int q = threadIdx.x & 7, grp = threadIdx.x >> 3;
    const size_t at = (size_t)blockIdx.x * 32 + 4 * q;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (at < stride) {
        const float* p = parts + at;
        for (int b0 = grp; b0 < nparts; b0 += U * G) {
            f32x4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                v[u] = b0 + u * G < nparts
                           ? *reinterpret_cast<const f32x4*>(p + (size_t)(b0 + u * G) * stride)
                           : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < U; ++u) sum += v[u];
        }
    }
    *reinterpret_cast<f32x4*>(&red[grp][4 * q]) = sum;
    __syncthreads();
    const size_t mine = (size_t)blockIdx.x * 32 + threadIdx.x;
    if (threadIdx.x < 32 && mine < n) {
        float s = red[0][threadIdx.x];
#pragma unroll
        for (int i = 1; i < G; ++i) s += red[i][threadIdx.x];
        dtable[mine] = s * scale;
    }
}

__global__ __launch_bounds__(kThreads) void embed_zero_kernel(float* __restrict__ p, size_t n) {
    for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < n;
         i += (size_t)gridDim.x * kThreads)
        p[i] = 0.f;
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
// A launch holds fewer than 2^32 threads: kernels whose work can be more loop over it.
constexpr int64_t kMaxBlocks = 1 << 22;
size_t pad256(size_t n) { return (n + 255) & ~(size_t)255; }

// Lanes that take a row of nvec vectors in embed_sum_kernel: as many as it has, up to the 16 that
// read 256 bytes of it.
int lanes_a_row(int64_t nvec) { return nvec > 8 ? 16 : nvec > 4 ? 8 : nvec > 2 ? 4 : 2; }

// What the gradient keeps in its workspace, as offsets in bytes.
struct BwdPlan {
    // Tables of few rows: parts of `tokens` tokens, their partial sums `stride` floats apart.
    bool hot;
    int parts;
    int64_t tokens;
    size_t stride;
    // The others.
    bool ranked;
    int passes;
    int64_t tiles, chunks;
    size_t keys[2], order[2], counts, totals, head, tail, bytes;
};
// `half`: dout has a 16-bit type (its calls need no more workspace than float32 ones).
BwdPlan bwd_plan(int64_t M, int64_t V, int64_t C, bool half) {
    BwdPlan p = {};
    if (hot_table(M, V, C)) {
        // As many blocks as CUs, with at least two steps of tokens a wave; up to eight where one
        // block can then take all tokens and the partials' kernel is saved (not where float32 steps
        // of many rows take longer than it: 900 tokens of 129 rows of 256 columns 17 us in blocks,
        // 32 in one; 700 of 30 rows of 100 columns 13.5 and 11).
        p.hot = true;
        const int64_t others = up(C, C > kHotCols ? 2 * kHotCols : kHotCols) * up(V, kHotRows);
        const int64_t want = std::max<int64_t>(1, 256 / others);
        const int64_t round = kStep * (C > kHotCols ? kHotWaves / 2 : kHotWaves);
        const int64_t least = (half || V <= 32) && M <= 8 * round ? M : 2 * round;
        p.tokens = up(std::max(up(M, want), std::min(M, least)), kStep) * kStep;
        p.parts = (int)up(M, p.tokens);
        p.stride = (size_t)up(V * C, 4) * 4;
        p.bytes = p.parts > 1 ? p.parts * p.stride * sizeof(float) : 16;
        return p;
    }
    p.ranked = M <= kRankMax;
    p.passes = 1;
    while ((V >> (8 * p.passes)) != 0) ++p.passes;  // keys are 0 .. V
    p.tiles = up(M, kTile);
    p.chunks = up(M, kThreads / lanes_a_row(up(C, 4)) * kRun);  // float32 rows have the most
    size_t at = 0;
    const auto take = [&](size_t n) {
        const size_t here = at;
        at += pad256(n);
        return here;
    };
    const int copies = p.ranked || p.passes == 1 ? 1 : 2;
    for (int i = 0; i < copies; ++i) {
        p.keys[i] = take((size_t)M * 4);
        p.order[i] = take((size_t)M * 4);
    }
    if (!p.ranked) {
        p.counts = take((size_t)p.tiles * kDigits * 4);
        p.totals = take(kDigits * 4);
    }
    p.head = take((size_t)p.chunks * C * 4);
    p.tail = take((size_t)p.chunks * C * 4);
    p.bytes = at;
    return p;
}

clk_status validate(const char* who, clk_dtype dtype, clk_dtype ids_dtype, int64_t M, int64_t V,
                    int64_t C) {
    if (dtype != CLK_F16 && dtype != CLK_BF16 && dtype != CLK_F32)
        return fail(CLK_INVALID_ARGUMENT, "%s: dtype %s not supported (f16, bf16, f32)", who,
                    dtype_name(dtype));
    if (ids_dtype != CLK_S32 && ids_dtype != CLK_S64)
        return fail(CLK_INVALID_ARGUMENT, "%s: ids of type %s not supported (s32, s64)", who,
                    dtype_name(ids_dtype));
    if (M < 0 || V < 0 || C <= 0)
        return fail(CLK_INVALID_ARGUMENT, "%s: ids [M], table [V,C] with C > 0 expected", who);
    // These keep token, row and chunk numbers in 31 bits and a launch's threads in 32.
    if (M > (1 << 30) || V > (1 << 30) - 1 || C > (1 << 20) || M * C > ((int64_t)1 << 37) ||
        V * C > ((int64_t)1 << 37))
        return fail(CLK_INVALID_ARGUMENT, "%s: M=%lld, [V,C] = [%lld,%lld] too large", who,
                    (long long)M, (long long)V, (long long)C);
    return CLK_OK;
}

template <typename TR, typename ID>
void launch_fwd(hipStream_t st, const void* table, const void* ids, void* out, int64_t M,
                int64_t V, int64_t C, float scale) {
    using E = typename TR::elem;
    constexpr int N = Vec<TR>::N;
    const bool whole = C % N == 0;
    const int64_t nvec = up(C, N);
    // About four vectors a thread.
    const int rows = (int)std::max<int64_t>(1, 4 * kThreads / nvec);
    const int grid = (int)std::min<int64_t>(up(M, rows), kMaxBlocks);
    KernelTimer timer("embedding", st);
    const auto kernel = whole ? embed_kernel<TR, ID, true> : embed_kernel<TR, ID, false>;
    kernel<<<grid, kThreads, 0, st>>>(static_cast<const E*>(table), static_cast<const ID*>(ids),
                                      static_cast<E*>(out), M, V, (int)C, rows,
                                      fast_div((uint32_t)nvec), scale);
}

template <typename ID>
void sort_tokens(hipStream_t st, const ID* ids, float* dtable, char* ws, const BwdPlan& p,
                 int64_t M, int64_t V, int64_t C, uint32_t** keys, uint32_t** order) {
    const auto at = [&](size_t off) { return reinterpret_cast<uint32_t*>(ws + off); };
    // Part k of the zeros, behind `first` other blocks: 16 KB a block, up to 8192 blocks.
    const size_t n = (size_t)V * C;
    const int parts = p.ranked ? 1 : 2 * p.passes;
    const auto zero = [&](int k, int64_t first) {
        const size_t beg = n / 4 * k / parts * 4, end = k + 1 == parts ? n : n / 4 * (k + 1) / parts * 4;
        return Zero{dtable, beg, end, (int)first, (int)std::min<int64_t>(up(end - beg, 4096), 8192)};
    };
    *keys = at(p.keys[0]);
    *order = at(p.order[0]);
    if (p.ranked) {
        const Zero z = zero(0, up(M, kRankTokens));
        KernelTimer timer("embedding_bwd_rank", st);
        embed_rank_kernel<ID><<<z.first + z.blocks, kThreads, 0, st>>>(ids, (int)M, (uint32_t)V,
                                                                       *keys, *order, z);
        return;
    }
    const bool few = p.tiles <= kFewTiles;
    const Counts counts = {at(p.counts), p.tiles, few ? 1 : (size_t)p.tiles, few ? kDigits : (size_t)1};
    for (int pass = 0; pass < p.passes; ++pass) {
        uint32_t *to_keys = at(p.keys[pass & 1]), *to_order = at(p.order[pass & 1]);
        const auto run = [&](auto src) {
            KernelTimer timer("embedding_bwd_sort", st);
            Zero z = zero(2 * pass, p.tiles);
            embed_count_kernel<<<z.first + z.blocks, kThreads, 0, st>>>(src, M, 8 * pass, counts,
                                                                        z);
            if (!few) embed_scan_kernel<<<kDigits, kThreads, 0, st>>>(counts, at(p.totals));
            z = zero(2 * pass + 1, p.tiles);
            embed_scatter_kernel<<<z.first + z.blocks, kThreads, 0, st>>>(
                src, M, 8 * pass, counts, few ? nullptr : at(p.totals), to_keys, to_order, z);
        };
        if (pass == 0) run(FirstKeys<ID>{ids, (uint32_t)V});
        else run(NextKeys{*keys, *order});
        *keys = to_keys;
        *order = to_order;
    }
}

template <typename TR, int LPR>
void launch_sum(hipStream_t st, const void* dout, const uint32_t* keys, const uint32_t* order,
                float* dtable, char* ws, const BwdPlan& p, int64_t M, int64_t V, int64_t C,
                float scale) {
    using E = typename TR::elem;
    constexpr int N = Vec<TR>::N;
    const auto kernel = C % N == 0 ? embed_sum_kernel<TR, LPR, true>
                                   : embed_sum_kernel<TR, LPR, false>;
    constexpr int tokens = chunk_tokens<LPR>();
    const int64_t chunks = up(M, tokens), slices = up(up(C, N), LPR);
    float* head = reinterpret_cast<float*>(ws + p.head);
    float* tail = reinterpret_cast<float*>(ws + p.tail);
    {
        KernelTimer timer("embedding_bwd_sum", st);
        kernel<<<(uint32_t)(chunks * slices), kThreads, 0, st>>>(
            static_cast<const E*>(dout), keys, order, dtable, head, tail, (uint32_t)M, (uint32_t)V,
            (int)C, fast_div((uint32_t)slices), scale);
    }
    if (chunks == 1) return;
    const int64_t join_slices = up(C, 256);
    KernelTimer timer("embedding_bwd_join", st);
    embed_join_kernel<<<(uint32_t)((chunks - 1) * join_slices), kThreads, 0, st>>>(
        keys, head, tail, dtable, (uint32_t)V, (int)C, (uint32_t)chunks, tokens,
        fast_div((uint32_t)join_slices), scale);
}

template <typename TR, typename ID, int VT, int WC, bool WHOLE>
void launch_hot(hipStream_t st, const void* dout, const void* ids, float* dtable, char* ws,
                const BwdPlan& p, int64_t M, int64_t V, int64_t C, float scale) {
    using E = typename TR::elem;
    float* parts = reinterpret_cast<float*>(ws);
    {
        KernelTimer timer("embedding_bwd_hot", st);
        embed_hot_kernel<TR, ID, VT, WC, WHOLE>
            <<<dim3(p.parts, (uint32_t)up(C, kHotCols * WC), (uint32_t)up(V, kHotRows)),
               64 * kHotWaves, 0, st>>>(
                static_cast<const E*>(dout), static_cast<const ID*>(ids),
                p.parts > 1 ? parts : dtable, p.stride, M, (int)V, (int)C, p.tokens,
                p.parts > 1 ? 1.f : scale);
    }
    if (p.parts > 1) {
        KernelTimer timer("embedding_bwd_parts", st);
        embed_parts_kernel<<<(uint32_t)up(V * C, 32), kThreads, 0, st>>>(
            parts, p.stride, p.parts, dtable, (size_t)V * C, scale);
    }
}

template <typename TR, typename ID>
void launch_bwd(hipStream_t st, const void* dout, const void* ids, float* dtable, char* ws,
                int64_t M, int64_t V, int64_t C, float scale) {
    constexpr int N = Vec<TR>::N;
    const BwdPlan p = bwd_plan(M, V, C, sizeof(typename TR::elem) == 2);
    if (p.hot) {
        const auto pick = [&](auto vt, auto wc) {
            constexpr int VT = decltype(vt)::value, WC = decltype(wc)::value;
            return C % 4 == 0 ? launch_hot<TR, ID, VT, WC, true> : launch_hot<TR, ID, VT, WC, false>;
        };
        const auto rows = [&](auto wc) {
            return V <= 32   ? pick(std::integral_constant<int, 2>(), wc)
                   : V <= 80 ? pick(std::integral_constant<int, 5>(), wc)
                             : pick(std::integral_constant<int, kHotRows / 16>(), wc);
        };
        const auto run = C > kHotCols ? rows(std::integral_constant<int, 2>())
                                      : rows(std::integral_constant<int, 1>());
        run(st, dout, ids, dtable, ws, p, M, V, C, scale);
        return;
    }
    uint32_t *keys = nullptr, *order = nullptr;
    sort_tokens<ID>(st, static_cast<const ID*>(ids), dtable, ws, p, M, V, C, &keys, &order);
    const int lanes = lanes_a_row(up(C, N));
    const auto sum = lanes == 16  ? launch_sum<TR, 16>
                     : lanes == 8 ? launch_sum<TR, 8>
                     : lanes == 4 ? launch_sum<TR, 4>
                                  : launch_sum<TR, 2>;
    sum(st, dout, keys, order, dtable, ws, p, M, V, C, scale);
}

// fn<TR, ID> for the two types of a call.
#define CLK_EMBED_TYPES(dtype, ids_dtype, fn, ...)                          \
    do {                                                                    \
        const bool wide = (ids_dtype) == CLK_S64;                           \
        if ((dtype) == CLK_BF16)                                            \
            wide ? fn<BF16, int64_t>(__VA_ARGS__) : fn<BF16, int32_t>(__VA_ARGS__); \
        else if ((dtype) == CLK_F16)                                        \
            wide ? fn<F16, int64_t>(__VA_ARGS__) : fn<F16, int32_t>(__VA_ARGS__);   \
        else                                                                \
            wide ? fn<F32, int64_t>(__VA_ARGS__) : fn<F32, int32_t>(__VA_ARGS__);   \
    } while (0)

}  // namespace
}  // namespace clk

using namespace clk;

extern "C" clk_status clk_embedding_fwd(hipStream_t stream, clk_dtype dtype, const void* table,
                                        clk_dtype ids_dtype, const void* ids, void* out,
                                        int64_t M, int64_t V, int64_t C, float scale) {
    const char* who = "embedding";
    const clk_status s = validate(who, dtype, ids_dtype, M, V, C);
    if (s != CLK_OK) return s;
    if (M == 0) return ok();
    if ((V > 0 && !table) || !ids || !out)
        return fail(CLK_INVALID_ARGUMENT, "%s: null pointer", who);
    if (!aligned16(table) || !aligned16(out))
        return fail(CLK_INVALID_ARGUMENT, "%s: table and out must be 16-byte aligned", who);
    const size_t elem = dtype == CLK_F32 ? 4 : 2, id = ids_dtype == CLK_S64 ? 8 : 4;
    if (overlap(out, M * C * elem, table, V * C * elem) || overlap(out, M * C * elem, ids, M * id))
        return fail(CLK_INVALID_ARGUMENT, "%s: out may not overlap table or ids", who);
    CLK_EMBED_TYPES(dtype, ids_dtype, launch_fwd, stream, table, ids, out, M, V, C, scale);
    return check_launch(who);
}

extern "C" size_t clk_embedding_bwd_workspace_size(int64_t M, int64_t V, int64_t C) {
    if (M <= 0 || V <= 0 || C <= 0 || validate("embedding_bwd", CLK_F32, CLK_S32, M, V, C) != CLK_OK)
        return 0;
    return bwd_plan(M, V, C, false).bytes;
}

extern "C" clk_status clk_embedding_bwd(hipStream_t stream, clk_dtype dtype, const void* dout,
                                        clk_dtype ids_dtype, const void* ids, float* dtable,
                                        void* workspace, size_t workspace_bytes, int64_t M,
                                        int64_t V, int64_t C, float scale) {
    const char* who = "embedding_bwd";
    const clk_status s = validate(who, dtype, ids_dtype, M, V, C);
    if (s != CLK_OK) return s;
    if (V == 0) return ok();
    if (!dtable || (M > 0 && (!dout || !ids || !workspace)))
        return fail(CLK_INVALID_ARGUMENT, "%s: null pointer", who);
    if (M == 0) {  // no tokens: the gradient is zero
        const size_t n = (size_t)V * C;
        embed_zero_kernel<<<(int)std::min<size_t>((n + kThreads - 1) / kThreads, 4096), kThreads,
                            0, stream>>>(dtable, n);
        return check_launch(who);
    }
    if (!aligned16(dout) || !aligned16(dtable) || !aligned16(workspace))
        return fail(CLK_INVALID_ARGUMENT,
                    "%s: dout, dtable and workspace must be 16-byte aligned", who);
    const size_t need = clk_embedding_bwd_workspace_size(M, V, C);
    if (workspace_bytes < need)
        return fail(CLK_INVALID_ARGUMENT, "%s: workspace %zu bytes, needs %zu", who,
                    workspace_bytes, need);
    const size_t in = M * C * (dtype == CLK_F32 ? 4 : 2), id = M * (ids_dtype == CLK_S64 ? 8 : 4);
    if (overlap(dtable, V * C * 4, dout, in) || overlap(dtable, V * C * 4, ids, id) ||
        overlap(workspace, need, dout, in) || overlap(workspace, need, ids, id) ||
        overlap(workspace, need, dtable, V * C * 4))
        return fail(CLK_INVALID_ARGUMENT, "%s: dout, ids, dtable and workspace may not overlap",
                    who);
    CLK_EMBED_TYPES(dtype, ids_dtype, launch_bwd, stream, dout, ids, dtable,
                    static_cast<char*>(workspace), M, V, C, scale);
    return check_launch(who);
}
