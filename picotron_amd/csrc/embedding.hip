// Scaled token embedding and its gradient by sorted tokens.
//
//   forward   out[t, :]  = scale * W[ids[t], :]                      one rounding, at the store
//   backward  dW[v, :]   = scale * sum over t with ids[t] = v of dOut[t, :]     (0 for a row nobody looked up)
//
// Both are bound by memory: the forward reads and writes one row per token, the backward reads one row per token and writes
// the whole table once.  The sums must not depend on the order in which blocks run, so nothing is added with atomics: the
// tokens are sorted by id with a stable radix sort (digits of up to 9 bits; up to kSmall tokens in the LDS of one block, more with
// two launches per digit), every table row then owns a run of the sorted order and is summed in token order, in fp32, and rounded
// once.  Frequent tokens would leave one block with thousands of rows: runs longer than kChunk are cut at the multiples of kChunk
// of the sorted order, the pieces are summed by blocks of their own into fp32 partial rows and joined in order by a last launch.
// Measured, bf16: 32768 tokens, table 131072 x 4096: forward 93 us (537 MB: 5.8 TB/s), sort 23, sums 286 (1.34 GB: 4.7 TB/s), join 16;
// 8192 tokens, table 32000 x 2048: 11, 21, 44 (165 MB: 3.8 TB/s) and 6.  The sorts are chains of short steps that wait for each other,
// not bytes.
#include "lds.h"

namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------------------------------------------
// 16-byte chunks (or single elements where a row is no whole number of them) as floats
// ---------------------------------------------------------------------------------------------------------------
template <typename T, bool WIDE>
struct Row;

template <>
struct Row<__bf16, true> {
    static constexpr int kVec = 8;
    typedef u32x4_t raw;
    __device__ static void unpack(const raw& r, float (&f)[kVec]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    __device__ static raw pack(const float (&f)[kVec]) {
        return raw{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
    }
};
template <>
struct Row<float, true> {
    static constexpr int kVec = 4;
    typedef f32x4_t raw;
    __device__ static void unpack(const raw& r, float (&f)[kVec]) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) f[i] = r[i];
    }
    __device__ static raw pack(const float (&f)[kVec]) { return raw{f[0], f[1], f[2], f[3]}; }
};
template <>
struct Row<__bf16, false> {
    static constexpr int kVec = 1;
    typedef uint16_t raw;
    __device__ static void unpack(const raw& r, float (&f)[1]) { f[0] = bf16_bits_to_f32(r); }
    __device__ static raw pack(const float (&f)[1]) { return (raw)f32_to_bf16_bits(f[0]); }
};
template <>
struct Row<float, false> {
    static constexpr int kVec = 1;
    typedef float raw;
    __device__ static void unpack(const raw& r, float (&f)[1]) { f[0] = r; }
    __device__ static raw pack(const float (&f)[1]) { return f[0]; }
};

// ---------------------------------------------------------------------------------------------------------------
// Forward: the chunks of all output rows in one line, kFwdChunks per thread, kThreads apart.
// ---------------------------------------------------------------------------------------------------------------
constexpr int kFwdChunks = 4;

template <typename R>
__global__ __launch_bounds__(kThreads) void embedding_fwd_kernel(const typename R::raw* __restrict__ weight, int64_t vocab, uint32_t row_chunks,
                                                                 const int64_t* __restrict__ ids, int64_t n_tokens, float scale,
                                                                 typename R::raw* __restrict__ out) {
    // the block's first chunk in 64 bits, the rest of the arithmetic relative to it
    const int64_t first = (int64_t)blockIdx.x * (kThreads * kFwdChunks);
    const int64_t row0 = first / row_chunks;
    const uint32_t col0 = (uint32_t)(first - row0 * row_chunks);
    typename R::raw v[kFwdChunks];
    bool in[kFwdChunks], good[kFwdChunks];
#pragma unroll
    for (int c = 0; c < kFwdChunks; ++c) {
        const uint32_t at = col0 + c * kThreads + threadIdx.x, down = at / row_chunks, col = at - down * row_chunks;
        in[c] = row0 + down < n_tokens;
        const int64_t id = in[c] ? ids[row0 + down] : -1;
        good[c] = id >= 0 && id < vocab;
        if (good[c]) v[c] = weight[id * (int64_t)row_chunks + col];
    }
#pragma unroll
    for (int c = 0; c < kFwdChunks; ++c) {
        if (!in[c]) continue;
        float f[R::kVec];
        if (good[c]) R::unpack(v[c], f);
#pragma unroll
        for (int i = 0; i < R::kVec; ++i) f[i] = good[c] ? f[i] * scale : __builtin_nanf("");
        out[first + c * kThreads + threadIdx.x] = R::pack(f);
    }
}

// ---------------------------------------------------------------------------------------------------------------
// Stable radix sort of (id, token) by id.  Ids outside the table and the padding id become the key `vocab`, which sorts
// behind every row.  A block ranks 1024 * ROUNDS tokens, a wave 64 * ROUNDS consecutive ones of them.
// ---------------------------------------------------------------------------------------------------------------
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kMaxDigitBits = 9, kMaxDigits = 1 << kMaxDigitBits;
constexpr int kSmallRounds = 8, kSmall = kSortThreads * kSmallRounds;

__device__ __forceinline__ uint32_t id_key(int64_t id, int64_t vocab, int64_t padding) {
    return id < 0 || id >= vocab || id == padding ? (uint32_t)vocab : (uint32_t)id;
}

struct SortPass {
    const int64_t* ids;    // first pass: the tokens' ids ...
    const uint32_t* keys;  // ... later ones: keys and tokens as the pass before left them
    const int32_t* vals;
    uint32_t* keys_out;
    int32_t* vals_out;
    int32_t* hist;  // [blocks][digits]
    int64_t n, vocab, padding;
    int shift, bits;
};

__device__ __forceinline__ uint32_t load_key(const SortPass& p, int64_t i) {
    return p.ids ? id_key(p.ids[i], p.vocab, p.padding) : p.keys[i];
}

// LDS accesses of one wavefront execute in order; this keeps the compiler from moving them
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// the rank of a lane's token among the wave's tokens of its digit: those counted in `seen` so far and those of lanes below
__device__ __forceinline__ int32_t wave_rank(int32_t* seen, uint32_t digit, int bits, bool in, int lane) {
    uint64_t same = __ballot(in);
    if (!in) same = ~same;
    for (int bit = 0; bit < bits; ++bit) {
        const bool set = (digit >> bit) & 1u;
        const uint64_t with = __ballot(set);
        same &= set ? with : ~with;
    }
    const int below = __popcll(same & ((1ull << lane) - 1));
    const int32_t had = in ? seen[digit] : 0;
    wave_sync();  // every lane has read the count before the first of its peers moves it on, ...
    if (in && below == 0) seen[digit] = had + __popcll(same);
    wave_sync();  // ... and it has moved before the next round reads it
    return had + below;
}

// exclusive sums of `v` over the first `digits` threads of the block
__device__ __forceinline__ int32_t block_scan(int32_t v, int32_t* wave_total, int lane, int wave) {
    int32_t scan = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int32_t o = __shfl_up(scan, off, 64);
        if (lane >= off) scan += o;
    }
    if (lane == 63) wave_total[wave] = scan;
    __syncthreads();
    int32_t before = scan - v;
    for (int w = 0; w < wave; ++w) before += wave_total[w];
    return before;
}

// Up to kSmall tokens: every pass in one block, keys and tokens in LDS between the passes.
__global__ __launch_bounds__(kSortThreads) void sort_small_kernel(SortPass p, int passes) {
    extern __shared__ int32_t lds[];
    uint32_t* keys = (uint32_t*)lds;                 // [kSmall]
    int32_t* vals = lds + kSmall;                    // [kSmall]
    int32_t* seen_all = lds + 2 * kSmall;            // [waves][digits]
    int32_t* wave_total = seen_all + kSortWaves * kMaxDigits;
    const int digits = 1 << p.bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rounds = (int)((p.n + kSortThreads - 1) / kSortThreads);
    int32_t* seen = seen_all + wave * kMaxDigits;
    uint32_t key[kSmallRounds];
    int32_t val[kSmallRounds], rank[kSmallRounds];
    for (int pass = 0; pass < passes; ++pass) {
        for (int d = lane; d < digits; d += 64) seen[d] = 0;
        wave_sync();
#pragma unroll
        for (int r = 0; r < kSmallRounds; ++r) {
            if (r >= rounds) break;
            const int i = wave * (64 * rounds) + r * 64 + lane;
            const bool in = i < p.n;
            key[r] = in ? (pass == 0 ? id_key(p.ids[i], p.vocab, p.padding) : keys[i]) : 0xFFFFFFFFu;
            val[r] = in ? (pass == 0 ? i : vals[i]) : -1;
            rank[r] = wave_rank(seen, (key[r] >> (pass * p.bits)) & (uint32_t)(digits - 1), p.bits, in, lane);
        }
        __syncthreads();
        int32_t all = 0;  // thread d: the waves' counts of digit d become what comes before each wave's tokens
        if ((int)threadIdx.x < digits) {
            for (int w = 0; w < kSortWaves; ++w) {
                const int32_t c = seen_all[w * kMaxDigits + threadIdx.x];
                seen_all[w * kMaxDigits + threadIdx.x] = all;
                all += c;
            }
        }
        const int32_t base = block_scan(all, wave_total, lane, wave);
        if ((int)threadIdx.x < digits)
            for (int w = 0; w < kSortWaves; ++w) seen_all[w * kMaxDigits + threadIdx.x] += base;
        __syncthreads();
        const bool last = pass == passes - 1;
#pragma unroll
        for (int r = 0; r < kSmallRounds; ++r) {
            if (r >= rounds || val[r] < 0) continue;
            const int to = seen[(key[r] >> (pass * p.bits)) & (uint32_t)(digits - 1)] + rank[r];
            (last ? p.keys_out : keys)[to] = key[r];
            (last ? p.vals_out : vals)[to] = val[r];
        }
        __syncthreads();
    }
}

template <int ROUNDS>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(SortPass p) {
    __shared__ int32_t count[kMaxDigits];
    const int digits = 1 << p.bits;
    for (int d = threadIdx.x; d < digits; d += kSortThreads) count[d] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int64_t i = (int64_t)blockIdx.x * (kSortThreads * ROUNDS) + r * kSortThreads + threadIdx.x;
        if (i < p.n) atomicAdd(&count[(load_key(p, i) >> p.shift) & (digits - 1)], 1);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kSortThreads) p.hist[(int64_t)blockIdx.x * digits + d] = count[d];
}

template <int ROUNDS>
__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(SortPass p) {
    __shared__ int32_t base[kMaxDigits];                // where the block's first token of a digit goes
    __shared__ int32_t seen[kSortWaves][kMaxDigits];    // tokens of a digit that a wave has ranked; then: those of the waves before
    __shared__ int32_t wave_total[kSortWaves];
    const int digits = 1 << p.bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = lane; d < digits; d += 64) seen[wave][d] = 0;
    wave_sync();

    // tokens of the same digit in all blocks and in earlier ones
    int32_t all = 0, before = 0;
    if ((int)threadIdx.x < digits) {
#pragma unroll 8
        for (int b = 0; b < (int)gridDim.x; ++b) {
            const int32_t c = p.hist[(int64_t)b * digits + threadIdx.x];
            all += c;
            before += b < (int)blockIdx.x ? c : 0;
        }
    }
    const int32_t smaller = block_scan(all, wave_total, lane, wave);
    if ((int)threadIdx.x < digits) base[threadIdx.x] = smaller + before;

    uint32_t key[ROUNDS];
    int32_t val[ROUNDS], rank[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int64_t i = (int64_t)blockIdx.x * (kSortThreads * ROUNDS) + wave * (64 * ROUNDS) + r * 64 + lane;
        const bool in = i < p.n;
        key[r] = in ? load_key(p, i) : 0xFFFFFFFFu;
        val[r] = in ? (p.ids ? (int32_t)i : p.vals[i]) : -1;
        rank[r] = wave_rank(seen[wave], (key[r] >> p.shift) & (uint32_t)(digits - 1), p.bits, in, lane);
    }
    __syncthreads();
    if ((int)threadIdx.x < digits) {
        int32_t sum = 0;
        for (int w = 0; w < kSortWaves; ++w) {
            const int32_t c = seen[w][threadIdx.x];
            seen[w][threadIdx.x] = sum;
            sum += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        if (val[r] < 0) continue;
        const uint32_t digit = (key[r] >> p.shift) & (uint32_t)(digits - 1);
        const int64_t to = (int64_t)base[digit] + seen[wave][digit] + rank[r];
        p.keys_out[to] = key[r];
        p.vals_out[to] = val[r];
    }
}

// ---------------------------------------------------------------------------------------------------------------
// Sums over the runs of the sorted order
// ---------------------------------------------------------------------------------------------------------------
constexpr int kChunk = 64;       // longest run that one group sums in one go, and the piece of a longer one
// table rows that a group of threads walks; with 4 the lookups in front of them cost 14 % at 131072 x 4096, with 16 and 32 the few blocks
// of a small table (5003 x 200) take 11 and 15 us instead of 9
constexpr int kRowsPerGroup = 8;

struct SumArgs {
    const uint32_t* keys;  // sorted
    const int32_t* vals;
    int64_t n, vocab;
    uint32_t row_chunks;
    float scale;
    float* partial;  // [chunks][2][row_chunks * kVec]: the sums of the runs that hold a chunk's first and last position
};

// The first of the sorted keys from `lo` on that is at least `key`, looked up by a wavefront: 64 places are probed at a time, so that
// a lookup among n keys waits for log64(n) loads in a row, not log2(n).
__device__ __forceinline__ int64_t first_at_least(const uint32_t* __restrict__ keys, int64_t lo, int64_t n, uint32_t key) {
    const int lane = threadIdx.x & 63;
    int64_t hi = n;  // the answer is in [lo, hi]
    while (hi > lo) {
        const int64_t step = (hi - lo + 63) / 64, at = lo + lane * step;
        const uint64_t less = __ballot(at < hi && keys[at < hi ? at : lo] < key);  // a prefix of the lanes
        const int k = __popcll(less);
        if (k == 0) return lo;
        if (step == 1) return lo + k;
        const int64_t from = lo + (int64_t)(k - 1) * step + 1;  // behind the last probe that is less, up to the next one
        hi = lo + k * step < hi ? lo + k * step : hi;
        lo = from;
    }
    return lo;
}

// adds the rows of places [from, to) of the sorted order; token(i): the token at place i, the same in every lane
template <typename R, typename F>
__device__ __forceinline__ void add_rows(const typename R::raw* __restrict__ d_out, const SumArgs& a, int64_t from, int64_t to, uint32_t col, F token,
                                         float (&sum)[R::kVec]) {
    constexpr int kAhead = 8;
    for (int64_t i = from; i < to; i += kAhead) {
        typename R::raw v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (i + u < to) v[u] = d_out[(int64_t)token(i + u) * a.row_chunks + col];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (i + u >= to) continue;
            float f[R::kVec];
            R::unpack(v[u], f);
#pragma unroll
            for (int e = 0; e < R::kVec; ++e) sum[e] += f[e];
        }
    }
}

// kVec fp32 sums of a partial row
template <typename R>
__device__ __forceinline__ void load_sums(const float* slot, float (&f)[R::kVec]) {
    if constexpr (R::kVec >= 4) {
#pragma unroll
        for (int i = 0; i < R::kVec; i += 4) {
            const f32x4_t v = *(const f32x4_t*)(slot + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) f[i + j] = v[j];
        }
    } else {
        f[0] = slot[0];
    }
}

// Groups of `group` threads (64 or 256) hold the columns of a row, blockIdx.y steps over wider rows.  The first
// chunk_blocks blocks sum the pieces of the runs longer than kChunk, which take the longest, the others write the table rows of the
// shorter ones.
template <typename R>
__global__ __launch_bounds__(kThreads) void sum_runs_kernel(const typename R::raw* __restrict__ d_out, SumArgs a, int group, int64_t chunk_blocks,
                                                            typename R::raw* __restrict__ d_weight) {
    const int groups = kThreads / group, g = threadIdx.x / group;
    const uint32_t col = blockIdx.y * group + threadIdx.x % group;
    const int lane = threadIdx.x & 63;
    if (blockIdx.x >= chunk_blocks) {
        const int64_t row0 = (((int64_t)blockIdx.x - chunk_blocks) * groups + g) * kRowsPerGroup;
        if (row0 >= a.vocab) return;
        // the sorted keys and their tokens from `window` on, one a lane
        int64_t at = first_at_least(a.keys, 0, a.n, (uint32_t)row0), window = at;
        uint32_t ahead = window + lane < a.n ? a.keys[window + lane] : 0xFFFFFFFFu;
        int32_t tokens = window + lane < a.n ? a.vals[window + lane] : 0;
        for (int r = 0; r < kRowsPerGroup; ++r) {
            const uint32_t row = (uint32_t)row0 + r;
            if (row >= a.vocab) break;
            const int64_t from = at;
            const uint64_t behind = __ballot(ahead > row);
            float sum[R::kVec] = {};
            if (behind) {
                at = window + (__ffsll((unsigned long long)behind) - 1);
                if (col < a.row_chunks)
                    add_rows<R>(d_out, a, from, at, col,
                                [&](int64_t i) { return __builtin_amdgcn_readlane(tokens, __builtin_amdgcn_readfirstlane((int)(i - window))); }, sum);
            } else {
                at = window = first_at_least(a.keys, window + 64, a.n, row + 1);
                ahead = window + lane < a.n ? a.keys[window + lane] : 0xFFFFFFFFu;
                tokens = window + lane < a.n ? a.vals[window + lane] : 0;
                if (at - from > kChunk) continue;
                if (col < a.row_chunks) add_rows<R>(d_out, a, from, at, col, [&](int64_t i) { return a.vals[i]; }, sum);
            }
            if (col >= a.row_chunks) continue;
#pragma unroll
            for (int e = 0; e < R::kVec; ++e) sum[e] *= a.scale;
            d_weight[(int64_t)row * a.row_chunks + col] = R::pack(sum);
        }
        return;
    }
    const int64_t chunk = (int64_t)blockIdx.x * groups + g, begin = chunk * kChunk;
    if (begin >= a.n) return;
    const int64_t end = begin + kChunk < a.n ? begin + kChunk : a.n;
    const uint32_t mine = a.keys[begin + lane < end ? begin + lane : end - 1];  // kChunk is a wavefront's width
    const int32_t tokens = a.vals[begin + lane < end ? begin + lane : end - 1];
    const uint32_t key0 = __builtin_amdgcn_readfirstlane(mine), key1 = __builtin_amdgcn_readlane(mine, 63);
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const uint32_t key = side ? key1 : key0;
        if (key >= a.vocab || (side && key1 == key0)) continue;
        const int64_t from = first_at_least(a.keys, 0, a.n, key), to = first_at_least(a.keys, from, a.n, key + 1);
        if (to - from <= kChunk || col >= a.row_chunks) continue;
        float sum[R::kVec] = {};
        add_rows<R>(d_out, a, from > begin ? from : begin, to < end ? to : end, col,
                    [&](int64_t i) { return __builtin_amdgcn_readlane(tokens, __builtin_amdgcn_readfirstlane((int)(i - begin))); }, sum);
        float* slot = a.partial + ((chunk * 2 + side) * (int64_t)a.row_chunks + col) * R::kVec;
#pragma unroll
        for (int e = 0; e < R::kVec; ++e) slot[e] = sum[e];
    }
}

// One group per chunk: where a run longer than kChunk begins in it, the run's pieces are added in order.
template <typename R>
__global__ __launch_bounds__(kThreads) void join_runs_kernel(SumArgs a, int group, typename R::raw* __restrict__ d_weight) {
    const int groups = kThreads / group, g = threadIdx.x / group;
    const uint32_t col = blockIdx.y * group + threadIdx.x % group;
    const int64_t chunk = (int64_t)blockIdx.x * groups + g, begin = chunk * kChunk;
    if (begin >= a.n) return;
    const int64_t end = begin + kChunk < a.n ? begin + kChunk : a.n;
    // a run that begins here and is longer than a chunk holds the chunk's last position
    const uint32_t key = a.keys[end - 1];
    if (key >= a.vocab || (begin > 0 && a.keys[begin - 1] == key)) return;
    const int64_t from = first_at_least(a.keys, begin, a.n, key), to = first_at_least(a.keys, from, a.n, key + 1);
    if (to - from <= kChunk) return;
    if (col >= a.row_chunks) return;
    float sum[R::kVec] = {};
    const int64_t last = (to - 1) / kChunk;
    constexpr int kAhead = 8;
    for (int64_t c0 = chunk; c0 <= last; c0 += kAhead) {
        float v[kAhead][R::kVec];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int64_t c = c0 + u < last ? c0 + u : last;
            const int side = c == chunk && from > begin;
            load_sums<R>(a.partial + ((c * 2 + side) * (int64_t)a.row_chunks + col) * R::kVec, v[u]);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int e = 0; e < R::kVec; ++e) sum[e] += c0 + u <= last ? v[u][e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < R::kVec; ++e) sum[e] *= a.scale;
    d_weight[(int64_t)key * a.row_chunks + col] = R::pack(sum);
}

// ---------------------------------------------------------------------------------------------------------------
int key_bits(int64_t vocab) {
    int bits = 1;
    while (((int64_t)1 << bits) <= vocab) ++bits;  // keys 0 .. vocab
    return bits;
}

bool sizes_fit(int dtype, int64_t n_tokens, int64_t vocab, int64_t hidden) {
    return (dtype == PICOMOE_F32 || dtype == PICOMOE_BF16) && n_tokens >= 0 && n_tokens < (1ll << 31) - (1 << 16) && vocab >= 1 && vocab < (1ll << 31) &&
           hidden >= 1 && hidden <= (1 << 20);
}

int64_t round16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

// Every block of a scatter reads all blocks' counts, so blocks are few: 64 up to a million tokens; below that, rounds are few
int sort_rounds(int64_t n) { return n <= 64 * kSortThreads ? 1 : (n <= 256 * kSortThreads ? 4 : 16); }
int64_t sort_blocks(int64_t n) { return (n + sort_rounds(n) * kSortThreads - 1) / (sort_rounds(n) * kSortThreads); }

struct BwdLayout {
    int64_t keys[2], vals[2], hist, partial, bytes;
};
BwdLayout bwd_layout(int64_t n, int64_t hidden) {
    BwdLayout l;
    int64_t at = 0;
    for (int i = 0; i < 2; ++i) {
        l.keys[i] = at;
        at += round16(n * 4);
        l.vals[i] = at;
        at += round16(n * 4);
    }
    l.hist = at;
    at += n > kSmall ? sort_blocks(n) * kMaxDigits * 4 : 0;
    l.partial = at;
    at += (n + kChunk - 1) / kChunk * 2 * hidden * 4;
    l.bytes = round16(at);
    return l;
}

bool wide_rows(int dtype, int64_t hidden, const void* a, const void* b) {
    return hidden * (dtype == PICOMOE_BF16 ? 2 : 4) % 16 == 0 && (((uintptr_t)a | (uintptr_t)b) & 15) == 0;
}

template <typename R>
int launch_fwd(const void* weight, int64_t vocab, int64_t hidden, const int64_t* ids, int64_t n_tokens, float scale, void* out, hipStream_t stream) {
    const uint32_t row_chunks = (uint32_t)(hidden / R::kVec);
    const int64_t blocks = (n_tokens * row_chunks + kThreads * kFwdChunks - 1) / (kThreads * kFwdChunks);
    if (blocks > 0x7FFFFFFF) return PICOMOE_ERR_TOO_LARGE;
    embedding_fwd_kernel<R><<<(unsigned)blocks, kThreads, 0, stream>>>((const typename R::raw*)weight, vocab, row_chunks, ids, n_tokens, scale,
                                                                       (typename R::raw*)out);
    return picomoe_launch_status();
}

template <typename R>
int launch_sum(const void* d_out, SumArgs a, int64_t hidden, void* d_weight, hipStream_t stream) {
    a.row_chunks = (uint32_t)(hidden / R::kVec);
    const int group = a.row_chunks <= 64 ? 64 : kThreads, groups = kThreads / group;
    const unsigned slabs = (a.row_chunks + group - 1) / group;
    const int64_t row_blocks = (a.vocab + groups * kRowsPerGroup - 1) / (groups * kRowsPerGroup);
    const int64_t chunks = (a.n + kChunk - 1) / kChunk, chunk_blocks = (chunks + groups - 1) / groups;
    if (row_blocks + chunk_blocks > 0x7FFFFFFF) return PICOMOE_ERR_TOO_LARGE;
    sum_runs_kernel<R><<<dim3((unsigned)(row_blocks + chunk_blocks), slabs), kThreads, 0, stream>>>((const typename R::raw*)d_out, a, group,
                                                                                                  chunk_blocks, (typename R::raw*)d_weight);
    if (a.n > kChunk) join_runs_kernel<R><<<dim3((unsigned)chunk_blocks, slabs), kThreads, 0, stream>>>(a, group, (typename R::raw*)d_weight);
    return picomoe_launch_status();
}

}  // namespace

extern "C" int picomoe_embedding_fwd(const void* weight, int dtype, int64_t vocab, int64_t hidden, const int64_t* ids, int64_t n_tokens, float scale,
                                     void* out, void* stream) {
    PICOMOE_CHECK_ARG(sizes_fit(dtype, n_tokens, vocab, hidden) && scale >= -3e38f && scale <= 3e38f);
    if (n_tokens == 0) return PICOMOE_OK;
    PICOMOE_CHECK_ARG(weight && ids && out);
    hipStream_t s = (hipStream_t)stream;
    const bool wide = wide_rows(dtype, hidden, weight, out);
    if (dtype == PICOMOE_BF16)
        return wide ? launch_fwd<Row<__bf16, true>>(weight, vocab, hidden, ids, n_tokens, scale, out, s)
                    : launch_fwd<Row<__bf16, false>>(weight, vocab, hidden, ids, n_tokens, scale, out, s);
    return wide ? launch_fwd<Row<float, true>>(weight, vocab, hidden, ids, n_tokens, scale, out, s)
                : launch_fwd<Row<float, false>>(weight, vocab, hidden, ids, n_tokens, scale, out, s);
}

extern "C" int64_t picomoe_embedding_bwd_workspace_bytes(int dtype, int64_t n_tokens, int64_t vocab, int64_t hidden) {
    if (!sizes_fit(dtype, n_tokens, vocab, hidden)) return -1;
    return bwd_layout(n_tokens, hidden).bytes;
}

extern "C" int picomoe_embedding_bwd(const void* d_out, int dtype, const int64_t* ids, int64_t n_tokens, int64_t vocab, int64_t hidden, float scale,
                                     int64_t padding_idx, void* d_weight, void* workspace, int64_t workspace_bytes, void* stream) {
    PICOMOE_CHECK_ARG(sizes_fit(dtype, n_tokens, vocab, hidden) && d_weight && scale >= -3e38f && scale <= 3e38f);
    const BwdLayout l = bwd_layout(n_tokens, hidden);
    PICOMOE_CHECK_ARG(n_tokens == 0 || (d_out && ids && workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= l.bytes));
    hipStream_t s = (hipStream_t)stream;
    char* ws = (char*)workspace;
    const int bits = key_bits(vocab), passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits, digit_bits = (bits + passes - 1) / passes;
    SumArgs a = {};
    for (int pass = 0; pass < passes && n_tokens > 0; ++pass) {
        SortPass p;
        p.ids = pass == 0 ? ids : nullptr;
        p.keys = (const uint32_t*)(ws + l.keys[(pass + 1) & 1]);
        p.vals = (const int32_t*)(ws + l.vals[(pass + 1) & 1]);
        p.keys_out = (uint32_t*)(ws + l.keys[pass & 1]);
        p.vals_out = (int32_t*)(ws + l.vals[pass & 1]);
        p.hist = (int32_t*)(ws + l.hist);
        p.n = n_tokens; p.vocab = vocab; p.padding = padding_idx;
        p.shift = pass * digit_bits; p.bits = digit_bits;
        a.keys = p.keys_out;
        a.vals = p.vals_out;
        if (n_tokens <= kSmall) {
            constexpr int kLds = (2 * kSmall + kSortWaves * kMaxDigits + kSortWaves) * 4;
            const hipError_t e = allow_lds<sort_small_kernel>(kLds);
            if (e != hipSuccess) return PICOMOE_ERR_HIP_BASE + (int)e;
            sort_small_kernel<<<1, kSortThreads, kLds, s>>>(p, passes);
            break;
        }
        const unsigned blocks = (unsigned)sort_blocks(n_tokens);
        const int rounds = sort_rounds(n_tokens);
        if (rounds == 1) {
            sort_count_kernel<1><<<blocks, kSortThreads, 0, s>>>(p);
            sort_scatter_kernel<1><<<blocks, kSortThreads, 0, s>>>(p);
        } else if (rounds == 4) {
            sort_count_kernel<4><<<blocks, kSortThreads, 0, s>>>(p);
            sort_scatter_kernel<4><<<blocks, kSortThreads, 0, s>>>(p);
        } else {
            sort_count_kernel<16><<<blocks, kSortThreads, 0, s>>>(p);
            sort_scatter_kernel<16><<<blocks, kSortThreads, 0, s>>>(p);
        }
    }
    a.n = n_tokens; a.vocab = vocab; a.scale = scale;
    a.partial = n_tokens > 0 ? (float*)(ws + l.partial) : nullptr;
    const bool wide = wide_rows(dtype, hidden, d_out, d_weight);
    if (dtype == PICOMOE_BF16)
        return wide ? launch_sum<Row<__bf16, true>>(d_out, a, hidden, d_weight, s) : launch_sum<Row<__bf16, false>>(d_out, a, hidden, d_weight, s);
    return wide ? launch_sum<Row<float, true>>(d_out, a, hidden, d_weight, s) : launch_sum<Row<float, false>>(d_out, a, hidden, d_weight, s);
}
