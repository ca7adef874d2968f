// Attention forward on MFMA: one pass over the keys with the running maximum and sum of the softmax.
//
// The query heads of a key head are one list of rows, row r = query r / group, head r % group of the group, so that a K / V
// tile in LDS serves all of them and one new token of a large group still fills a fragment.  A wavefront owns 32 rows, one per
// lane pair (lane, lane + 32): S^T[key, row] = K Q^T keeps a row's scores in its two lanes -- maximum and sum need one exchange
// between them --, and O^T[d, row] = V^T P^T takes P from registers.  Tiles are loaded straight into one of two LDS buffers while
// the other is multiplied, one barrier per tile.
//
// The accumulated O is only rescaled when a row's maximum grows by more than 2^8: until then P is at most 2^8 instead of 1,
// which costs bf16 nothing and fp32 sums nothing, and the 64 multiplications per tile fall away in all but the first tiles.
// bf16: in blocks that hold rows with few keys, and in the form for few rows, P enters the products in two parts.  Other rows are divided by
// the sum of P and of what rounding added to the largest one: where a key outweighs the others, its rounding then shows neither in out nor in
// the backward's D, beside which the others' dP - D are small (a key of 2^7.8 times the weight of another, in a later tile: dq off by 0.22
// without this, by 0.003 with it).
//
// Bound: the issue of vector instructions.  A wavefront's MFMAs keep the matrix pipe busy for 50 % of the cycles; its softmax takes a
// vector instruction of every SIMD for as long again, and an MFMA occupies the port that issues them for about half its own time.
// Measured, causal, 16 query over 4 key heads, bf16: 16384 tokens, head_dim 128: 1.05 ms = 1045 TFLOP/s (a library GEMM of 8192^3:
// 1157), with softcap 1.33 ms; 2 x 8192 tokens, head_dim 64: 0.32 ms = 865; 8192 tokens, 8 over 4 heads of 256: 0.40 ms = 690 (512
// registers, one wavefront per SIMD).  fp32, 4096 tokens, 8 over 2 heads of 128: 0.46 ms = 75 (GEMM: 154).  One new token for each of 8
// sequences over 32768 keys, 32 over 8 heads: 0.210 ms = 5.1 TB/s of K and V (a copy: 4.9 read and written), + 7 us for the join; P in two
// parts is 1 % of that.  2 x 8192 tokens: documents of 1024 0.154 ms, of 40, where every row has few keys, 0.081; 16384 tokens, window 64:
// 0.135 ms, window 1024: 0.220.
// Tried and slower: tiles of 128 keys; of 32 keys with three wavefronts per SIMD (1.32 ms); blocks of eight wavefronts; a higher
// priority for the wavefront in its MFMAs (+7 %); the panel tiles of the backward (one token: 239 us).
#include "attention_tiles.h"

namespace {

constexpr float kLazy = 8.f;

// KEYS: the four waves share 32 rows and split every tile's keys among them (few rows: one new token); otherwise every wave
// has 32 rows of its own and all of the tile's keys.  The first, which waits for K and V and not for its products, takes P of all rows
// in two bf16 parts.
template <typename T, int DP, bool KEYS>
struct FwdShape {
    static constexpr int kTile = KEYS ? 32 * kWaves : (sizeof(T) == 2 ? 64 : 32);  // keys of a tile
    static constexpr int kWaveKeys = KEYS ? 32 : kTile;
    static constexpr int kRows = KEYS ? 32 : 32 * kWaves;  // rows of a block
    typedef Tile<T, DP, kTile> Tl;
    static constexpr int kTileBytes = Tl::kBytes;
    static constexpr int kBuffers = kTileBytes <= 36 * 1024 ? 2 : 1;  // two of 128 KB do not fit
    static constexpr int kBuf = 2 * kTileBytes + kTile * 4;       // K, V, document ids
    static constexpr int kLds = kBuffers * kBuf;
    static constexpr int kWavesPerSimd = sizeof(T) == 4 || DP == 256 ? 1 : (DP == 64 && !KEYS ? 3 : 2);  // as the registers allow
};

// four elements of out, and of its residual where it is wanted
template <typename T>
__device__ __forceinline__ void store_out(const AttnArgs& a, int64_t at, f32x4_t v) {
    if constexpr (sizeof(T) == 2) {
        const u32x2_t w = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        *(u32x2_t*)((T*)a.out + at) = w;
        if (a.residual) {
            f32x4_t rest;
#pragma unroll
            for (int e = 0; e < 4; ++e) rest[e] = v[e] - __uint_as_float(e & 1 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16);
            *(u32x2_t*)((T*)a.residual + at) = u32x2_t{pack_bf16x2(rest[0], rest[1]), pack_bf16x2(rest[2], rest[3])};
        }
    } else {
        *(f32x4_t*)((T*)a.out + at) = v;
    }
}

template <typename T, int DP, bool KEYS, int MODE>
__global__ __launch_bounds__(kThreads, (FwdShape<T, DP, KEYS>::kWavesPerSimd)) void attention_fwd_kernel(MfmaArgs m) {
    typedef FwdShape<T, DP, KEYS> Sh;
    typedef typename Sh::Tl Tl;
    constexpr int kSub = Sh::kWaveKeys / 32, kSteps = DP / 16, kCols = DP / 32;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const AttnArgs& a = m.a;
    const int lane = threadIdx.x & 63, wave = wave_index(), hi = lane >> 5;

    // blocks of one key head lie on one XCD where there are 8 heads or more; those with the most keys (the last rows) go first
    const int heads = (int)a.batch * a.kv_heads, bh = blockIdx.x % heads, tile = m.blocks - 1 - blockIdx.x / heads, split = blockIdx.y;
    const int b = bh / a.kv_heads, kvh = bh % a.kv_heads;
    const int row0 = tile * Sh::kRows + (KEYS ? 0 : wave * 32);
    int row = row0 + (lane & 31);
    const bool row_in = row < m.rows;
    row = row_in ? row : m.rows - 1;  // rows past the end repeat the last one
    const int s = m.div(row), head = kvh * a.group + row - s * a.group, pos = s + a.kv_len - a.q_len;
    const RowSpan span = row_span(a, b, s);
    const int key_span = span.hi - span.lo;  // negative: no keys
    const float slope2 = a.slopes ? a.slopes[head] * kLog2e : 0.f;

    Frag<T> qf[kSteps];
    const T* q = (const T*)a.q.p + b * a.q.sb + s * a.q.ss + head * a.q.sh;
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) qf[ks] = load_frag<T>(q, 16 * ks + 8 * hi, a.D);

    const bool some = key_span >= 0;
    const Reach w = wave_reach(some, span);
    bool two_parts = sizeof(T) == 2 && !KEYS && __any(some && has_few(m, b, s, key_span));
    const Reach blk = KEYS ? w : block_reach(w, two_parts);
    const int32_t* doc_min = a.docs ? m.key_docs.lowest + (int64_t)b * m.key_docs.tiles : nullptr;
    const int32_t* doc_max = a.docs ? m.key_docs.highest + (int64_t)b * m.key_docs.tiles : nullptr;
    const bool any = blk.hi_max >= blk.lo_min;
    const int first = any ? blk.lo_min / Sh::kTile : 0, end = any ? blk.hi_max / Sh::kTile + 1 : 0;
    auto active = [&](int, int d0, int d1) { return !a.docs || (d1 >= blk.doc_min && d0 <= blk.doc_max); };
    Share share = {1, 0, 0x7FFFFFFF};
    if (m.splits > 1) {
        share = share_of(a.docs ? count_tiles(first, end, doc_min, doc_max, active) : end - first, split, m);
        if (split == 0 && threadIdx.x == 0) m.parts[bh * m.blocks + tile] = share.parts;
        if (split >= share.parts) return;
    }

    const T* kbase = (const T*)a.k.p + b * a.k.sb + kvh * a.k.sh;
    const T* vbase = (const T*)a.v.p + b * a.v.sb + kvh * a.v.sh;
    if (a.D < DP) clear_lds(lds, Sh::kLds);
    // rows of a tile within 2^31 bytes, whole tiles: no vector arithmetic for the addresses
    const uint32_t k_step = (uint32_t)(a.k.ss * (int)sizeof(T)), v_step = (uint32_t)(a.v.ss * (int)sizeof(T));
    const bool even = a.D == DP && a.k.ss < (1 << 22) && a.v.ss < (1 << 22);
    const typename Tl::Source k_src(k_step), v_src(v_step);
    auto fetch = [&](int t, int buf) __attribute__((always_inline)) {
        const uint32_t kt = lds_address(lds) + buf * Sh::kBuf;
        // keys past the end are hidden by every row's interval
        auto key_at = [&](int r) { return (int64_t)min(t * Sh::kTile + r, a.kv_len - 1); };
        if (even && (t + 1) * Sh::kTile <= a.kv_len) {
            Tl::load_even(kt, (const char*)(kbase + (int64_t)t * Sh::kTile * a.k.ss), k_step, k_src);
            Tl::load_even(kt + Sh::kTileBytes, (const char*)(vbase + (int64_t)t * Sh::kTile * a.v.ss), v_step, v_src);
        } else {
            Tl::load(kt, a.D, [&](int r) { return kbase + key_at(r) * a.k.ss; });
            Tl::load(kt + Sh::kTileBytes, a.D, [&](int r) { return vbase + key_at(r) * a.v.ss; });
        }
        if (a.docs && wave < Sh::kTile / 64)
            load4_to_lds(a.docs + (int64_t)b * a.kv_len + key_at(wave * 64 + lane), kt + 2 * Sh::kTileBytes + wave * 256);
        if (a.docs && Sh::kTile < 64 && wave == 0 && lane < Sh::kTile) load4_to_lds(a.docs + (int64_t)b * a.kv_len + key_at(lane), kt + 2 * Sh::kTileBytes);
    };

    const typename Tl::Lane ln;
    const ScoreScale sc = score_scale<MODE>(a);
    f32x16_t o[kCols];
    float top = -INFINITY, total = 0.f;  // what P refers to (log2 units), this lane's share of the sum
    float largest = -INFINITY, over = 0.f;  // the maximum, and what the rounding of its P to bf16 added to it

    auto run = [&](auto which, auto parts) __attribute__((always_inline)) {
        constexpr Walk kWalk = decltype(which)::value;
        constexpr int kParts = decltype(parts)::value;
        constexpr bool kOneRounded = sizeof(T) == 2 && kParts == 1;
        top = largest = -INFINITY;
        total = over = 0.f;
#pragma unroll
        for (int t = 0; t < kCols; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[t][i] = 0.f;

        TileWalk<decltype(active)> walk(first, end, doc_min, doc_max, active, share.skip, share.left);
        WalkTile cur = walk.next();
        int buf = 0;
        if (cur.t >= 0) fetch(cur.t, 0);
        while (cur.t >= 0) {
            lds_loads_done();
            __syncthreads();  // the tile is there, and every wave is done with the other buffer
            const WalkTile following = walk.next();
            if (Sh::kBuffers == 2 && following.t >= 0) fetch(following.t, buf ^ 1);
            const char* kt = lds + buf * Sh::kBuf;
            const char* vt = kt + Sh::kTileBytes;
            const int32_t* docs = (const int32_t*)(vt + Sh::kTileBytes);
            const uint32_t ka = lds_address(kt) + (KEYS ? wave * 32 * Tl::kRowBytes : 0), va = ka + Sh::kTileBytes;
            const int sub0 = KEYS ? wave * 32 : 0, key0 = cur.t * Sh::kTile + sub0, key1 = key0 + Sh::kWaveKeys - 1;
            bool in = key0 <= w.hi_max && key1 >= w.lo_min, full = key0 >= w.lo_max && key1 <= w.hi_min;
            if (a.docs) {
                in = in && cur.doc_max >= w.doc_min && cur.doc_min <= w.doc_max;
                full = full && cur.doc_min == cur.doc_max && cur.doc_min == w.doc_min && cur.doc_min == w.doc_max;
            }
            if (in) {
                const typename Tl::Rows k_rows(ln, ka);
                const typename Tl::Cols v_cols(ln, va);
                f32x16_t x[kSub];
#pragma unroll
                for (int u = 0; u < kSub; ++u) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[u][i] = 0.f;
#pragma unroll
                    for (int ks = 0; ks < kSteps; ++ks) mma(x[u], Tl::frag(k_rows, u * 32, ks), qf[ks]);
                }
                if (sizeof(T) == 2) read_ahead<1, 1, kSub * kSteps, 2>();
                if (MODE == kPlain) {
                } else if (sc.cap2 > 0.f) {
#pragma unroll
                    for (int u = 0; u < kSub; ++u)
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[u][i] = sc.cap2 * capped<MODE>(x[u][i], sc.mul);
                } else {
#pragma unroll
                    for (int u = 0; u < kSub; ++u)
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[u][i] *= sc.mul;
                }
                if (MODE != kPlain && a.slopes) {
                    const float away = (float)(pos - key0 - 4 * hi);
#pragma unroll
                    for (int u = 0; u < kSub; ++u)
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[u][i] -= slope2 * __builtin_fabsf(away - (float)(u * 32 + 8 * (i / 4) + i % 4));
                }
                if (!full) {
                    const int from = span.lo - key0 - 4 * hi;  // the lane's first key is 0
                    const uint32_t seen_keys = (uint32_t)key_span;
#pragma unroll
                    for (int u = 0; u < kSub; ++u)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            x[u][i] = (uint32_t)(u * 32 + 8 * (i / 4) + i % 4 - from) <= seen_keys ? x[u][i] : -INFINITY;
                    if (key_span < 0) {
#pragma unroll
                        for (int u = 0; u < kSub; ++u)
#pragma unroll
                            for (int i = 0; i < 16; ++i) x[u][i] = -INFINITY;
                    }
                    if (a.docs) {
                        typedef __attribute__((ext_vector_type(4))) int i32x4_t;
#pragma unroll
                        for (int u = 0; u < kSub; ++u)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const i32x4_t d = *(const i32x4_t*)(docs + sub0 + u * 32 + 8 * j + 4 * hi);
#pragma unroll
                                for (int i = 0; i < 4; ++i) x[u][4 * j + i] = d[i] == span.doc ? x[u][4 * j + i] : -INFINITY;
                            }
                    }
                }
                float mx = x[0][0];
#pragma unroll
                for (int u = 0; u < kSub; ++u)
#pragma unroll
                    for (int i = 0; i < 16; ++i) mx = __builtin_fmaxf(mx, x[u][i]);
                const float raw_mx = other_max(mx);
                mx = raw_mx * (MODE == kPlain ? sc.mul : 1.f);
                if (__any(mx > top + kLazy)) {
                    const float old = top;
                    top = __builtin_fmaxf(top, mx);
                    const float shrink = __builtin_amdgcn_exp2f(old - (top == -INFINITY ? 0.f : top));
                    total *= shrink;
                    if constexpr (kOneRounded) over *= shrink;
#pragma unroll
                    for (int t = 0; t < kCols; ++t)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[t][i] *= shrink;
                }
                const float base = top == -INFINITY ? 0.f : top;
                if (kOneRounded && __any(mx > largest)) {
                    const float p = __builtin_amdgcn_exp2f(MODE == kPlain ? __builtin_fmaf(raw_mx, sc.mul, -base) : raw_mx - base);
                    over = mx > largest ? (float)(__bf16)p - p : over;
                    largest = __builtin_fmaxf(largest, mx);
                }
#pragma unroll
                for (int u = 0; u < kSub; ++u)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        x[u][i] = __builtin_amdgcn_exp2f(MODE == kPlain ? __builtin_fmaf(x[u][i], sc.mul, -base) : x[u][i] - base);
                        total += x[u][i];
                    }
#pragma unroll
                for (int st = 0; st < 2 * kSub; ++st) {
                    const Frag<T> p = to_frag<T>(x[st / 2], st & 1);
                    Frag<T> rest;
                    if constexpr (kParts == 2) rest = rest_frag<T>(x[st / 2], st & 1);
#pragma unroll
                    for (int t = 0; t < kCols; ++t) {
                        Frag<T> v = Tl::frag_t(v_cols, 16 * st, t);
                        if (kWalk == kCareful) zero_not_finite(v);
                        mma(o[t], v, p);
                        if constexpr (kParts == 2) mma(o[t], v, rest);
                    }
                }
                if (sizeof(T) == 2 && kWalk != kCareful) read_ahead<2, kParts, 2 * kSub * kCols, 2>();
                if (kWalk == kCareful) {
                    bool bad = false;
                    if (lane < Sh::kWaveKeys) bad = Tl::row_not_finite(vt, sub0 + lane);
                    for (uint64_t left = __ballot(bad); left; left &= left - 1) {
                        const int key = __builtin_ctzll(left), j = key0 + key;
                        const bool see = j >= span.lo && j <= span.hi && (!a.docs || docs[sub0 + key] == span.doc);
#pragma unroll
                        for (int t = 0; t < kCols; ++t)
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const float v = Tl::element(vt, sub0 + key, 32 * t + 8 * (i / 4) + 4 * hi + i % 4);
                                if (see && !(__builtin_fabsf(v) < INFINITY)) o[t][i] += v;
                            }
                    }
                }
            }
            cur = following;
            if (Sh::kBuffers == 2) {
                buf ^= 1;
            } else if (cur.t >= 0) {
                __syncthreads();
                fetch(cur.t, 0);
            }
        }
    };
    typedef std::integral_constant<int, 1> One;
    typedef std::integral_constant<int, 2> Two;
    auto walk_all = [&](auto which) __attribute__((always_inline)) {
        if constexpr (sizeof(T) == 4) {
            run(which, One());
        } else if constexpr (KEYS) {
            run(which, Two());
        } else {
            if (two_parts) run(which, Two());
            else run(which, One());
        }
    };
    walk_all(std::integral_constant<Walk, kMain>());
    lds_loads_done();  // also where no tile was walked: nothing may land in LDS after the block is gone
    bool bad = false;
#pragma unroll
    for (int t = 0; t < kCols; ++t) bad |= not_finite(o[t]);
    if (__syncthreads_or(bad)) {
        walk_all(std::integral_constant<Walk, kCareful>());
        __syncthreads();
    }
    total = other_sum(total);

    if (KEYS) {  // the four waves' sums over their keys, through LDS (the tile is no longer needed)
        float* part = (float*)lds;  // [wave][32 rows][DP]
        __shared__ float part_top[kWaves][32], part_total[kWaves][32];
#pragma unroll
        for (int t = 0; t < kCols; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x4_t v = {o[t][4 * j], o[t][4 * j + 1], o[t][4 * j + 2], o[t][4 * j + 3]};
                *(f32x4_t*)(part + (wave * 32 + (lane & 31)) * DP + 32 * t + 8 * j + 4 * hi) = v;
            }
        if (lane < 32) {
            part_top[wave][lane] = top;
            part_total[wave][lane] = total;
        }
        __syncthreads();
        if (wave != 0) return;
        const int r = lane & 31;
        float t0 = -INFINITY;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) t0 = __builtin_fmaxf(t0, part_top[i][r]);
        const float base = t0 == -INFINITY ? 0.f : t0;
        float weight[kWaves];
        total = 0.f;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            weight[i] = __builtin_amdgcn_exp2f(part_top[i][r] - base);
            total += weight[i] * part_total[i][r];
        }
        top = t0;
#pragma unroll
        for (int t = 0; t < kCols; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < kWaves; ++i) sum += weight[i] * *(const f32x4_t*)(part + (i * 32 + r) * DP + 32 * t + 8 * j + 4 * hi);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[t][4 * j + e] = sum[e];
            }
    }

    const float inv = total == 0.f ? 0.f : 1.f / (total + over);
    const float lse2 = total == 0.f ? -INFINITY : (top == -INFINITY ? 0.f : top) + log2f(total);
    if (!row_in) return;
    if (share.parts > 1) {
        const int64_t at = ((int64_t)split * heads + bh) * m.rows + row;
        float* to = m.part_out + at * a.D;
        if (hi == 0) m.part_lse[at] = lse2;
#pragma unroll
        for (int t = 0; t < kCols; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int d = 32 * t + 8 * j + 4 * hi;
                if (d < a.D) *(f32x4_t*)(to + d) = f32x4_t{o[t][4 * j] * inv, o[t][4 * j + 1] * inv, o[t][4 * j + 2] * inv, o[t][4 * j + 3] * inv};
            }
        return;
    }
    T* to = (T*)a.out + (((int64_t)b * a.q_len + s) * a.heads + head) * a.D;
    if (hi == 0) a.lse[((int64_t)b * a.heads + head) * a.q_len + s] = lse2 * (1.f / kLog2e);
#pragma unroll
    for (int t = 0; t < kCols; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = 32 * t + 8 * j + 4 * hi;
            if (d >= a.D) continue;
            store_out<T>(a, (to - (T*)a.out) + d, f32x4_t{o[t][4 * j] * inv, o[t][4 * j + 1] * inv, o[t][4 * j + 2] * inv, o[t][4 * j + 3] * inv});
        }
}

// Joins the parts of a row: out = sum 2^(lse_i - max) out_i / sum 2^(lse_i - max).  32 lanes per row, four columns at a time a lane.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_join_kernel(MfmaArgs m, int block_rows) {
    const AttnArgs& a = m.a;
    const int lane = threadIdx.x & 31, heads = (int)a.batch * a.kv_heads;
    const int64_t index = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), per_split = (int64_t)heads * m.rows;
    if (index >= per_split) return;
    const int bh = (int)(index / m.rows), row = (int)(index - (int64_t)bh * m.rows), b = bh / a.kv_heads, kvh = bh - b * a.kv_heads;
    const int parts = m.parts[bh * m.blocks + row / block_rows];
    if (parts == 1) return;  // written by its block
    const int s = m.div(row), head = kvh * a.group + row - s * a.group;
    float top = -INFINITY;
    for (int i = 0; i < parts; ++i) top = __builtin_fmaxf(top, m.part_lse[i * per_split + index]);
    const float base = top == -INFINITY ? 0.f : top;
    for (int d = 4 * lane; d < a.D; d += 128) {
        float total = 0.f;
        f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int i = 0; i < parts; ++i) {
            const float lse2 = m.part_lse[i * per_split + index];  // -inf: saw no key
            const float weight = __builtin_amdgcn_exp2f(lse2 - base);
            total += weight;
            sum += weight * *(const f32x4_t*)(m.part_out + (i * per_split + index) * a.D + d);
        }
        if (d == 0) a.lse[((int64_t)b * a.heads + head) * a.q_len + s] = total == 0.f ? -INFINITY : (base + log2f(total)) * (1.f / kLog2e);
        const int64_t at = (((int64_t)b * a.q_len + s) * a.heads + head) * a.D + d;
        store_out<T>(a, at, sum * (total == 0.f ? 0.f : 1.f / total));
    }
}

// What the kernel wants to know of the documents: the ranges of the key tiles, and (bf16) which queries have few keys
__global__ __launch_bounds__(kThreads) void attention_documents_kernel(MfmaArgs m, int tile, int key_blocks) {
    if ((int)blockIdx.x < key_blocks)
        document_range(m.a.docs, m.a.kv_len, blockIdx.x, tile, m.key_docs.tiles, m.a.kv_len, 0, GroupDiv{0u, 0}, (int32_t*)m.key_docs.lowest,
                       (int32_t*)m.key_docs.highest);
    else
        few_queries(m.a, blockIdx.x - key_blocks, (uint64_t*)m.few);
}

template <typename T, int DP, bool KEYS, int MODE>
int launch(const MfmaArgs& m, hipStream_t s) {
    typedef FwdShape<T, DP, KEYS> Sh;
    const hipError_t e = allow_lds<attention_fwd_kernel<T, DP, KEYS, MODE>>(Sh::kLds);
    if (e != hipSuccess) return PICOMOE_ERR_HIP_BASE + (int)e;
    const int64_t blocks = (int64_t)m.blocks * m.a.batch * m.a.kv_heads;
    if (blocks > 0x7FFFFFFF) return PICOMOE_ERR_TOO_LARGE;
    attention_fwd_kernel<T, DP, KEYS, MODE><<<dim3((unsigned)blocks, (unsigned)m.splits), kThreads, Sh::kLds, s>>>(m);
    if (m.splits > 1) {
        const int64_t rows = (int64_t)m.a.batch * m.a.kv_heads * m.rows;
        attention_join_kernel<T><<<(unsigned)((rows + 7) / 8), kThreads, 0, s>>>(m, Sh::kRows);
    }
    return picomoe_launch_status();
}
template <typename T, int DP, bool KEYS>
int launch_mode(const MfmaArgs& m, hipStream_t s) {
    // the running maximum is taken of the unscaled products: scale > 0
    const ScoreMode mode = score_mode(m.a, m.a.softcap == 0.f && !m.a.slopes && m.a.scale > 0.f);
    if (mode == kPlain) return launch<T, DP, KEYS, kPlain>(m, s);
    if constexpr (sizeof(T) == 2)
        if (mode == kFast) return launch<T, DP, KEYS, kFast>(m, s);
    return launch<T, DP, KEYS, kAccurate>(m, s);
}
template <typename T, int DP>
int launch_for(const MfmaArgs& m, bool keys, hipStream_t s) {
    return keys ? launch_mode<T, DP, true>(m, s) : launch_mode<T, DP, false>(m, s);
}

struct Plan {
    bool keys;  // the waves of a block share 32 rows
    int tile, blocks, key_tiles, splits, target;
    int64_t doc_bytes, few_bytes, parts_bytes, out_bytes, lse_bytes;
};
int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

Plan plan(int dtype, int64_t batch, int64_t q_len, int64_t kv_len, int q_heads, int kv_heads, int head_dim) {
    Plan p;
    const int64_t rows = q_len * (q_heads / kv_heads), heads = batch * kv_heads;
    p.keys = rows <= 32;
    p.tile = p.keys ? 128 : (dtype == PICOMOE_BF16 ? 64 : 32);
    const int per = p.keys ? 32 : 32 * kWaves;
    p.blocks = (int)((rows + per - 1) / per);
    p.key_tiles = (int)((kv_len + p.tile - 1) / p.tile);
    // Walks are cut where they are longer than what each of the 512 blocks that the chip holds gets of all rows x all keys
    const int64_t share = (heads * p.blocks * p.key_tiles + 511) / 512, shortest = p.keys ? 2 : 4, longest = (p.key_tiles + 255) / 256;
    int64_t target = share > shortest ? share : shortest;
    target = target > longest ? target : longest;
    p.target = (int)(target < p.key_tiles || p.key_tiles == 0 ? target : p.key_tiles);
    p.splits = p.key_tiles > p.target ? (p.key_tiles + p.target - 1) / p.target : 1;
    p.doc_bytes = round16(batch * p.key_tiles * 8);
    p.few_bytes = dtype == PICOMOE_BF16 && !p.keys ? round16(batch * few_words(q_len) * 8) : 0;
    p.parts_bytes = p.splits > 1 ? round16(heads * p.blocks * 4) : 0;
    p.out_bytes = p.splits > 1 ? round16((int64_t)p.splits * heads * rows * head_dim * 4) : 0;
    p.lse_bytes = p.splits > 1 ? round16((int64_t)p.splits * heads * rows * 4) : 0;
    return p;
}

}  // namespace

bool attention_mfma_supported(int dtype, int head_dim) { return head_dim <= (dtype == PICOMOE_BF16 ? 256 : 128); }

int64_t attention_mfma_fwd_workspace(int dtype, int64_t batch, int64_t q_len, int64_t kv_len, int q_heads, int kv_heads, int head_dim) {
    const Plan p = plan(dtype, batch, q_len, kv_len, q_heads, kv_heads, head_dim);
    return p.doc_bytes + p.few_bytes + p.parts_bytes + p.out_bytes + p.lse_bytes + 16;
}

int attention_mfma_fwd(const AttnArgs& a, hipStream_t s) {
    const Plan p = plan(a.dtype, a.batch, a.q_len, a.kv_len, a.heads, a.kv_heads, a.D);
    MfmaArgs m = {};
    m.a = a;
    m.div = group_div(a.group);
    m.rows = a.q_len * a.group;
    m.blocks = p.blocks;
    m.splits = p.splits;
    m.target = p.target;
    char* ws = a.ws;
    auto take = [&](int64_t bytes) {
        char* at = ws;
        ws += bytes;
        return at;
    };
    int32_t* lowest = (int32_t*)take(p.doc_bytes);
    m.key_docs = {lowest, lowest + a.batch * p.key_tiles, p.key_tiles};
    const uint64_t* few = (const uint64_t*)take(p.few_bytes);
    m.parts = (int32_t*)take(p.parts_bytes);
    m.part_out = (float*)take(p.out_bytes);
    m.part_lse = (float*)take(p.lse_bytes);
    if (a.docs && p.key_tiles > 0) {
        const bool count_few = p.few_bytes > 0;
        const int64_t key_blocks = a.batch * range_blocks(p.key_tiles), blocks = key_blocks + (count_few ? a.batch * few_blocks(a.q_len) : 0);
        if (blocks > 0x7FFFFFFF) return PICOMOE_ERR_TOO_LARGE;
        m.few = count_few ? few : nullptr;
        m.few_words = few_words(a.q_len);
        attention_documents_kernel<<<(unsigned)blocks, kThreads, 0, s>>>(m, p.tile, (int)key_blocks);
    }
    if (a.D > 128) return launch_for<__bf16, 256>(m, p.keys, s);
    if (a.dtype == PICOMOE_BF16) return a.D <= 64 ? launch_for<__bf16, 64>(m, p.keys, s) : launch_for<__bf16, 128>(m, p.keys, s);
    return a.D <= 64 ? launch_for<float, 64>(m, p.keys, s) : launch_for<float, 128>(m, p.keys, s);
}
