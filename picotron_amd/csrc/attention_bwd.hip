// Attention backward on MFMA, without atomics: one launch forms dq, another dk and dv, P recomputed from lse in both.
//
// Seven products instead of the five of the formulas (S and dP are formed twice); what that buys is that every sum has one owner
// and one order.  dq: a wavefront owns 32 rows (as in the forward), walks the key tiles: S^T = K Q^T, dP^T = V dO^T,
// dq^T += K^T dx^T.  dk, dv: a wavefront owns 32 keys, walks the row tiles of the key head -- all its query heads, so that their
// gradients meet in one accumulator: S = Q K^T, dP = dO V^T, dv^T += dO^T P, dk^T += Q^T dx.  Blocks with long walks are cut
// into parts (MfmaArgs) whose fp32 sums a last launch adds in order; a first one forms D = dO . out.  Both kinds of blocks in one
// launch were slower (8.3 ms for what then took 4.7 + 2.3): the registers of the two spill more together.
//
// Bound: dq as the forward (MFMAs 59 % of the cycles).  dk / dv, which reads three LDS fragments for two MFMAs and has a tile of 32 rows
// between barriers, is at 40 %; its loads, which mostly miss the L2, are not what holds it (walks from the last
// tile on, in step over an XCD's blocks so that they share them: -1.5 % at 16384 tokens, +4 % with documents).  Tiles of 64 rows with eight wavefronts
// take 2 % less at 16384 tokens and 23 % more at 4096.
// Measured, bf16, 16384 causal tokens, 16 over 4 heads of 128: prepare 0.03, dq 1.39 ms = 1190 TFLOP/s of its three products, dk / dv
// 2.45 ms = 895 of its four, join 0.06; with softcap 1.69 and 3.10.  2048 tokens: 56 + 100 + 20 + 7 us.  2 x 8192 tokens, head_dim 64:
// 0.40 and 0.86 ms.  fp32, 4096 tokens, 8 over 2 heads of 128: 0.60 and 0.82 ms = 86 and 83 TFLOP/s.  2 x 8192 tokens: documents of 1024
// 0.18 and 0.35 ms, of 40 0.078 and 0.197 (dk / dv without its second walk: two thirds of that); 16384 tokens, window 64: 0.08 and 0.24 ms.
#include "attention_tiles.h"

namespace {

// ---------------------------------------------------------------------------------------------------------------
// dq
// ---------------------------------------------------------------------------------------------------------------
template <typename T, int DP>
struct DqShape {
    static constexpr int kTile = sizeof(T) == 2 ? 64 : 32;
    typedef PanelTile<T, DP, kTile> Tl;
    static constexpr int kTileBytes = Tl::kBytes;
    static constexpr int kBuf = 2 * kTileBytes + kTile * 4;  // K, V, document ids
    static constexpr int kLds = 2 * kBuf;
};

template <typename T, int DP, int MODE>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 && DP <= 128 ? 2 : 1) void attention_dq_kernel(MfmaArgs m) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    typedef DqShape<T, DP> Sh;
    typedef typename Sh::Tl Tl;
    constexpr int kSub = Sh::kTile / 32, kSteps = DP / 16, kCols = DP / 32;
    const AttnArgs& a = m.a;
    const int lane = threadIdx.x & 63, wave = wave_index(), hi = lane >> 5;

    const int heads = (int)a.batch * a.kv_heads, bh = blockIdx.x % heads, split = blockIdx.y, tile = m.blocks - 1 - blockIdx.x / heads;
    const int b = bh / a.kv_heads, kvh = bh % a.kv_heads;
    int row = tile * 32 * kWaves + wave * 32 + (lane & 31);
    const bool row_in = row < m.rows;
    row = row_in ? row : m.rows - 1;
    const int s = m.div(row), head = kvh * a.group + row - s * a.group, pos = s + a.kv_len - a.q_len;
    const RowSpan span = row_span(a, b, s);
    const int key_span = span.hi - span.lo;
    const float slope2 = a.slopes ? a.slopes[head] * kLog2e : 0.f;
    const int64_t out_row = ((int64_t)b * a.q_len + s) * a.heads + head;

    const bool some = key_span >= 0;
    const Reach w = wave_reach(some, span);
    bool two_parts = sizeof(T) == 2 && __any(some && has_few(m, b, s, key_span));
    const Reach blk = block_reach(w, two_parts);
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

    Frag<T> qf[kSteps], gf[kSteps];
    {
        const T* q = (const T*)a.q.p + b * a.q.sb + s * a.q.ss + head * a.q.sh;
        const T* g = (const T*)a.d_out + out_row * a.D;
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) {
            qf[ks] = load_frag<T>(q, 16 * ks + 8 * hi, a.D);
            gf[ks] = load_frag<T>(g, 16 * ks + 8 * hi, a.D);
        }
    }
    const float* stats = m.stats + ((int64_t)bh * m.row_docs.tiles + row / 32) * (kStats * 32) + row % 32;
    const float delta = stats[kDelta * 32], lse2 = stats[kLse2 * 32];

    const T* kbase = (const T*)a.k.p + b * a.k.sb + kvh * a.k.sh;
    const T* vbase = (const T*)a.v.p + b * a.v.sb + kvh * a.v.sh;
    if (a.D < DP) clear_lds(lds, Sh::kLds);
    const uint32_t k_step = (uint32_t)(a.k.ss * (int)sizeof(T)), v_step = (uint32_t)(a.v.ss * (int)sizeof(T));
    const bool even = a.D == DP && a.k.ss < (1 << 22) && a.v.ss < (1 << 22);  // as in the forward
    const uint32_t k_off = Tl::lane_offset(Tl::lane_row() * k_step), v_off = Tl::lane_offset(Tl::lane_row() * v_step);
    auto fetch = [&](int t, int buf) __attribute__((always_inline)) {
        const uint32_t kt = lds_address(lds) + buf * Sh::kBuf;
        auto key_at = [&](int r) { return (int64_t)min(t * Sh::kTile + r, a.kv_len - 1); };
        if (even && (t + 1) * Sh::kTile <= a.kv_len) {
            Tl::load_even(kt, (const char*)(kbase + (int64_t)t * Sh::kTile * a.k.ss), k_off, [&](int r) { return (uint64_t)(r * k_step); });
            Tl::load_even(kt + Sh::kTileBytes, (const char*)(vbase + (int64_t)t * Sh::kTile * a.v.ss), v_off, [&](int r) { return (uint64_t)(r * v_step); });
        } else {
            Tl::load(kt, a.D, [&](int r) { return kbase + key_at(r) * a.k.ss; });
            Tl::load(kt + Sh::kTileBytes, a.D, [&](int r) { return vbase + key_at(r) * a.v.ss; });
        }
        if (a.docs && wave == 0 && lane < Sh::kTile) load4_to_lds(a.docs + (int64_t)b * a.kv_len + key_at(lane), kt + 2 * Sh::kTileBytes);
    };

    const typename Tl::Lane ln;
    const ScoreScale sc = score_scale<MODE>(a);
    f32x16_t dq[kCols];
    auto run = [&](auto which, auto parts) __attribute__((always_inline)) {
        constexpr Walk kWalk = decltype(which)::value;
        constexpr int kParts = decltype(parts)::value;
#pragma unroll
        for (int t = 0; t < kCols; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) dq[t][i] = 0.f;
        TileWalk<decltype(active)> walk(first, end, doc_min, doc_max, active, share.skip, share.left);
        WalkTile cur = walk.next();
        int buf = 0;
        if (cur.t >= 0) fetch(cur.t, 0);
        while (cur.t >= 0) {
            lds_loads_done();
            __syncthreads();
            const WalkTile following = walk.next();
            if (following.t >= 0) fetch(following.t, buf ^ 1);
            const char* kt = lds + buf * Sh::kBuf;
            const char* vt = kt + Sh::kTileBytes;
            const int32_t* docs = (const int32_t*)(vt + Sh::kTileBytes);
            const uint32_t ka = lds_address(kt), va = ka + Sh::kTileBytes;
            const int key0 = cur.t * Sh::kTile, key1 = key0 + Sh::kTile - 1;
            bool in = key0 <= w.hi_max && key1 >= w.lo_min, full = key0 >= w.lo_max && key1 <= w.hi_min;
            if (a.docs) {
                in = in && cur.doc_max >= w.doc_min && cur.doc_min <= w.doc_max;
                full = full && cur.doc_min == cur.doc_max && cur.doc_min == w.doc_min && cur.doc_min == w.doc_max;
            }
            if (in) {
                const typename Tl::Rows k_rows(ln, ka), v_rows(ln, va);
                const typename Tl::Cols k_cols(ln, ka);
#pragma unroll
                for (int u = 0; u < kSub; ++u) {
                    f32x16_t x, dp;
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] = dp[i] = 0.f;
#pragma unroll
                    for (int ks = 0; ks < kSteps; ++ks) {
                        mma(x, Tl::frag(k_rows, u * 32, ks), qf[ks]);
                        mma(dp, Tl::frag(v_rows, u * 32, ks), gf[ks]);
                    }
                    if (sizeof(T) == 2) read_ahead<2, 2, kSteps, 2>();
#pragma unroll
                    for (int i = 0; i < 16; ++i) dp[i] -= delta;
                    if (MODE == kPlain) {
                    } else if (sc.cap2 > 0.f) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float t = capped<MODE>(x[i], sc.mul);
                            x[i] = sc.cap2 * t;
                            dp[i] *= 1.f - t * t;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[i] *= sc.mul;
                    }
                    if (MODE != kPlain && a.slopes) {
                        const float away = (float)(pos - key0 - 4 * hi);
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[i] -= slope2 * __builtin_fabsf(away - (float)(u * 32 + 8 * (i / 4) + i % 4));
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] = __builtin_amdgcn_exp2f(MODE == kPlain ? __builtin_fmaf(x[i], sc.mul, -lse2) : x[i] - lse2) * dp[i];
                    if (!full) {
                        const int from = span.lo - key0 - 4 * hi;
                        const uint32_t seen_keys = (uint32_t)key_span;
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            x[i] = (uint32_t)(u * 32 + 8 * (i / 4) + i % 4 - from) <= seen_keys && key_span >= 0 ? x[i] : 0.f;
                        if (a.docs) {
                            typedef __attribute__((ext_vector_type(4))) int i32x4_t;
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const i32x4_t d = *(const i32x4_t*)(docs + u * 32 + 8 * j + 4 * hi);
#pragma unroll
                                for (int i = 0; i < 4; ++i) x[4 * j + i] = d[i] == span.doc ? x[4 * j + i] : 0.f;
                            }
                        }
                    }
#pragma unroll
                    for (int st = 0; st < 2; ++st) {
                        const Frag<T> dx = to_frag<T>(x, st);
                        Frag<T> rest;
                        if constexpr (kParts == 2) rest = rest_frag<T>(x, st);
#pragma unroll
                        for (int t = 0; t < kCols; ++t) {
                            Frag<T> k = Tl::frag_t(k_cols, u * 32 + 16 * st, t);
                            if (kWalk == kCareful) zero_not_finite(k);
                            mma(dq[t], k, dx);
                            if constexpr (kParts == 2) mma(dq[t], k, rest);
                        }
                    }
                    if (sizeof(T) == 2 && kWalk != kCareful) read_ahead<2, kParts, 2 * kCols, 3>();
                }
                if (kWalk == kCareful) {
                    bool bad = false;
                    if (lane < Sh::kTile) bad = Tl::row_not_finite(kt, lane);
                    for (uint64_t left = __ballot(bad); left; left &= left - 1) {
                        const int key = __builtin_ctzll(left), j = key0 + key;
                        const bool see = j >= span.lo && j <= span.hi && (!a.docs || docs[key] == span.doc);
#pragma unroll
                        for (int t = 0; t < kCols; ++t)
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const float v = Tl::element(kt, key, 32 * t + 8 * (i / 4) + 4 * hi + i % 4);
                                if (see && !(__builtin_fabsf(v) < INFINITY)) dq[t][i] += v - v;  // its score is not finite either
                            }
                    }
                }
            }
            cur = following;
            buf ^= 1;
        }
    };
    auto walk_all = [&](auto which) __attribute__((always_inline)) {
        if constexpr (sizeof(T) == 2) {
            if (two_parts) run(which, std::integral_constant<int, 2>());
            else run(which, std::integral_constant<int, 1>());
        } else {
            run(which, std::integral_constant<int, 1>());
        }
    };
    walk_all(std::integral_constant<Walk, kMain>());
    lds_loads_done();  // also where no tile was walked: nothing may land in LDS after the block is gone
    bool bad = false;
#pragma unroll
    for (int t = 0; t < kCols; ++t) bad |= not_finite(dq[t]);
    if (__syncthreads_or(bad)) walk_all(std::integral_constant<Walk, kCareful>());

    if (!row_in) return;
    T* to = (T*)a.dq + out_row * a.D;
#pragma unroll
    for (int t = 0; t < kCols; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = 32 * t + 8 * j + 4 * hi;
            if (d >= a.D) continue;
            const f32x4_t v = {dq[t][4 * j] * a.scale, dq[t][4 * j + 1] * a.scale, dq[t][4 * j + 2] * a.scale, dq[t][4 * j + 3] * a.scale};
            if (share.parts > 1) *(f32x4_t*)(m.part_out + ((int64_t)split * a.batch * a.q_len * a.heads + out_row) * a.D + d) = v;
            else if constexpr (sizeof(T) == 2) *(u32x2_t*)(to + d) = u32x2_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
            else *(f32x4_t*)(to + d) = v;
        }
}

// ---------------------------------------------------------------------------------------------------------------
// dk, dv
// ---------------------------------------------------------------------------------------------------------------
// What a launch of the kernel forms.  At head_dim 256 the 256 accumulation registers of a lane hold dk and dv and nothing else, S and dP
// spill: one launch for each there, which forms S twice (five products instead of four; 8192 tokens, 8 heads over 4: 0.74 + 0.44 ms, together 2.7).
enum Grads { kDk = 1, kDv = 2, kBoth = 3 };

template <typename T, int DP, int GRADS>
struct DkvShape {
    static constexpr int kTile = 32;              // rows of a tile
    static constexpr int kKeys = 32 * kWaves;     // keys of a block
    typedef PanelTile<T, DP, kTile> Tl;
    typedef PanelTile<T, DP, kKeys> VTl;
    static constexpr int kTileBytes = Tl::kBytes;
    static constexpr int kBuf = 2 * kTileBytes + kStats * kTile * 4;
    // V's fragments are the ones that do not fit the registers of a lane (dk, dv, K, S, dP do; 256 at head_dim 128, 512 at 256): read from LDS
    static constexpr bool kVInLds = DP >= 128 && (GRADS & kDk);
    static constexpr int kVBytes = kVInLds ? VTl::kBytes : 0;
    static constexpr int kLds = 2 * kBuf + kVBytes;
    static constexpr int kWavesPerSimd = sizeof(T) == 2 && (DP <= 128 || GRADS == kDv) ? 2 : 1;
};

template <typename T, int DP, int MODE, int GRADS>
__global__ __launch_bounds__(kThreads, (DkvShape<T, DP, GRADS>::kWavesPerSimd)) void attention_dkv_kernel(MfmaArgs m) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    typedef DkvShape<T, DP, GRADS> Sh;
    typedef typename Sh::Tl Tl;
    constexpr int kSteps = DP / 16, kCols = DP / 32, kBuf = Sh::kBuf;
    const AttnArgs& a = m.a;
    const int lane = threadIdx.x & 63, wave = wave_index(), hi = lane >> 5;
    const int heads = (int)a.batch * a.kv_heads, bh = blockIdx.x % heads, split = blockIdx.y, block = blockIdx.x / heads;
    const int b = bh / a.kv_heads, kvh = bh % a.kv_heads;
    const int block0 = block * Sh::kKeys, block1 = min(block0 + Sh::kKeys, a.kv_len) - 1;
    const int wave0 = block0 + wave * 32, wave1 = wave0 + 31;
    const int key = wave0 + (lane & 31), key_in = key < a.kv_len, key_at = key_in ? key : a.kv_len - 1;

    // keys past the end get a document of their own; without documents every key and row has document 0
    const int doc = a.docs ? (key_in ? a.docs[(int64_t)b * a.kv_len + key] : -1) : 0;
    const int w_doc_min = wave_min_i32(doc), w_doc_max = wave_max_i32(doc);
    int blk_doc_min = 0, blk_doc_max = 0;
    if (a.docs) {
        __shared__ int range[kWaves][2];
        if (lane == 0) {
            range[wave][0] = w_doc_min;
            range[wave][1] = w_doc_max;
        }
        __syncthreads();
        blk_doc_min = __builtin_amdgcn_readfirstlane(min(min(range[0][0], range[1][0]), min(range[2][0], range[3][0])));
        blk_doc_max = __builtin_amdgcn_readfirstlane(max(max(range[0][1], range[1][1]), max(range[2][1], range[3][1])));
    }
    const int32_t* doc_min = a.docs ? m.row_docs.lowest + (int64_t)b * m.row_docs.tiles : nullptr;
    const int32_t* doc_max = a.docs ? m.row_docs.highest + (int64_t)b * m.row_docs.tiles : nullptr;
    const int prefix = a.prefix && a.prefix[b] > 0 ? a.prefix[b] : 0, off = a.kv_len - a.q_len;
    // first and last key of the interval of query s (documents aside): both grow with s
    auto lo_of = [&](int q) { return a.window > 0 ? max(0, q + off - a.window + 1) : 0; };
    auto hi_of = [&](int q) {
        int last = a.kv_len - 1;
        if (a.causal) last = min(last, max(q + off, prefix - 1));
        if (a.window > 0) last = min(last, q + off + a.window - 1);
        return last;
    };
    auto first_query = [&](int t) { return m.div(t * Sh::kTile); };
    auto last_query = [&](int t) { return m.div(min(t * Sh::kTile + Sh::kTile, m.rows) - 1); };

    const int row_tiles = (m.rows + Sh::kTile - 1) / Sh::kTile;
    auto active = [&](int t, int d0, int d1) {
        if (hi_of(last_query(t)) < block0 || lo_of(first_query(t)) > block1) return false;
        return !a.docs || (d1 >= max(0, blk_doc_min) && d0 <= blk_doc_max);
    };
    Share share = {1, 0, 0x7FFFFFFF};
    if (m.splits > 1) {
        share = share_of(count_tiles(0, row_tiles, doc_min, doc_max, active), split, m);
        if (split == 0 && threadIdx.x == 0) m.parts[bh * m.blocks + block] = share.parts;
        if (split >= share.parts) return;
    }

    if (a.D < DP) clear_lds(lds, Sh::kLds);
    Frag<T> kf[kSteps], vf[kSteps];
    const uint32_t vtile = lds_address(lds) + 2 * kBuf;
    if (Sh::kVInLds) {
        const T* v = (const T*)a.v.p + b * a.v.sb + kvh * a.v.sh;
        Sh::VTl::load(vtile, a.D, [&](int r) { return v + (int64_t)min(block0 + r, a.kv_len - 1) * a.v.ss; });
    }
    {
        const T* k = (const T*)a.k.p + b * a.k.sb + (int64_t)key_at * a.k.ss + kvh * a.k.sh;
        const T* v = (const T*)a.v.p + b * a.v.sb + (int64_t)key_at * a.v.ss + kvh * a.v.sh;
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) {
            kf[ks] = load_frag<T>(k, 16 * ks + 8 * hi, a.D);
            if (!Sh::kVInLds && (GRADS & kDk)) vf[ks] = load_frag<T>(v, 16 * ks + 8 * hi, a.D);
        }
    }
    const T* qbase = (const T*)a.q.p + b * a.q.sb + (int64_t)(kvh * a.group) * a.q.sh;
    const T* gbase = (const T*)a.d_out + ((int64_t)b * a.q_len * a.heads + kvh * a.group) * a.D;
    // 32 rows of a tile that are whole queries, at constant offsets within 2^31 bytes from the first: as in the forward
    const bool even = a.D == DP && 32 % a.group == 0 && a.q.ss < (1 << 22) && a.q.sh < (1 << 22) && a.heads * a.D < (1 << 22);
    const int per_tile = 32 / a.group, lane_s = Tl::lane_row() / a.group, lane_h = Tl::lane_row() % a.group;
    const uint32_t q_off = Tl::lane_offset((uint32_t)(lane_s * a.q.ss + lane_h * a.q.sh) * (uint32_t)sizeof(T));
    const uint32_t g_off = Tl::lane_offset((uint32_t)((lane_s * a.heads + lane_h) * a.D) * (uint32_t)sizeof(T));
    auto fetch = [&](int t, int buf) __attribute__((always_inline)) {
        const uint32_t qt = lds_address(lds) + buf * kBuf;
        if (even && (t + 1) * Sh::kTile <= m.rows && Tl::kLoadRows % a.group == 0) {
            const int64_t s0 = (int64_t)t * per_tile;
            Tl::load_even(qt, (const char*)(qbase + s0 * a.q.ss), q_off, [&](int r) { return (uint64_t)(r / a.group * a.q.ss * (int)sizeof(T)); });
            Tl::load_even(qt + Sh::kTileBytes, (const char*)(gbase + s0 * a.heads * a.D), g_off,
                          [&](int r) { return (uint64_t)(r / a.group * a.heads * a.D * (int)sizeof(T)); });
        } else {
            auto row_at = [&](int r) { return min(t * Sh::kTile + r, m.rows - 1); };
            Tl::load(qt, a.D, [&](int r) {
                const int s = m.div(row_at(r)), h = row_at(r) - s * a.group;
                return qbase + s * a.q.ss + h * a.q.sh;
            });
            Tl::load(qt + Sh::kTileBytes, a.D, [&](int r) {
                const int s = m.div(row_at(r)), h = row_at(r) - s * a.group;
                return gbase + ((int64_t)s * a.heads + h) * a.D;
            });
        }
        if (wave == 0) load16_to_lds(m.stats + ((int64_t)bh * row_tiles + t) * (kStats * 32) + lane * 4, qt + 2 * Sh::kTileBytes);
    };

    const typename Tl::Lane ln;
    typename Sh::VTl::Lane vl;
    vl.row = ln.row;
    vl.row2 = ln.row2;
    const typename Sh::VTl::Rows v_rows(vl, vtile + wave * 32 * Tl::kRowBytes);
    const ScoreScale sc = score_scale<MODE>(a);
    f32x16_t dk[kCols], dv[kCols];
    auto run = [&](auto which, auto active, int first, int end, Share share) __attribute__((always_inline)) {
        constexpr Walk kWalk = decltype(which)::value;
        if (kWalk != kRest) {
#pragma unroll
            for (int t = 0; t < kCols; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) dk[t][i] = dv[t][i] = 0.f;
        }
        TileWalk<decltype(active)> walk(first, end, doc_min, doc_max, active, share.skip, share.left);
        WalkTile cur = walk.next();
        int buf = 0;
        if (cur.t >= 0) fetch(cur.t, 0);
        while (cur.t >= 0) {
            lds_loads_done();
            __syncthreads();
            const WalkTile following = walk.next();
            if (following.t >= 0) fetch(following.t, buf ^ 1);
            const char* qt = lds + buf * kBuf;
            const char* gt = qt + Sh::kTileBytes;
            const uint32_t qa = lds_address(qt), ga = qa + Sh::kTileBytes;
            const float* stats = (const float*)(gt + Sh::kTileBytes);
            const int s0 = first_query(cur.t), s1 = last_query(cur.t);
            bool in = hi_of(s1) >= wave0 && lo_of(s0) <= wave1;
            bool full = lo_of(s1) <= wave0 && hi_of(s0) >= wave1 && (cur.t + 1) * Sh::kTile <= m.rows;
            if (a.docs) {
                in = in && cur.doc_max >= max(0, w_doc_min) && cur.doc_min <= w_doc_max;
                full = full && cur.doc_min == cur.doc_max && cur.doc_min == w_doc_min && cur.doc_min == w_doc_max && cur.doc_min >= 0;
            }
            if (in) {
                const typename Tl::Rows q_rows(ln, qa), g_rows(ln, ga);
                const typename Tl::Cols q_cols(ln, qa), g_cols(ln, ga);
                f32x16_t x, dp;
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = dp[i] = 0.f;
#pragma unroll
                for (int ks = 0; ks < kSteps; ++ks) {
                    mma(x, Tl::frag(q_rows, 0, ks), kf[ks]);
                    if constexpr (Sh::kVInLds) {
                        mma(dp, Tl::frag(g_rows, 0, ks), Sh::VTl::frag(v_rows, 0, ks));
                    } else if constexpr (GRADS & kDk) {
                        mma(dp, Tl::frag(g_rows, 0, ks), vf[ks]);
                    }
                }
                constexpr int kProducts = GRADS & kDk ? 2 : 1;
                if (sizeof(T) == 2) read_ahead<kProducts + Sh::kVInLds, kProducts, kSteps, 2>();
                typedef __attribute__((ext_vector_type(4))) int i32x4_t;
                auto stat4 = [&](RowStat which, int j) { return *(const f32x4_t*)(stats + which * Sh::kTile + 8 * j + 4 * hi); };
                auto stat4i = [&](RowStat which, int j) { return *(const i32x4_t*)(stats + which * Sh::kTile + 8 * j + 4 * hi); };
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x4_t delta = stat4(kDelta, j);
#pragma unroll
                    for (int i = 0; i < 4; ++i) dp[4 * j + i] -= delta[i];
                }
                if (MODE == kPlain) {
                } else if (sc.cap2 > 0.f) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float t = capped<MODE>(x[i], sc.mul);
                        x[i] = sc.cap2 * t;
                        dp[i] *= 1.f - t * t;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] *= sc.mul;
                }
                if (MODE != kPlain && a.slopes) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const f32x4_t slope2 = stat4(kSlope2, j);
                        const auto pos = stat4i(kPos, j);
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[4 * j + i] -= slope2[i] * __builtin_fabsf((float)(pos[i] - key));
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x4_t lse2 = stat4(kLse2, j);
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[4 * j + i] = __builtin_amdgcn_exp2f(MODE == kPlain ? __builtin_fmaf(x[4 * j + i], sc.mul, -lse2[i]) : x[4 * j + i] - lse2[i]);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) dp[i] *= x[i];
                if (!full) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const auto lo = stat4i(kFirst, j), keys = stat4i(kKeys, j), row_doc = stat4i(kDoc, j);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const bool see = (uint32_t)(key - lo[i]) <= (uint32_t)keys[i] && row_doc[i] == doc;
                            x[4 * j + i] = see ? x[4 * j + i] : 0.f;
                            dp[4 * j + i] = see ? dp[4 * j + i] : 0.f;
                        }
                    }
                }
                if constexpr (kWalk == kRest) {
                    take_rest(x);
                    take_rest(dp);
                }
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    const Frag<T> p = to_frag<T>(x, st), dx = to_frag<T>(dp, st);
#pragma unroll
                    for (int t = 0; t < kCols; ++t) {
                        if constexpr (GRADS & kDv) {
                            Frag<T> g = Tl::frag_t(g_cols, 16 * st, t);
                            if (kWalk != kMain) zero_not_finite(g);
                            mma(dv[t], g, p);
                        }
                        if constexpr (GRADS & kDk) {
                            Frag<T> q = Tl::frag_t(q_cols, 16 * st, t);
                            if (kWalk != kMain) zero_not_finite(q);
                            mma(dk[t], q, dx);
                        }
                    }
                }
                constexpr int kGrads = GRADS == kBoth ? 2 : 1;
                if (sizeof(T) == 2 && kWalk == kMain) read_ahead<2 * kGrads, kGrads, 2 * kCols, 2>();
                if (kWalk == kCareful) {
                    const bool bad = Tl::row_not_finite(hi ? gt : qt, lane & 31);
                    for (uint64_t left = __ballot(bad); left; left &= left - 1) {
                        const int which = __builtin_ctzll(left), r = which & 31;
                        const char* from = which >> 5 ? gt : qt;
                        const int32_t* of = (const int32_t*)stats + r;
                        const bool see = (uint32_t)(key - of[kFirst * 32]) <= (uint32_t)of[kKeys * 32] && of[kDoc * 32] == doc;
#pragma unroll
                        for (int t = 0; t < kCols; ++t)
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const float v = Tl::element(from, r, 32 * t + 8 * (i / 4) + 4 * hi + i % 4);
                                const bool add = see && !(__builtin_fabsf(v) < INFINITY);
                                dv[t][i] += add && which >= 32 ? v : 0.f;
                                dk[t][i] += add && which < 32 ? v - v : 0.f;
                            }
                    }
                }
            }
            cur = following;
            buf ^= 1;
        }
    };
    run(std::integral_constant<Walk, kMain>(), active, 0, row_tiles, share);
    lds_loads_done();  // also where no tile was walked: nothing may land in LDS after the block is gone
    bool bad = false;
#pragma unroll
    for (int t = 0; t < kCols; ++t) bad |= not_finite(dk[t]) || not_finite(dv[t]);
    if (__syncthreads_or(bad)) {
        run(std::integral_constant<Walk, kCareful>(), active, 0, row_tiles, share);
        __syncthreads();
    }
    if constexpr (sizeof(T) == 2) {
        // Without documents and a narrow window only the first keys have such rows.  A query's interval grows with the query and, once its window
        // has left the first key behind, shrinks (at the last keys): the shortest of a tile is at one of its ends.  The parts of a cut walk take
        // such tiles in turn, else the first part has them all (2048 tokens: 106 us instead of 97); with documents, where the tiles lie here and
        // there, each looks for them among its own, else in all tiles (2 x 8192 tokens in documents of 1024: 363 us instead of 335).  Where its own
        // tiles begin and end is looked up again here: kept in registers through the first walk it costs that up to 4 %.
        if (a.docs || block0 < kFewKeys || (a.window > 0 && a.window < kFewKeys)) {
            auto keys_of = [&](int q) { return hi_of(q) - lo_of(q); };
            auto few = [&](int t, int d0, int d1) {
                if ((!a.docs && share.parts > 1 && t % share.parts != split) || !active(t, d0, d1)) return false;
                const int q0 = first_query(t), q1 = last_query(t);
                return m.few ? any_has_few(m, b, q0, q1) : min(keys_of(q0), keys_of(q1)) < kFewKeys - 1;
            };
            int first = 0, end = row_tiles;
            if (a.docs && share.parts > 1) {
                TileWalk<decltype(active)> from(0, row_tiles, doc_min, doc_max, active, share.skip, 1);
                first = max(0, from.next().t);
                TileWalk<decltype(active)> to(first, row_tiles, doc_min, doc_max, active, share.left - 1, 1);
                end = to.next().t + 1;
            }
            run(std::integral_constant<Walk, kRest>(), few, first, end, Share{1, 0, 0x7FFFFFFF});
        }
    }

    if (!key_in) return;
    const int64_t out_row = ((int64_t)b * a.kv_len + key) * a.kv_heads + kvh, rows = a.batch * a.kv_len * a.kv_heads;
#pragma unroll
    for (int t = 0; t < kCols; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = 32 * t + 8 * j + 4 * hi;
            if (d >= a.D) continue;
            const f32x4_t u = {dk[t][4 * j] * a.scale, dk[t][4 * j + 1] * a.scale, dk[t][4 * j + 2] * a.scale, dk[t][4 * j + 3] * a.scale};
            const f32x4_t v = {dv[t][4 * j], dv[t][4 * j + 1], dv[t][4 * j + 2], dv[t][4 * j + 3]};
            if (share.parts > 1) {
                float* to = m.part_out + ((int64_t)split * 2 * rows + out_row) * a.D + d;
                if (GRADS & kDk) *(f32x4_t*)to = u;
                if (GRADS & kDv) *(f32x4_t*)(to + rows * a.D) = v;
            } else if constexpr (sizeof(T) == 2) {
                if (GRADS & kDk) *(u32x2_t*)((T*)a.dk + out_row * a.D + d) = u32x2_t{pack_bf16x2(u[0], u[1]), pack_bf16x2(u[2], u[3])};
                if (GRADS & kDv) *(u32x2_t*)((T*)a.dv + out_row * a.D + d) = u32x2_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
            } else {
                if (GRADS & kDk) *(f32x4_t*)((T*)a.dk + out_row * a.D + d) = u;
                if (GRADS & kDv) *(f32x4_t*)((T*)a.dv + out_row * a.D + d) = v;
            }
        }
}

struct JoinArgs {  // blockIdx.y: one of dq, dk, dv; the parts of its quads of elements
    void* to[3];
    const float* from[3];
    const int32_t* parts[3];
    int64_t quads[3], stride[3];  // stride: between the parts of one, in quads
    int length[3], heads[3], group[3], rows[3], blocks[3];  // rows: of a block
};

// the gradients of the blocks that were cut, four elements a thread
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_grad_join_kernel(JoinArgs j, int quads_per_row, int kv_heads) {
    const int w = blockIdx.y;
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= j.quads[w]) return;
    const int64_t row = i / quads_per_row, token = row / j.heads[w], b = token / j.length[w];
    const int head = (int)(row - token * j.heads[w]), at = (int)(token - b * j.length[w]);  // row of the key head: at * group + head % group
    const int block = (at * j.group[w] + head % j.group[w]) / j.rows[w];
    const int parts = j.parts[w][(b * kv_heads + head / j.group[w]) * j.blocks[w] + block];
    if (parts == 1) return;  // written by its block
    const f32x4_t* from = (const f32x4_t*)j.from[w] + i;
    f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int p = 0; p < parts; ++p) sum += from[p * j.stride[w]];
    T* to = (T*)j.to[w] + 4 * i;
    if constexpr (sizeof(T) == 2) *(u32x2_t*)to = u32x2_t{pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
    else *(f32x4_t*)to = sum;
}

// What the two kernels want to know of the rows, D = dO . (out + residual) among it -- a group of lanes per row of a key head, 16 bytes a
// lane -- and the document ranges of the tiles
constexpr int prepare_lanes(int DP, int per) { return (DP <= 128 ? 128 : DP) / per; }  // of a row
template <typename T, int DP, bool DOCS>
__global__ __launch_bounds__(kThreads) void attention_prepare_kernel(MfmaArgs m, int delta_blocks, int key_tile, int row_tile, int key_blocks, int row_blocks) {
    const AttnArgs& a = m.a;
    constexpr int kPer = 16 / (int)sizeof(T), kLanes = prepare_lanes(DP, kPer), kRows = kThreads / kLanes;
    if (!DOCS || (int)blockIdx.x < delta_blocks) {
        const int blocks = m.row_docs.tiles * 32 / kRows;  // of a key head
        const int bh = blockIdx.x / blocks, row = (blockIdx.x - bh * blocks) * kRows + threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
        const int at = row < m.rows ? row : m.rows - 1, b = bh / a.kv_heads, s = m.div(at), head = (bh - b * a.kv_heads) * a.group + at - s * a.group;
        const int64_t from = (((int64_t)b * a.q_len + s) * a.heads + head) * a.D + lane * kPer;
        float delta = 0.f;
        if (lane * kPer < a.D) {
            typedef __attribute__((ext_vector_type(kPer))) T vec;
            const vec gv = *(const vec*)((const T*)a.d_out + from), ov = *(const vec*)((const T*)a.out + from);
            vec rv = {};
            if (sizeof(T) == 2 && a.residual) rv = *(const vec*)((const T*)a.residual + from);
#pragma unroll
            for (int e = 0; e < kPer; ++e) delta += (float)gv[e] * ((float)ov[e] + (float)rv[e]);
        }
#pragma unroll
        for (int off = kLanes / 2; off > 0; off >>= 1) delta += __shfl_xor(delta, off, 64);
        if (lane < kStats) {
            const RowSpan span = row_span(a, b, s);
            const bool some = row < m.rows && span.hi >= span.lo;
            float v = delta;
            if (lane == kLse2) {
                const float lse = a.lse[((int64_t)b * a.heads + head) * a.q_len + s];
                v = !some || lse == -INFINITY ? INFINITY : lse * kLog2e;
            }
            if (lane == kSlope2) v = a.slopes ? a.slopes[head] * kLog2e : 0.f;
            if (lane == kPos) v = __int_as_float(s + a.kv_len - a.q_len);
            if (lane == kFirst) v = __int_as_float(some ? span.lo : 0x7FFFFFFF);
            if (lane == kKeys) v = __int_as_float(some ? span.hi - span.lo : 0);
            if (lane == kDoc) v = __int_as_float(span.doc);
            m.stats[((int64_t)bh * m.row_docs.tiles + row / 32) * (kStats * 32) + lane * 32 + row % 32] = v;
        }
        return;
    }
    const int block = blockIdx.x - delta_blocks;
    if (block < key_blocks)
        document_range(a.docs, a.kv_len, block, key_tile, m.key_docs.tiles, a.kv_len, 0, GroupDiv{0u, 0}, (int32_t*)m.key_docs.lowest,
                       (int32_t*)m.key_docs.highest);
    else if (block - key_blocks >= row_blocks)
        few_queries(a, block - key_blocks - row_blocks, (uint64_t*)m.few);
    else
        document_range(a.docs, a.kv_len, block - key_blocks, row_tile, m.row_docs.tiles, m.rows, a.kv_len - a.q_len, m.div,
                       (int32_t*)m.row_docs.lowest, (int32_t*)m.row_docs.highest);
}

// ---------------------------------------------------------------------------------------------------------------
int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

struct Cut {
    int blocks, splits, target;
};
// A mask leaves the blocks unequal walks (causal: the last rows see all keys, the first one).  The work of all blocks without a mask is
// thought of as `pieces` walks, and longer ones are cut, into parts of `shortest` tiles or more -- a part costs its sums in fp32 each
// way -- and 16 parts at most.
Cut cut(int64_t heads, int64_t blocks, int64_t tiles, int64_t shortest, int64_t pieces) {
    const int64_t share = (heads * blocks * tiles + pieces - 1) / pieces, longest = (tiles + 15) / 16;
    int64_t target = share > shortest ? share : shortest;
    target = target > longest ? target : longest;
    return {(int)blocks, tiles > target ? (int)((tiles + target - 1) / target) : 1, (int)target};
}

struct Plan {
    int key_tile, key_tiles, row_tiles;
    Cut dq, dkv;
    int64_t key_docs, row_docs, few_bytes, stats_bytes, dq_parts, dkv_parts, dq_bytes, dkv_bytes;
};
Plan plan(int dtype, int64_t batch, int64_t q_len, int64_t kv_len, int q_heads, int kv_heads, int head_dim) {
    Plan p;
    const int64_t rows = q_len * (q_heads / kv_heads), heads = batch * kv_heads, per = 32 * kWaves;
    p.key_tile = dtype == PICOMOE_BF16 ? 64 : 32;
    p.key_tiles = (int)((kv_len + p.key_tile - 1) / p.key_tile);
    p.row_tiles = (int)((rows + 31) / 32);
    // Pieces for each block that the chip holds at a time.  dq's longest walks go first, the short ones fill up behind them: with four
    // or eight pieces instead of two it takes 6 to 12 % more (16384 causal tokens: 1.59 and 1.72 ms; 4096 tokens, 16 heads, two batches:
    // 267, 302 and 300 us) and the join twice as long.  dk / dv, whose first blocks are the longest but all about as long as the
    // second ones, takes 2.88 ms with four, 2.65 with eight and as much with twelve (4096 tokens: 485 us with twelve, 443 with eight).
    const int64_t resident = head_dim <= 128 ? 512 : 256;
    p.dq = cut(heads, (rows + per - 1) / per, p.key_tiles, 8, 2 * resident);
    p.dkv = cut(heads, (kv_len + per - 1) / per, p.row_tiles, 16, 8 * resident);
    p.key_docs = round16(batch * p.key_tiles * 8);
    p.row_docs = round16(batch * p.row_tiles * 8);
    p.few_bytes = dtype == PICOMOE_BF16 ? round16(batch * few_words(q_len) * 8) : 0;
    p.stats_bytes = heads * p.row_tiles * (kStats * 32 * 4);
    p.dq_parts = p.dq.splits > 1 ? round16(heads * p.dq.blocks * 4) : 0;
    p.dkv_parts = p.dkv.splits > 1 ? round16(heads * p.dkv.blocks * 4) : 0;
    p.dq_bytes = p.dq.splits > 1 ? p.dq.splits * batch * q_len * q_heads * head_dim * 4 : 0;
    p.dkv_bytes = p.dkv.splits > 1 ? p.dkv.splits * 2 * batch * kv_len * kv_heads * head_dim * 4 : 0;
    return p;
}

template <typename T, int DP, int MODE>
int launch(MfmaArgs m, const Plan& p, hipStream_t s) {
    typedef DqShape<T, DP> Q;
    hipError_t e = allow_lds<attention_dq_kernel<T, DP, MODE>>(Q::kLds);
    constexpr int kOne = DP == 256 ? kDk : kBoth, kTwo = DP == 256 ? kDv : kBoth;  // the same: one launch
    if (e == hipSuccess) e = allow_lds<attention_dkv_kernel<T, DP, MODE, kOne>>(DkvShape<T, DP, kOne>::kLds);
    if (e == hipSuccess) e = allow_lds<attention_dkv_kernel<T, DP, MODE, kTwo>>(DkvShape<T, DP, kTwo>::kLds);
    if (e != hipSuccess) return PICOMOE_ERR_HIP_BASE + (int)e;
    const AttnArgs& a = m.a;
    const int64_t heads = a.batch * a.kv_heads, q_quads = a.batch * a.q_len * a.heads * (a.D / 4), k_quads = a.batch * a.kv_len * a.kv_heads * (a.D / 4);
    const int64_t join_blocks = ((q_quads > k_quads ? q_quads : k_quads) + kThreads - 1) / kThreads;
    const int64_t delta_blocks = heads * p.row_tiles * 32 / (kThreads / prepare_lanes(DP, 16 / (int)sizeof(T)));
    const int64_t key_ranges = a.docs ? a.batch * range_blocks(p.key_tiles) : 0, row_ranges = a.docs ? a.batch * range_blocks(p.row_tiles) : 0;
    const bool count_few = a.docs && sizeof(T) == 2;
    const int64_t few_ranges = count_few ? a.batch * few_blocks(a.q_len) : 0, prepare_blocks = delta_blocks + key_ranges + row_ranges + few_ranges;
    if (heads * p.dq.blocks > 0x7FFFFFFF || heads * p.dkv.blocks > 0x7FFFFFFF || join_blocks > 0x7FFFFFFF ||
        prepare_blocks > 0x7FFFFFFF)
        return PICOMOE_ERR_TOO_LARGE;
    char* ws = a.ws;
    auto take = [&](int64_t bytes) {
        char* at = ws;
        ws += bytes;
        return at;
    };
    int32_t *key_docs = (int32_t*)take(p.key_docs), *row_docs = (int32_t*)take(p.row_docs);
    uint64_t* few = (uint64_t*)take(p.few_bytes);
    int32_t *dq_parts = (int32_t*)take(p.dq_parts), *dkv_parts = (int32_t*)take(p.dkv_parts);
    m.stats = (float*)take(p.stats_bytes);
    float *dq_sums = (float*)take(p.dq_bytes), *dkv_sums = (float*)take(p.dkv_bytes);
    m.key_docs = {key_docs, key_docs + a.batch * p.key_tiles, p.key_tiles};
    m.row_docs = {row_docs, row_docs + a.batch * p.row_tiles, p.row_tiles};
    m.few = count_few ? few : nullptr;
    m.few_words = few_words(a.q_len);
    const auto prepare = a.docs ? attention_prepare_kernel<T, DP, true> : attention_prepare_kernel<T, DP, false>;
    prepare<<<(unsigned)prepare_blocks, kThreads, 0, s>>>(m, (int)delta_blocks, p.key_tile, 32, (int)key_ranges, (int)row_ranges);
    auto use = [&](const Cut& c, int32_t* parts, float* sums) {
        m.blocks = c.blocks;
        m.splits = c.splits;
        m.target = c.target;
        m.parts = parts;
        m.part_out = sums;
        return dim3((unsigned)(heads * c.blocks), (unsigned)c.splits);
    };
    const dim3 dkv_grid = use(p.dkv, dkv_parts, dkv_sums);
    // How much documents leave of the walks is not known here; half the length takes 364 us, joined, for 2 x 8192 tokens of documents of
    // about 1024, the whole 450, a third 391
    if (a.docs && m.target >= 32) m.target /= 2;
    attention_dkv_kernel<T, DP, MODE, kOne><<<dkv_grid, kThreads, DkvShape<T, DP, kOne>::kLds, s>>>(m);
    if (kTwo != kOne) attention_dkv_kernel<T, DP, MODE, kTwo><<<dkv_grid, kThreads, DkvShape<T, DP, kTwo>::kLds, s>>>(m);
    const dim3 dq_grid = use(p.dq, dq_parts, dq_sums);
    attention_dq_kernel<T, DP, MODE><<<dq_grid, kThreads, Q::kLds, s>>>(m);
    JoinArgs j = {};
    unsigned n = 0;
    auto join = [&](void* to, const float* from, const int32_t* parts, int64_t quads, int64_t stride, int length, int of_heads, int group, int rows, int blocks) {
        j.to[n] = to; j.from[n] = from; j.parts[n] = parts; j.quads[n] = quads; j.stride[n] = stride;
        j.length[n] = length; j.heads[n] = of_heads; j.group[n] = group; j.rows[n] = rows; j.blocks[n] = blocks;
        ++n;
    };
    if (p.dq.splits > 1) join(a.dq, dq_sums, dq_parts, q_quads, q_quads, a.q_len, a.heads, a.group, 32 * kWaves, p.dq.blocks);
    if (p.dkv.splits > 1) {
        join(a.dk, dkv_sums, dkv_parts, k_quads, 2 * k_quads, a.kv_len, a.kv_heads, 1, 32 * kWaves, p.dkv.blocks);
        join(a.dv, dkv_sums + 4 * k_quads, dkv_parts, k_quads, 2 * k_quads, a.kv_len, a.kv_heads, 1, 32 * kWaves, p.dkv.blocks);
    }
    if (n > 0) attention_grad_join_kernel<T><<<dim3((unsigned)join_blocks, n), kThreads, 0, s>>>(j, a.D / 4, a.kv_heads);
    return picomoe_launch_status();
}

template <typename T, int DP>
int launch_for(const MfmaArgs& m, const Plan& p, hipStream_t s) {
    const ScoreMode mode = score_mode(m.a, m.a.softcap == 0.f && !m.a.slopes);
    if (mode == kPlain) return launch<T, DP, kPlain>(m, p, s);
    if constexpr (sizeof(T) == 2)
        if (mode == kFast) return launch<T, DP, kFast>(m, p, s);
    return launch<T, DP, kAccurate>(m, p, s);
}

}  // namespace

int64_t attention_mfma_bwd_workspace(int dtype, int64_t batch, int64_t q_len, int64_t kv_len, int q_heads, int kv_heads, int head_dim) {
    const Plan p = plan(dtype, batch, q_len, kv_len, q_heads, kv_heads, head_dim);
    return p.key_docs + p.row_docs + p.few_bytes + p.stats_bytes + p.dq_parts + p.dkv_parts + p.dq_bytes + p.dkv_bytes + 16;
}

int attention_mfma_bwd(const AttnArgs& a, hipStream_t s) {
    const Plan p = plan(a.dtype, a.batch, a.q_len, a.kv_len, a.heads, a.kv_heads, a.D);
    MfmaArgs m = {};
    m.a = a;
    m.div = group_div(a.group);
    m.rows = a.q_len * a.group;
    if (a.D > 128) return launch_for<__bf16, 256>(m, p, s);
    if (a.dtype == PICOMOE_BF16) return a.D <= 64 ? launch_for<__bf16, 64>(m, p, s) : launch_for<__bf16, 128>(m, p, s);
    return a.D <= 64 ? launch_for<float, 64>(m, p, s) : launch_for<float, 128>(m, p, s);
}
