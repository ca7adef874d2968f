// Pieces shared by the MFMA attention kernels (forward, dq, dk + dv): fragments, LDS tiles, the walk over tiles that the masks leave.
//
// Every product runs on 32 x 32 x 16 blocks (bf16: one v_mfma_f32_32x32x16_bf16; fp32: eight v_mfma_f32_32x32x2_f32 on the same
// fragment layout): operand fragments hold 8 consecutive k of one row, k = 8 * (lane / 32) + e, row = lane % 32; results hold
// column lane % 32 and rows 8 * (i / 4) + 4 * (lane / 32) + i % 4, i = 0 .. 15.  The first products of an attention are formed
// transposed -- S^T[key, query] in the forward and dq kernels, S[query, key] in the dk / dv kernel -- so that eight consecutive
// accumulators of a lane are, as they lie, the fragment of P (or dx) for the product that follows, with its k (keys or queries)
// in the order 16 s + {4 hi + 0..3, 8 + 4 hi + 0..3}; the other operand is read from LDS in that order.  P never passes through LDS.
#pragma once
#include "attention.h"
#include "lds.h"

namespace {

constexpr int kThreads = 256, kWaves = 4;

template <typename T>
struct Frag;
template <>
struct Frag<__bf16> {
    bf16x8_t v;
};
template <>
struct Frag<float> {
    float v[8];
};

__device__ __forceinline__ void mma(f32x16_t& c, const Frag<__bf16>& a, const Frag<__bf16>& b) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16_t& c, const Frag<float>& a, const Frag<float>& b) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[e], b.v[e], c, 0, 0, 0);
}

// Order of a run of STEPS steps of READS LDS reads and MFMAS products each: the reads AHEAD steps in front of the products that take
// them.  Left to itself the compiler reads, waits and multiplies step by step, and two wavefronts per SIMD do not hide that.
template <int READS, int MFMAS, int STEPS, int AHEAD>
__device__ __forceinline__ void read_ahead() {
    constexpr int kRead = 0x100, kMfma = 0x8;
    __builtin_amdgcn_sched_group_barrier(kRead, READS * AHEAD, 0);
#pragma unroll
    for (int i = 0; i < STEPS - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(kMfma, MFMAS, 0);
        __builtin_amdgcn_sched_group_barrier(kRead, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(kMfma, MFMAS * AHEAD, 0);
}

// eight accumulators -> the fragment of the next product.  bf16: P in [0, 2^8] and dx are rounded to bf16 here, a relative
// error of at most 2^-8 per term of the sums over keys (queries); the normaliser sums the unrounded P.
template <typename T>
__device__ __forceinline__ Frag<T> to_frag(const f32x16_t& c, int half);
template <>
__device__ __forceinline__ Frag<__bf16> to_frag<__bf16>(const f32x16_t& c, int half) {
    u32x4_t w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(c[8 * half + 2 * i], c[8 * half + 2 * i + 1]);
    return {__builtin_bit_cast(bf16x8_t, w)};
}
template <>
__device__ __forceinline__ Frag<float> to_frag<float>(const f32x16_t& c, int half) {
    Frag<float> f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = c[8 * half + i];
    return f;
}

// what to_frag left of them, rounded to bf16 in turn: together they are off by 2^-16 of a term
template <typename T>
__device__ __forceinline__ Frag<T> rest_frag(const f32x16_t& c, int half) {
    static_assert(sizeof(T) == 2);
    u32x4_t w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = c[8 * half + 2 * i], b = c[8 * half + 2 * i + 1];
        w[i] = pack_bf16x2(a - (float)(__bf16)a, b - (float)(__bf16)b);
    }
    return {__builtin_bit_cast(bf16x8_t, w)};
}

// A kernel's walk over its tiles.  kMain.  kCareful, instead of it where its sums are not finite: values that are not finite are kept out of the
// products, where 0 * inf would reach rows that do not see them, and added one by one to the rows that do.  Both, in bf16, take P and dx in two
// parts (to_frag and rest_frag) in blocks that hold rows with few keys -- the first ones of a sequence or of a document, short documents,
// narrow windows --: 6 batches of two tokens have dq to 0.0017 with it, 0.0034 without (the rounding of dq itself: 0.0017).  dk / dv, whose
// registers two parts would spill (650 and more), adds what to_frag left in a second walk over the tiles of such rows, kRest.
enum Walk { kMain, kCareful, kRest };
constexpr int kFewKeys = 128;
__device__ __forceinline__ void take_rest(f32x16_t& c) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float v = c[i] - (float)(__bf16)c[i];
        c[i] = __builtin_fabsf(v) < INFINITY ? v : 0.f;
    }
}

// eight elements of a global row from column col on; zeros from column D on
template <typename T>
__device__ __forceinline__ Frag<T> load_frag(const T* row, int col, int D) {
    Frag<T> f;
    if constexpr (sizeof(T) == 2) {
        f.v = col < D ? *(const bf16x8_t*)(row + col) : bf16x8_t{};
    } else {
        const f32x4_t z = {0.f, 0.f, 0.f, 0.f};
        const f32x4_t a = col < D ? *(const f32x4_t*)(row + col) : z, b = col < D ? *(const f32x4_t*)(row + col + 4) : z;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f.v[i] = a[i];
            f.v[4 + i] = b[i];
        }
    }
    return f;
}

template <typename T>
__device__ __forceinline__ float frag_dot(const Frag<T>& a, const Frag<T>& b) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s += (float)a.v[e] * (float)b.v[e];
    return s;
}

__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }
__device__ __forceinline__ const char* uniform(const void* p) {
    const uint64_t v = (uint64_t)(uintptr_t)p;
    return (const char*)(uintptr_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
                                    (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v));
}
// keeps the compiler from taking an address apart into what is uniform and what is not, one addition per LDS read
__device__ __forceinline__ uint32_t whole(uint32_t v) {
    asm("" : "+v"(v));
    return v;
}

// A 16-byte (4-byte) direct-to-LDS load as an instruction sequence that the compiler does not look into: lane l lands at
// lds + 16 l (4 l); lanes that are switched off leave their place alone.  With the builtin the compiler waits for all loads in
// front of every LDS read that it cannot prove disjoint, so that nothing would be in flight under the products.  The kernels
// wait themselves, with lds_loads_done() and a barrier.  M0 is written here and cannot be named as clobbered: nothing else in
// these kernels may use it (the Makefile looks).
__device__ __forceinline__ uint32_t lds_address(const char* l) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)l; }
__device__ __forceinline__ void load16_to_lds(const void* from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(from) : "memory");
}
__device__ __forceinline__ void load4_to_lds(const void* from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(from) : "memory");
}
// a uniform base and 32 bits of offset per lane: no vector arithmetic for the address
__device__ __forceinline__ void load16_to_lds(const char* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void lds_loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// zeros over a block's dynamic LDS: rows narrower than DP are padded by what no load writes
__device__ __forceinline__ void clear_lds(char* lds, int bytes) {
    for (int i = threadIdx.x * 16; i < bytes; i += kThreads * 16) *(u32x4_t*)(lds + i) = u32x4_t{0u, 0u, 0u, 0u};
    __syncthreads();
}

// Tiles in LDS: groups of columns 128 bytes wide (64 bf16, 32 fp32), in a group ROWS rows of eight 16-byte chunks, chunk c of a row at
// c ^ swizzle(row).  The 16 rows that a ds_read_b128 serves at a time, and the 4 rows x 64 bytes of a transposing read, then lie on
// different banks; the fragments of a tile are at constant distances from eight addresses of a lane (rows of the tile's whole width: from
// sixteen).  For the forward, which has the registers: with the panels below one new token over 32768 keys took 239 us, not 205.
template <typename T, int DP, int ROWS>
struct Tile {
    static constexpr int kSize = (int)sizeof(T), kPerChunk = 16 / kSize, kRowBytes = 128, kGroupCols = 128 / kSize;
    static constexpr int kGroups = DP / kGroupCols, kStride = ROWS * kRowBytes, kBytes = kGroups * kStride;
    typedef __attribute__((address_space(3))) const bf16x8_t lds_bf16x8;
    typedef __attribute__((address_space(3))) const f32x4_t lds_f32x4;
    typedef __attribute__((address_space(3))) const float lds_f32;

    __device__ static __forceinline__ uint32_t swizzle(int row) { return (((row >> 1) & 1) << 2) | ((row >> 2) & 3); }
    __device__ static __forceinline__ uint32_t at(int row, int col) {
        return col / kGroupCols * kStride + row * kRowBytes + (((uint32_t)(col % kGroupCols / kPerChunk) ^ swizzle(row)) << 4) + col % kPerChunk * kSize;
    }

    // this lane's offsets: [16 columns of a group][half of eight elements] of row lane % 32; of the transposed tile
    struct Lane {
        uint32_t row[kGroupCols / 16][kSize / 2], col[2][2];
        __device__ __forceinline__ Lane() {
            const int lane = threadIdx.x & 63, hi = lane >> 5;
#pragma unroll
            for (int g = 0; g < kGroupCols / 16; ++g)
#pragma unroll
                for (int h = 0; h < kSize / 2; ++h) row[g][h] = at(lane & 31, 16 * g + 8 * hi + 4 * h);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int up = 0; up < 2; ++up) {
                    if (kSize == 2)  // [32 columns of a group][rows + 8]; a transposing read: lane l of 16 gives the address of 4 elements
                                     // of row l / 4 and gets column l of the 4 rows
                        col[i][up] = at(4 * hi + ((lane >> 2) & 3) + 8 * up, 32 * i + 16 * ((lane >> 4) & 1) + 4 * (lane & 3));
                    else             // [rows + 2][rows + 8]
                        col[i][up] = at(4 * hi + 2 * i + 8 * up, lane & 31);
                }
        }
    };

    // the same in the tile at LDS address `tile`
    struct Rows {
        uint32_t at[kGroupCols / 16][kSize / 2];
        __device__ __forceinline__ Rows(const Lane& l, uint32_t tile) {
#pragma unroll
            for (int g = 0; g < kGroupCols / 16; ++g)
#pragma unroll
                for (int h = 0; h < kSize / 2; ++h) at[g][h] = whole(l.row[g][h] + tile);
        }
    };
    struct Cols {
        uint32_t at[2][2];
        __device__ __forceinline__ Cols(const Lane& l, uint32_t tile) {
#pragma unroll
            for (int i = 0; i < 4; ++i) at[i / 2][i % 2] = whole(l.col[i / 2][i % 2] + tile);
        }
    };

    // rows row0 (a multiple of 32) + lane % 32, elements 16 ks + 8 hi ..
    __device__ static __forceinline__ Frag<T> frag(const Rows& r, int row0, int ks) {
        constexpr int kPer = kGroupCols / 16;
        Frag<T> f;
        const uint32_t off = row0 * kRowBytes + ks / kPer * kStride;
        if constexpr (kSize == 2) {
            f.v = *(lds_bf16x8*)(uintptr_t)(r.at[ks % kPer][0] + off);
        } else {
            const f32x4_t a = *(lds_f32x4*)(uintptr_t)(r.at[ks % kPer][0] + off), b = *(lds_f32x4*)(uintptr_t)(r.at[ks % kPer][1] + off);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f.v[i] = a[i];
                f.v[4 + i] = b[i];
            }
        }
        return f;
    }

    // the tile transposed: column 32 t + lane % 32, rows row0 (a multiple of 16) + {4 hi + 0..3, 8 + 4 hi + 0..3}
    __device__ static __forceinline__ Frag<T> frag_t(const Cols& c, int row0, int t) {
        constexpr int kPer = kGroupCols / 32;
        Frag<T> f;
        const uint32_t off = row0 * kRowBytes + t / kPer * kStride;
        if constexpr (kSize == 2) {
            typedef __attribute__((ext_vector_type(4))) short s16x4_t;
            typedef __attribute__((ext_vector_type(8))) short s16x8_t;
            typedef __attribute__((address_space(3))) s16x4_t lds4;
            const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(uintptr_t)(c.at[t % kPer][0] + off));
            const s16x4_t up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(uintptr_t)(c.at[t % kPer][1] + off));
            const s16x8_t v = {lo[0], lo[1], lo[2], lo[3], up[0], up[1], up[2], up[3]};
            f.v = __builtin_bit_cast(bf16x8_t, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) f.v[e] = *(lds_f32*)(uintptr_t)(c.at[(e >> 1) & 1][e >> 2] + off + (e & 1) * kRowBytes);
        }
        return f;
    }

    // Staging with direct-to-LDS loads of 1 KB, 8 rows of a group each.  Columns from D on are left as they are (zeros: clear_lds).
    // row_of(r): where row r of the tile is.
    template <typename F>
    __device__ static __forceinline__ void load(uint32_t tile, int D, F row_of) {
        const int lane = threadIdx.x & 63, wave = wave_index();
#pragma unroll
        for (int i = 0; i < kGroups * ROWS / 8 / kWaves; ++i) {
            const int unit = i * kWaves + wave, group = unit % kGroups, r0 = unit / kGroups * 8, row = r0 + lane / 8;
            const int chunk = (int)((uint32_t)(lane % 8) ^ swizzle(row)), col = group * kGroupCols + chunk * kPerChunk;
            if (col < D) load16_to_lds(row_of(row) + col, tile + group * kStride + r0 * kRowBytes);
        }
    }
    // The same for rows `stride` bytes apart from base on, D == DP; rows of a tile lie within 2^31 bytes.  A lane's offset depends on the
    // half of 16 rows, which a wavefront keeps from load to load (kGroups < kWaves) or changes with each.
    struct Source {
        uint32_t off[kGroups < kWaves ? 1 : 2];
        __device__ __forceinline__ explicit Source(uint32_t stride) {
            const int lane = threadIdx.x & 63;
#pragma unroll
            for (int i = 0; i < (kGroups < kWaves ? 1 : 2); ++i) {
                const int half = kGroups < kWaves ? wave_index() / kGroups & 1 : i;
                off[i] = lane / 8 * stride + (((uint32_t)(lane % 8) ^ swizzle(8 * half + lane / 8)) << 4);
            }
        }
    };
    __device__ static __forceinline__ void load_even(uint32_t tile, const char* base, uint32_t stride, const Source& src) {
        static_assert((kWaves % kGroups == 0 && (kWaves / kGroups) % 2 == 0) || kGroups == kWaves, "a wavefront's half of 16 rows");
        const int wave = wave_index();
#pragma unroll
        for (int i = 0; i < kGroups * ROWS / 8 / kWaves; ++i) {
            const int unit = i * kWaves + wave, group = unit % kGroups, r0 = unit / kGroups * 8;
            load16_to_lds(uniform(base + (uint64_t)(r0 * stride) + group * kRowBytes), src.off[kGroups < kWaves ? 0 : i & 1],
                          tile + group * kStride + r0 * kRowBytes);
        }
    }
    __device__ static __forceinline__ float element(const char* tile, int row, int col) { return to_f32(*(const T*)(tile + at(row, col))); }
    // whether row `row` holds a value that is not finite
    __device__ static __forceinline__ bool row_not_finite(const char* tile, int row) {
        bool bad = false;
        for (int c = 0; c < DP; ++c) bad |= !(__builtin_fabsf(element(tile, row, c)) < INFINITY);
        return bad;
    }
};

// The same tiles in panels of 16 columns, in a panel ROWS rows of 32 (fp32: 64) bytes in 16-byte chunks, chunk c of a row at
// c ^ swizzle(row); 128 bytes between panels.  Every fragment is at a constant distance from a lane's first: three address registers
// instead of eight.  For the backward, where the eight spill -- and a reload from scratch waits for the tile in flight -- although the
// loads touch 32-byte pieces of rows: dk / dv of 16384 tokens x 16 heads took 3.9 ms against 4.3.
template <typename T, int DP, int ROWS>
struct PanelTile {
    static constexpr int kSize = (int)sizeof(T), kPerChunk = 16 / kSize, kRowBytes = 16 * kSize, kRowChunks = kSize;  // of a panel
    static constexpr int kPanels = DP / 16, kStride = ROWS * kRowBytes + 128, kBytes = kPanels * kStride;
    typedef __attribute__((address_space(3))) const bf16x8_t lds_bf16x8;
    typedef __attribute__((address_space(3))) const f32x4_t lds_f32x4;
    typedef __attribute__((address_space(3))) const float lds_f32;

    __device__ static __forceinline__ uint32_t swizzle(int row) { return kSize == 2 ? (row >> 3) & 1 : (row >> 2) & 3; }
    __device__ static __forceinline__ uint32_t at(int row, int col) {
        return col / 16 * kStride + row * kRowBytes + (((uint32_t)(col % 16 / kPerChunk) ^ swizzle(row)) << 4) + col % kPerChunk * kSize;
    }

    // this lane's offsets: fragments of rows lane % 32, and of the transposed tile
    struct Lane {
        uint32_t row, row2, col, col2;
        __device__ __forceinline__ Lane() {
            const int lane = threadIdx.x & 63, hi = lane >> 5;
            row = at(lane & 31, hi * 8);
            row2 = row ^ 16;  // fp32: the second half of the eight
            if (kSize == 2) {
                // a transposing read: lane l of 16 gives the address of 4 elements of row l / 4 and gets column l of the 4 rows
                col = at(4 * hi + ((lane >> 2) & 3), 16 * ((lane >> 4) & 1) + 4 * (lane & 3));
                col2 = at(4 * hi + ((lane >> 2) & 3) + 8, 16 * ((lane >> 4) & 1) + 4 * (lane & 3));
            } else {
                col = at(4 * hi, lane & 31);
                col2 = at(4 * hi + 8, lane & 31);
            }
        }
    };

    // the same in the tile at LDS address `tile`
    struct Rows {
        uint32_t at, at2;
        __device__ __forceinline__ Rows(const Lane& l, uint32_t tile) : at(whole(l.row + tile)), at2(kSize == 2 ? 0 : whole(l.row2 + tile)) {}
    };
    struct Cols {
        uint32_t at, at2;
        __device__ __forceinline__ Cols(const Lane& l, uint32_t tile) : at(whole(l.col + tile)), at2(whole(l.col2 + tile)) {}
    };

    // rows row0 (a multiple of 32) + lane % 32, elements 16 ks + 8 hi ..
    __device__ static __forceinline__ Frag<T> frag(const Rows& r, int row0, int ks) {
        Frag<T> f;
        const uint32_t off = row0 * kRowBytes + ks * kStride;
        if constexpr (kSize == 2) {
            f.v = *(lds_bf16x8*)(uintptr_t)(r.at + off);
        } else {
            const f32x4_t a = *(lds_f32x4*)(uintptr_t)(r.at + off), b = *(lds_f32x4*)(uintptr_t)(r.at2 + off);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f.v[i] = a[i];
                f.v[4 + i] = b[i];
            }
        }
        return f;
    }

    // the tile transposed: column 32 t + lane % 32, rows row0 (a multiple of 16) + {4 hi + 0..3, 8 + 4 hi + 0..3}
    __device__ static __forceinline__ Frag<T> frag_t(const Cols& c, int row0, int t) {
        Frag<T> f;
        const uint32_t off = row0 * kRowBytes + 2 * t * kStride;
        if constexpr (kSize == 2) {
            typedef __attribute__((ext_vector_type(4))) short s16x4_t;
            typedef __attribute__((ext_vector_type(8))) short s16x8_t;
            typedef __attribute__((address_space(3))) s16x4_t lds4;
            const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(uintptr_t)(c.at + off));
            const s16x4_t up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(uintptr_t)(c.at2 + off));
            const s16x8_t v = {lo[0], lo[1], lo[2], lo[3], up[0], up[1], up[2], up[3]};
            f.v = __builtin_bit_cast(bf16x8_t, v);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f.v[e] = *(lds_f32*)(uintptr_t)(c.at + off + e * kRowBytes);
                f.v[4 + e] = *(lds_f32*)(uintptr_t)(c.at2 + off + e * kRowBytes);
            }
        }
        return f;
    }

    // Staging with direct-to-LDS loads of 1 KB, a panel's next 32 (fp32: 16) rows each; a wavefront takes neighbouring panels, so
    // that the lines it touches are used whole.  Columns from D on are left as they are (zeros: clear_lds).  row_of(r): where row r is.
    static constexpr int kLoadRows = 64 / kRowChunks, kMine = kPanels / kWaves;
    template <typename F>
    __device__ static __forceinline__ void load(uint32_t tile, int D, F row_of) {
        const int lane = threadIdx.x & 63, wave = wave_index();
#pragma unroll
        for (int r0 = 0; r0 < ROWS; r0 += kLoadRows) {
            const int row = r0 + lane / kRowChunks;
            const uint32_t chunk = (uint32_t)(lane % kRowChunks) ^ swizzle(row);
            const char* from = (const char*)row_of(row) + chunk * 16;
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const int panel = wave * kMine + i;
                if (panel * 16 + (int)chunk * kPerChunk < D) load16_to_lds(from + panel * kRowBytes, tile + panel * kStride + r0 * kRowBytes);
            }
        }
    }
    // The same for D == DP and rows at constant offsets from a uniform base: `off(lane's row of the first kLoadRows)`, and r0 rows on
    // `step(r0)` bytes further.
    __device__ static __forceinline__ uint32_t lane_offset(uint32_t row_offset) {
        const int lane = threadIdx.x & 63;
        return row_offset + (((uint32_t)(lane % kRowChunks) ^ swizzle(lane / kRowChunks)) << 4);
    }
    __device__ static __forceinline__ int lane_row() { return (int)(threadIdx.x & 63) / kRowChunks; }
    template <typename F>
    __device__ static __forceinline__ void load_even(uint32_t tile, const char* base, uint32_t offset, F step) {
        const int wave = wave_index();
#pragma unroll
        for (int r0 = 0; r0 < ROWS; r0 += kLoadRows)
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const int panel = wave * kMine + i;
                load16_to_lds(uniform(base + step(r0) + panel * kRowBytes), offset, tile + panel * kStride + r0 * kRowBytes);
            }
    }
    __device__ static __forceinline__ float element(const char* tile, int row, int col) { return to_f32(*(const T*)(tile + at(row, col))); }
    // whether row `row` holds a value that is not finite
    __device__ static __forceinline__ bool row_not_finite(const char* tile, int row) {
        bool bad = false;
        for (int c = 0; c < DP; ++c) bad |= !(__builtin_fabsf(element(tile, row, c)) < INFINITY);
        return bad;
    }
};

template <typename T>
__device__ __forceinline__ void zero_not_finite(Frag<T>& f) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (!(__builtin_fabsf((float)f.v[e]) < INFINITY)) f.v[e] = (T)0.f;
}

__device__ __forceinline__ bool not_finite(const f32x16_t& c) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 16; ++i) bad |= !(__builtin_fabsf(c[i]) < INFINITY);
    return bad;
}

// both halves of a wavefront: what lanes l and l + 32 hold
__device__ __forceinline__ float other_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float other_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ int wave_min_i32(int v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const int o = __shfl_xor(v, off, 64);
        v = o < v ? o : v;
    }
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max_i32(int v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const int o = __shfl_xor(v, off, 64);
        v = o > v ? o : v;
    }
    return __builtin_amdgcn_readfirstlane(v);
}

// r / group for the rows of a key head, r < 2^31: a multiplication (exact: mul = floor(2^(31 + shift) / group) + 1, 2^shift >= group)
struct GroupDiv {
    uint32_t mul;
    int shift;
    __device__ __forceinline__ int operator()(int r) const { return shift == 0 ? r : (int)(__umulhi((uint32_t)r, mul) >> (shift - 1)); }
};
inline GroupDiv group_div(int group) {
    int shift = 0;
    while ((1 << shift) < group) ++shift;
    return {shift == 0 ? 0u : (uint32_t)(((uint64_t)1 << (31 + shift)) / (uint32_t)group + 1), shift};
}

struct DocRanges {  // lowest and highest document of every tile: [batch, tiles], -1 among them where a token has no document
    const int32_t *lowest, *highest;
    int tiles;
};

struct MfmaArgs {
    AttnArgs a;
    GroupDiv div;
    int rows;  // of a key head: q_len * group
    // Forward and dq: row blocks that walk key tiles; dk / dv: key blocks that walk row tiles.  A block whose walk is longer than
    // `target` tiles is cut into at most `splits` parts of consecutive tiles; how many is noted in parts.
    int blocks, splits, target;
    int32_t* parts;
    float* part_out;
    float* part_lse;
    DocRanges key_docs, row_docs;
    const uint64_t* few;  // bf16 with documents: a bit for each query, words of 64 per batch element (few_queries); else NULL
    int few_words;
    float* stats;  // backward: [key heads][row tiles of 32][kStats][32], see RowStat
};

// What the backward knows of a row, in LDS by a kind and a row of the tile.  Rows that see nothing, and those past the end: kFirst is
// INT_MAX, kKeys 0 -- no key is that far -- and kLse2 +inf, which makes P zero.
enum RowStat { kLse2, kDelta, kSlope2, kPos, kFirst, kKeys, kDoc, kStats = 8 };  // from kPos on: int32

// what a set of query rows may see, and which documents it has; of a wavefront's rows that are `in`
struct Reach {
    int lo_min, lo_max, hi_min, hi_max, doc_min, doc_max;
};
__device__ __forceinline__ Reach wave_reach(bool in, const RowSpan& span) {
    Reach w;
    w.lo_min = wave_min_i32(in ? span.lo : 0x7FFFFFFF);
    w.hi_max = wave_max_i32(in ? span.hi : -1);
    w.lo_max = wave_max_i32(in ? span.lo : 0x7FFFFFFF);
    w.hi_min = wave_min_i32(in ? span.hi : -1);
    w.doc_min = wave_min_i32(in ? span.doc : 0x7FFFFFFF);
    w.doc_max = wave_max_i32(in ? span.doc : -1);
    return w;
}
// of all wavefronts of a block, lo_max and hi_min aside; and whether `flag` holds in one of them
__device__ __forceinline__ Reach block_reach(const Reach& w, bool& flag) {
    __shared__ int lds[kWaves][5];
    const int at = wave_index();
    if ((threadIdx.x & 63) == 0) {
        lds[at][0] = w.lo_min;
        lds[at][1] = w.hi_max;
        lds[at][2] = w.doc_min;
        lds[at][3] = w.doc_max;
        lds[at][4] = flag;
    }
    __syncthreads();
    Reach blk = w;
    int any = 0;
    for (int i = 0; i < kWaves; ++i) {
        blk.lo_min = min(blk.lo_min, lds[i][0]);
        blk.hi_max = max(blk.hi_max, lds[i][1]);
        blk.doc_min = min(blk.doc_min, lds[i][2]);
        blk.doc_max = max(blk.doc_max, lds[i][3]);
        any |= lds[i][4];
    }
    blk.lo_min = __builtin_amdgcn_readfirstlane(blk.lo_min);
    blk.hi_max = __builtin_amdgcn_readfirstlane(blk.hi_max);
    blk.doc_min = __builtin_amdgcn_readfirstlane(blk.doc_min);
    blk.doc_max = __builtin_amdgcn_readfirstlane(blk.doc_max);
    flag = __builtin_amdgcn_readfirstlane(any) != 0;
    return blk;
}

// The walk over the tiles of [first, end) that pass `active(t, lowest document, highest document)`, 64 at a time, the first `skip` of
// those left out and `left` taken; the same in every wave of a block.  The documents of a tile come with it: a load of them where
// they are needed would wait for the next tile, which is in flight by then.
struct WalkTile {
    int t, doc_min, doc_max;  // t < 0: none
};
template <typename F>
struct TileWalk {
    F active;
    const int32_t *lowest, *highest;  // NULL: no documents
    int base, end, skip, left, doc_min, doc_max;
    uint64_t mask;
    __device__ __forceinline__ TileWalk(int first, int end_, const int32_t* lowest_, const int32_t* highest_, F f, int skip_, int left_)
        : active(f), lowest(lowest_), highest(highest_), base(first - 64), end(end_), skip(skip_), left(left_), doc_min(0), doc_max(0), mask(0) {}
    __device__ __forceinline__ WalkTile next() {
        if (left <= 0) return {-1, 0, 0};
        while (mask == 0) {
            base += 64;
            if (base >= end) return {-1, 0, 0};
            const int t = min(base + (int)(threadIdx.x & 63), end - 1);
            if (lowest) {
                doc_min = lowest[t];
                doc_max = highest[t];
            }
            mask = __ballot(base + (int)(threadIdx.x & 63) < end && active(t, doc_min, doc_max));
            const int here = __builtin_popcountll(mask);
            if (skip >= here) {
                skip -= here;
                mask = 0;
            }
            for (; skip > 0 && mask; --skip) mask &= mask - 1;
        }
        const int lane = __builtin_ctzll(mask);
        mask &= mask - 1;
        --left;
        return {base + lane, __builtin_amdgcn_readlane(doc_min, lane), __builtin_amdgcn_readlane(doc_max, lane)};
    }
};

// Lowest and highest document of the tiles of `per` rows that block `block` of a launch looks at, a wavefront a tile; row r
// stands for token r / group + offset, -1 where that is none.  range_blocks(tiles) blocks per batch element.
__host__ __device__ inline int range_blocks(int tiles) { return (tiles + kWaves - 1) / kWaves; }
__device__ __forceinline__ void document_range(const int32_t* __restrict__ docs, int kv_len, int block, int per, int tiles, int rows, int offset,
                                               const GroupDiv& div, int32_t* __restrict__ lowest, int32_t* __restrict__ highest) {
    const int b = block / range_blocks(tiles), lane = threadIdx.x & 63;
    const int tile = (block - b * range_blocks(tiles)) * kWaves + (threadIdx.x >> 6);
    if (tile >= tiles) return;
    int lo = 0x7FFFFFFF, hi = -1;
    for (int i = lane; i < per; i += 64) {
        const int row = tile * per + i;
        if (row >= rows) break;
        const int pos = div(row) + offset;
        const int doc = pos >= 0 ? docs[(int64_t)b * kv_len + pos] : -1;
        lo = min(lo, doc);
        hi = max(hi, doc);
    }
    lo = wave_min_i32(lo);
    hi = wave_max_i32(hi);
    if (lane == 0) {
        lowest[(int64_t)b * tiles + tile] = lo;
        highest[(int64_t)b * tiles + tile] = hi;
    }
}

// Which queries see fewer than kFewKeys keys where there are documents: without them the interval says it.  A wavefront looks at 64 queries and
// counts the keys of their documents in their intervals, block by block of 64 from the queries' own positions to the front and then to the
// back, until every query has enough, a block holds none of what those that lack some look for, or after kFewReach blocks.  Exact for
// documents that lie in one piece; a query whose document goes on behind a gap, or is mixed with 8 and more others, may be taken to have
// few, which costs time and nothing else.  few_blocks(q_len) blocks per batch element.
constexpr int kFewReach = 16;
__host__ __device__ inline int few_words(int64_t q_len) { return (int)((q_len + 63) / 64); }
__host__ __device__ inline int few_blocks(int64_t q_len) { return (few_words(q_len) + kWaves - 1) / kWaves; }
__device__ __forceinline__ void few_queries(const AttnArgs& a, int block, uint64_t* __restrict__ few) {
    const int words = few_words(a.q_len), per = few_blocks(a.q_len), b = block / per, lane = threadIdx.x & 63;
    const int word = (block - b * per) * kWaves + (int)(threadIdx.x >> 6);
    if (word >= words) return;
    const int s = word * 64 + lane, pos0 = word * 64 + a.kv_len - a.q_len;
    const RowSpan span = row_span(a, b, s < a.q_len ? s : a.q_len - 1);
    const bool some = s < a.q_len && span.hi >= span.lo;
    const uint32_t reach = some ? (uint32_t)(span.hi - span.lo) : 0u;
    const int32_t* docs = a.docs + (int64_t)b * a.kv_len;
    int n = 0;
    for (int way = -1; way <= 1; way += 2) {
        for (int i = way < 0 ? 0 : 1; i <= kFewReach; ++i) {
            const int j0 = pos0 + 64 * way * i;
            if (__ballot(some && n < kFewKeys && (way < 0 ? span.lo <= j0 + 63 : span.hi >= j0)) == 0) break;
            const int doc = j0 + lane >= 0 && j0 + lane < a.kv_len ? docs[j0 + lane] : -1, doc0 = __builtin_amdgcn_readfirstlane(doc);
            int here = 0;
            if (__ballot(doc != doc0) == 0) {  // one document
                here = doc0 == span.doc ? max(0, min(span.hi, j0 + 63) - max(span.lo, j0) + 1) : 0;
            } else {
                for (int u = 0; u < 64; ++u)
                    here += __builtin_amdgcn_readlane(doc, u) == span.doc && (uint32_t)(j0 + u - span.lo) <= reach;
            }
            // the queries' own block holds them themselves
            if (i > 0 && __ballot(some && n < kFewKeys && here > 0) == 0) break;
            n += here;
        }
    }
    const uint64_t bits = __ballot(some && n < kFewKeys);
    if (lane == 0) few[(int64_t)b * words + word] = bits;
}
// whether query s, whose interval holds key_span + 1 keys, has few
__device__ __forceinline__ bool has_few(const MfmaArgs& m, int b, int s, int key_span) {
    if (!m.few) return key_span < kFewKeys - 1;
    return m.few[(int64_t)b * m.few_words + (s >> 6)] >> (s & 63) & 1;
}
// whether one of queries q0 .. q1, at most 64, has
__device__ __forceinline__ bool any_has_few(const MfmaArgs& m, int b, int q0, int q1) {
    const uint64_t* words = m.few + (int64_t)b * m.few_words;
    uint64_t bits = words[q0 >> 6] >> (q0 & 63);
    if (q0 >> 6 != q1 >> 6) bits |= words[q1 >> 6] << (64 - (q0 & 63));  // q0 & 63 is not 0 then
    return bits << (63 - (q1 - q0)) != 0;
}

// the tiles that a walk passes
template <typename F>
__device__ __forceinline__ int count_tiles(int first, int end, const int32_t* lowest, const int32_t* highest, F active) {
    TileWalk<F> walk(first, end, lowest, highest, active, 0x7FFFFFFF, 1);
    walk.next();
    return 0x7FFFFFFF - walk.skip;
}
// a block's share of its walk: tiles skip .. skip + left - 1 of those that the walk passes
struct Share {
    int parts, skip, left;
};
__device__ __forceinline__ Share share_of(int tiles, int split, const MfmaArgs& m) {
    Share s;
    s.parts = (tiles + m.target / 2) / m.target;  // a walk a little longer than the target stays whole
    s.parts = s.parts < 1 ? 1 : (s.parts < m.splits ? s.parts : m.splits);
    s.skip = (int)((int64_t)tiles * split / s.parts);
    s.left = (int)((int64_t)tiles * (split + 1) / s.parts) - s.skip;
    return s;
}

// What becomes of q . k.  kPlain: scale alone, folded into the exponent's multiply-add.  kFast and kAccurate: scale, softcap and slopes,
// with softcap tanh(y) = 1 - 2 / (1 + e^(2y)) from the hardware's exponential and reciprocal or from the library's tanh.  The first is off
// by up to some 2^-22 of softcap, which bf16 has room for up to a softcap of 1024 (2^-12 in a score, where P is rounded to 2^-8).
enum ScoreMode { kPlain, kFast, kAccurate };
constexpr float kFastCap = 1024.f;

struct ScoreScale {
    float mul;   // log2(e) * scale, or with softcap: scale / softcap (kAccurate), 2 log2(e) scale / softcap (kFast)
    float cap2;  // softcap * log2(e), 0: none
};
template <int MODE>
__device__ __forceinline__ ScoreScale score_scale(const AttnArgs& a) {
    if (MODE != kPlain && a.softcap > 0.f) return {a.scale / a.softcap * (MODE == kFast ? 2.f * kLog2e : 1.f), a.softcap * kLog2e};
    return {a.scale * kLog2e, 0.f};
}
template <int MODE>
__device__ __forceinline__ float capped(float x, float mul) {  // tanh(x * scale / softcap)
    if (MODE == kFast) return 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * mul));
    return tanhf(x * mul);
}
inline ScoreMode score_mode(const AttnArgs& a, bool plain) {
    return plain ? kPlain : (a.dtype == PICOMOE_BF16 && a.softcap <= kFastCap ? kFast : kAccurate);
}

}  // namespace
