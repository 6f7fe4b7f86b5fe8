// Attention of drafted tokens over the hot buffer (kvx/kvx_attn.h).
//
// A workgroup of four waves takes up to 16 * RW * WR queries (node, head) of
// one request and walks a range of the request's keys, the selected slots and
// then the drafted tokens' own, 32 at a time.  A wave holds RW * 16 queries in
// registers with their whole output (512 columns, 32 bits): WR waves share the
// keys in LDS with queries of their own, and 4 / WR groups of waves take every
// (4 / WR)-th tile of keys; their outputs are joined at the end.
//
// Scores are held transposed, S^T = K Q^T (keys down, queries across the
// lanes), so that a lane's scores, its running maximum and its sum all belong
// to the query lane % 16, and so that the weights are, as they come, the
// operand of O^T = V^T P^T, where V is the first 512 columns of the same rows:
// the matrix product takes its 32 keys in any order, here 4 of the tile's
// upper and 4 of its lower half for each group of 16 lanes.
#include <algorithm>

#include "row_format.h"

namespace kvx {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 32;                 // keys a tile
constexpr int kPanels = kDim / 64;        // a row in LDS: 9 panels of 64 values (128 bytes)
constexpr int kPanelBytes = kTile * 128;
constexpr int kTileBytes = kPanels * kPanelBytes;
constexpr int kChunk = 64;                // tiles whose rows are looked up at a time
constexpr int kAhead = 2;                 // panels whose operands are read ahead
constexpr float kRise = 8.0f;             // a maximum may rise by 2^8 before the output is scaled down again

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
#define KVX_LDS __attribute__((address_space(3)))
#define KVX_GLB __attribute__((address_space(1)))

// what a key without a row reads
__device__ __align__(128) uint8_t kvx_no_row[kDim * 2];

template <int DTYPE>
struct Elem;
template <>
struct Elem<KVX_DTYPE_BF16> {
    typedef __bf16 T;
    static constexpr uint32_t special = 0x7F80u;   // exponent of infinities and NaN
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t from_codes(uint32_t codes, float scale, bool high)
    {
        return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true)
                                                 : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false));
    }
};
template <>
struct Elem<KVX_DTYPE_FP16> {
    typedef _Float16 T;
    static constexpr uint32_t special = 0x7C00u;
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
    static __device__ __forceinline__ uint32_t from_codes(uint32_t codes, float scale, bool high)
    {
        return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, true)
                                                 : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, false));
    }
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    typedef T T2 __attribute__((ext_vector_type(2)));
    T2 v;
    v[0] = static_cast<T>(a);
    v[1] = static_cast<T>(b);
    return __builtin_bit_cast(uint32_t, v);
}

// Over the four lanes that hold scores of one query (lane % 16).
template <typename F>
__device__ __forceinline__ float over_query(float x, F f)
{
    typedef unsigned int u2 __attribute__((ext_vector_type(2)));
    u2 v = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(v[0]), __uint_as_float(v[1]));
    v = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(v[0]), __uint_as_float(v[1]));
}

// The output stays in the accumulation registers: without this the compiler
// keeps second copies of it around each place that scales it, and spills.
__device__ __forceinline__ void keep_in_acc(f32x4 &x) { asm volatile("" : "+a"(x)); }

// Byte of the 16-byte chunk c (0..7) of row r in a panel: rows one after
// another are 128 bytes apart, so the chunks of 8 rows are permuted to spread a
// column over the banks.
__device__ __forceinline__ uint32_t chunk_at(uint32_t r, uint32_t c) { return r * 128u + ((c ^ (r & 7u)) << 4); }

// 16 bytes a lane from memory to LDS at base + lane * 16, not waited for: the
// caller counts the loads (wait_loads).
__device__ __forceinline__ void load_to_lds(const uint8_t *from, uint32_t base)
{
    // (a wait state between the write of m0 and its use)
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(base) : "memory");
}

template <int LEFT>
__device__ __forceinline__ void wait_loads()
{
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
}

// Every wave's LDS reads are done and what it waited for is there.
__device__ __forceinline__ void meet() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int DTYPE, int QUANT, int RW, int WR>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(1, 1))) void kvx_tree_attention(AttnArgs a)
{
    typedef Elem<DTYPE> E;
    typedef typename E::T T;
    using F = RowForm<QUANT>;
    constexpr bool kCodes = QUANT != KVX_QUANT_NONE;
    constexpr int WK = 4 / WR;                       // groups of waves that take keys of their own
    constexpr int kRows = RW * 16;                   // queries of a wave
    constexpr int kBuffers = kCodes ? (WR == 1 ? 1 : 2) : WR;   // of a group
    constexpr int kGroups = 4 / WR;                  // groups of 8 rows that a wave loads
    constexpr int kLoads = kGroups * kPanels;        // loads of a tile by a wave (16-bit rows)
    constexpr int kJoinCols = kLatent / RW;
    constexpr int kJoinStride = kJoinCols + 4;       // floats
    constexpr int kJoinBytes = WK > 1 ? 4 * kRows * kJoinStride * 4 : 0;
    constexpr int kTilesBytes = WK * kBuffers * kTileBytes;

    __shared__ __align__(128) uint8_t tiles[kTilesBytes > kJoinBytes ? kTilesBytes : kJoinBytes];
    __shared__ int32_t rowOf[kChunk * kTile];        // hot row within the request of each key, -1: none
    __shared__ float stat[4][kRows][2], weigh[4][kRows];

    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t col = lane & 15u, grp = lane >> 4;
    const uint32_t wr = wave % WR, wk = wave / WR;
    const uint32_t queries = a.draft * a.heads;

    // consecutive workgroups of one XCD's share take the same keys
    const uint32_t total = a.reqs * a.splits * a.queryTiles, share = (total + 7u) / 8u;
    const uint32_t item = (blockIdx.x & 7u) * share + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= share || item >= total) return;
    const uint32_t qt = item % a.queryTiles, split = item / a.queryTiles % a.splits;
    const uint32_t req = item / a.queryTiles / a.splits;

    const uint32_t keys = a.topK + (a.draftSlots != 0 ? a.draft : 0u);
    const uint32_t allTiles = (keys + kTile - 1) / kTile;
    const uint32_t tile0 = static_cast<uint32_t>(static_cast<uint64_t>(allTiles) * split / a.splits);
    const uint32_t tile1 = static_cast<uint32_t>(static_cast<uint64_t>(allTiles) * (split + 1) / a.splits);
    // slots of the chunk from tile c0 on, kThreads apart (-1 past the range)
    constexpr int kSlots = kChunk * kTile / kThreads;
    auto readSlots = [&](uint32_t c0, int32_t (&slot)[kSlots]) {
#pragma unroll
        for (int n = 0; n < kSlots; ++n) {
            const uint32_t k = c0 * kTile + n * kThreads + threadIdx.x;
            slot[n] = -1;
            if (k < min(keys, tile1 * kTile)) {
                slot[n] = k < a.topK ? reinterpret_cast<const KVX_GLB int32_t *>(a.slots)[static_cast<uint64_t>(req) * a.topK + k]
                                     : reinterpret_cast<const KVX_GLB int32_t *>(a.draftSlots)[static_cast<uint64_t>(req) * a.draft + k - a.topK];
            }
        }
    };
    auto lookUp = [&](const int32_t (&slot)[kSlots]) {
#pragma unroll
        for (int n = 0; n < kSlots; ++n) {
            rowOf[n * kThreads + threadIdx.x] = hot_row(slot[n], req, a.reqStride, a.hotRows, a.overflowSlot) < 0 ? -1 : slot[n];
        }
    };
    int32_t firstSlots[kSlots];
    readSlots(tile0, firstSlots);                    // (before the queries: the rows' addresses wait for them)

    uint32_t query[RW];
    u32x4 q[RW][kDim / 32];
    uint64_t sees[RW];                               // drafted tokens that the query sees
#pragma unroll
    for (int w = 0; w < RW; ++w) {
        query[w] = (qt * WR + wr) * kRows + w * 16 + col;
        const uint32_t real = min(query[w], queries - 1);      // (what lies past the last query is not stored)
        const uint32_t node = real / a.heads, head = real % a.heads;
        const uint64_t at = a.q + req * a.qStrideB + node * a.qStrideT + head * a.qStrideH + grp * 16;
#pragma unroll
        for (int s = 0; s < kDim / 32; ++s) q[w][s] = *reinterpret_cast<const KVX_GLB u32x4 *>(at + s * 64);
        sees[w] = a.treeMask != 0 ? reinterpret_cast<const KVX_GLB uint64_t *>(a.treeMask)[req * a.draft + node]
                                  : ~0ull >> (63u - node);
    }
    lookUp(firstSlots);
    const uint32_t flip = a.negate ? 0x80008000u : 0u;               // a negative scale: negative queries
#pragma unroll
    for (int w = 0; w < RW; ++w) {
#pragma unroll
        for (int s = 0; s < kDim / 32; ++s) q[w][s] ^= flip;
    }
    float top[RW], sum[RW];
    f32x4 o[kLatent / 16][RW];
#pragma unroll
    for (int w = 0; w < RW; ++w) {
        top[w] = -INFINITY;
        sum[w] = 0.0f;
#pragma unroll
        for (int d = 0; d < kLatent / 16; ++d) o[d][w] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const uint8_t *hot = reinterpret_cast<const uint8_t *>(a.hot) + req * a.reqStride * F::bytes;
    const uint32_t ldsTiles = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((KVX_LDS uint8_t *)tiles));
    const uint32_t ldsGroup = ldsTiles + wk * kBuffers * kTileBytes;
    // this lane's bytes of a tile: its key's chunk for a score step (two steps
    // a panel), and its four columns of four keys for an output step
    const uint32_t atKey[2] = {chunk_at(col, grp), chunk_at(col, grp + 4)};
    uint32_t atValue[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) atValue[d] = chunk_at(grp * 4 + (col >> 2), d * 2 + ((col & 3u) >> 1)) + (col & 1u) * 8u;

    // ---- bringing a tile in ----
    // 16-bit rows: straight to LDS, 8 rows by 128 bytes a load
    auto fetch = [&](uint32_t t, uint32_t buffer) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const uint32_t r = (wr * kGroups + g) * 8 + (lane >> 3);
            const int32_t row = rowOf[t * kTile + r];
            const uint8_t *from = row < 0 ? kvx_no_row : hot + static_cast<uint64_t>(static_cast<uint32_t>(row)) * F::bytes;
            from += ((lane & 7u) ^ (lane >> 3)) * 16;
#pragma unroll
            for (int p = 0; p < kPanels; ++p) {
                load_to_lds(from + p * 128, ldsGroup + buffer * kTileBytes + p * kPanelBytes + (wr * kGroups + g) * 1024);
            }
        }
    };
    // 8-bit rows: through registers, 16 rows by a panel of 64 codes a load
    constexpr int kParts = WR == 1 ? 2 : 1;          // halves of the tile's rows that a wave brings in
    constexpr int kStep = WR == 4 ? 2 : 1;           // ... and every how many panels
    constexpr int kCodePanels = F::codes / 64;
    constexpr int kHeld = (kPanels + kStep - 1) / kStep;
    u32x4 held[kParts][kHeld], rawHigh[kParts], scaleLow[kParts];
    uint32_t scaleHigh[kParts];
    const uint32_t firstPanel = WR == 4 ? wr >> 1 : 0u;
    const uint32_t j4 = lane & 3u;
    auto load = [&](uint32_t t) {
#pragma unroll
        for (int h = 0; h < kParts; ++h) {
            const uint32_t r = (WR == 1 ? h : wr & 1u) * 16 + (lane >> 2);
            const int32_t row = rowOf[t * kTile + r];
            const uint64_t at = reinterpret_cast<uint64_t>(row < 0 ? kvx_no_row : hot + static_cast<uint64_t>(static_cast<uint32_t>(row)) * F::bytes);
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                const uint32_t p = i * kStep + firstPanel;
                if (i * kStep + kStep > kPanels && p >= kPanels) continue;
                // (a panel kept in 16 bits: 32 bytes a lane)
                const uint64_t from = at + p * 64 + (F::raw != 0 && p == kCodePanels ? j4 * 32 : j4 * 16);
                held[h][i] = *reinterpret_cast<const KVX_GLB u32x4 *>(from);
                if (F::raw != 0 && p == kCodePanels) rawHigh[h] = *reinterpret_cast<const KVX_GLB u32x4 *>(from + 16);
            }
            scaleLow[h] = *reinterpret_cast<const KVX_GLB u32x4 *>(at + F::scaleAt);
            if (F::scales > 16) scaleHigh[h] = *reinterpret_cast<const KVX_GLB uint32_t *>(at + F::scaleAt + 16);
        }
    };
    auto store = [&](uint32_t buffer) {
#pragma unroll
        for (int h = 0; h < kParts; ++h) {
            const uint32_t r = (WR == 1 ? h : wr & 1u) * 16 + (lane >> 2);
            const uint32_t base = ldsGroup + buffer * kTileBytes;
            const uint32_t low = base + chunk_at(r, j4 * 2), high = base + chunk_at(r, j4 * 2 + 1);
            const uint32_t shift = (j4 >> 1) * 8;
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                const uint32_t p = i * kStep + firstPanel;
                if (i * kStep + kStep > kPanels && p >= kPanels) continue;
                u32x4 x = held[h][i], y = rawHigh[h];
                if (F::raw == 0 || p != kCodePanels) {
                    // panel p's two groups: bytes 2p and 2p + 1
                    const uint32_t four = i * kStep / 2 < 4 ? scaleLow[h][i * kStep / 2] : scaleHigh[h];
                    const float scale = __uint_as_float(((four >> ((p & 1u) * 16 + shift)) & 255u) << 23);
                    const u32x4 c = held[h][i];
                    x = u32x4{E::from_codes(c[0], scale, false), E::from_codes(c[0], scale, true),
                              E::from_codes(c[1], scale, false), E::from_codes(c[1], scale, true)};
                    y = u32x4{E::from_codes(c[2], scale, false), E::from_codes(c[2], scale, true),
                              E::from_codes(c[3], scale, false), E::from_codes(c[3], scale, true)};
                }
                *(KVX_LDS u32x4 *)(uintptr_t)(low + p * kPanelBytes) = x;
                *(KVX_LDS u32x4 *)(uintptr_t)(high + p * kPanelBytes) = y;
            }
        }
    };

    for (uint32_t c0 = tile0; c0 < tile1; c0 += kChunk) {
        const uint32_t chunk = min(static_cast<uint32_t>(kChunk), tile1 - c0);
        if (c0 != tile0) {
            int32_t slots[kSlots];
            readSlots(c0, slots);
            __syncthreads();
            lookUp(slots);
        }
        __syncthreads();
        const uint32_t steps = (chunk + WK - 1) / WK;

        // tile i * WK + wk of the chunk, in its buffer
        auto work = [&](uint32_t i, uint32_t buffer) {
            const uint32_t t = min(i * WK + wk, static_cast<uint32_t>(kChunk - 1));
            const bool past = i * WK + wk >= chunk;
            const uint32_t live = past ? 0u : static_cast<uint32_t>(__ballot(rowOf[t * kTile + (lane & 31u)] >= 0));
            const uint32_t k0 = (c0 + t) * kTile;
            // (the same for every wave of the workgroup)
            const bool drafted = (c0 + i * WK + WK) * kTile > a.topK && a.draftSlots != 0;
            if (live == 0 && !(drafted && WR > 1)) return;
            const KVX_LDS uint8_t *tile = (KVX_LDS uint8_t *)(uintptr_t)(ldsGroup + buffer * kTileBytes);

            // the operands of the next panels are on their way while one panel's are multiplied
            f32x4 s[2][RW] = {};
            u32x4 key[kAhead + 1][4];
            auto readKeys = [&](int p) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    key[p % (kAhead + 1)][i] = *reinterpret_cast<const KVX_LDS u32x4 *>(tile + atKey[i >> 1] + p * kPanelBytes + (i & 1) * 2048);
                }
            };
#pragma unroll
            for (int p = 0; p < kAhead; ++p) readKeys(p);
#pragma unroll
            for (int p = 0; p < kPanels; ++p) {
                if (p + kAhead < kPanels) readKeys(p + kAhead);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
#pragma unroll
                    for (int w = 0; w < RW; ++w) s[i & 1][w] = E::mfma(key[p % (kAhead + 1)][i], q[w][p * 2 + (i >> 1)], s[i & 1][w]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (live != ~0u || drafted) {
                const uint32_t selected = k0 >= a.topK ? 0u : (a.topK - k0 >= 32u ? ~0u : (1u << (a.topK - k0)) - 1u);
#pragma unroll
                for (int w = 0; w < RW; ++w) {
                    uint32_t own = 0;                // drafted tokens' bits of this tile
                    if (drafted) own = static_cast<uint32_t>(k0 >= a.topK ? sees[w] >> (k0 - a.topK) : sees[w] << min(a.topK - k0, 63u));
                    const uint32_t seen = (live & (selected | (own & ~selected))) >> (grp * 4);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const bool is = (seen & (1u << ((j >> 2) * 16 + (j & 3)))) != 0;
                        s[j >> 2][w][j & 3] = is ? s[j >> 2][w][j & 3] : -INFINITY;
                    }
                }
            }
            float most[RW];
            bool rise = false;
#pragma unroll
            for (int w = 0; w < RW; ++w) {
                float m = s[0][w][0];                // (a NaN is left out; its weight is one)
#pragma unroll
                for (int j = 1; j < 8; ++j) m = fmaxf(m, s[j >> 2][w][j & 3]);
                most[w] = over_query(m, [](float x, float y) { return fmaxf(x, y); }) * a.scaleLog2;
                rise = rise || most[w] > top[w] + kRise;
            }
            // The weights are exp2(score - top) for a top at most 2^8 below the
            // largest score so far: the output is scaled only when one rose by more.
            if (__any(rise)) {
                float keep[RW];
                bool any = false;                    // (nothing is there to scale at the first tile)
#pragma unroll
                for (int w = 0; w < RW; ++w) {
                    const float now = fmaxf(top[w], most[w]);
                    any = any || top[w] != -INFINITY;
                    keep[w] = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top[w] - now);
                    top[w] = now;
                }
                if (__any(any)) {
#pragma unroll
                    for (int w = 0; w < RW; ++w) {
                        sum[w] *= keep[w];
#pragma unroll
                        for (int d = 0; d < kLatent / 16; ++d) {
                            keep_in_acc(o[d][w]);
                            o[d][w] *= keep[w];
                            keep_in_acc(o[d][w]);
                        }
                    }
                }
            }
            // A drafted row that holds a NaN or an infinity must not reach the
            // queries that do not see it, whose weight 0 would turn it into a NaN;
            // those that see it have a score that is one already.
            if (drafted) {
                if (WR > 1) meet();
                constexpr uint32_t kWords = kTile * kLatent / 2;
                for (uint32_t i2 = wr * 64 + lane; i2 < kWords; i2 += WR * 64) {
                    const uint32_t r = i2 / (kLatent / 2), c = i2 % (kLatent / 2);
                    if (k0 + r < a.topK) continue;
                    KVX_LDS uint32_t *v = (KVX_LDS uint32_t *)(tile + (c >> 5) * kPanelBytes + chunk_at(r, (c >> 2) & 7u) + (c & 3u) * 4u);
                    uint32_t x = *v;
                    if ((x & E::special) == E::special) x &= 0xFFFF0000u;
                    if ((x & (E::special << 16)) == (E::special << 16)) x &= 0xFFFFu;
                    *v = x;
                }
                if (WR > 1) meet();
            }
            u32x4 value[kAhead + 1][4];
            auto readValues = [&](int p) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    KVX_LDS s16x4 *at = (KVX_LDS s16x4 *)(tile + atValue[i] + p * kPanelBytes);
                    const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at);
                    const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at + 2048 / 8);
                    value[p % (kAhead + 1)][i] = __builtin_bit_cast(u32x4, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
                }
            };
#pragma unroll
            for (int p = 0; p < kAhead; ++p) readValues(p);
            u32x4 weight[RW];
#pragma unroll
            for (int w = 0; w < RW; ++w) {
                const float base = top[w] == -INFINITY ? 0.0f : top[w];
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j >> 2][w][j & 3], a.scaleLog2, -base));
                    sum[w] += p[j];
                }
                weight[w] = u32x4{pack2<T>(p[0], p[1]), pack2<T>(p[2], p[3]), pack2<T>(p[4], p[5]), pack2<T>(p[6], p[7])};
            }
#pragma unroll
            for (int p = 0; p < kLatent / 64; ++p) {
                if (p + kAhead < kLatent / 64) readValues(p + kAhead);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
#pragma unroll
                    for (int w = 0; w < RW; ++w) o[p * 4 + i][w] = E::mfma(value[p % (kAhead + 1)][i], weight[w], o[p * 4 + i][w]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };

        if constexpr (!kCodes && WR > 1) {
            // a tile's loads are under way while kBuffers - 1 others are worked on
            for (uint32_t i = 0; i + 1 < kBuffers && i < steps; ++i) fetch(i * WK + wk, i);
            uint32_t buffer = 0, next = kBuffers - 1;
            for (uint32_t i = 0; i < steps; ++i) {
                if (i + kBuffers - 2 < steps - 1) wait_loads<(kBuffers - 2) * kLoads>();
                else wait_loads<0>();
                meet();
                if (i + kBuffers - 1 < steps) fetch((i + kBuffers - 1) * WK + wk, next);
                work(i, buffer);
                buffer = buffer + 1 == kBuffers ? 0 : buffer + 1;
                next = next + 1 == kBuffers ? 0 : next + 1;
            }
        } else if constexpr (!kCodes) {
            for (uint32_t i = 0; i < steps; ++i) {
                if (i * WK + wk >= chunk) break;
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the tile before has been read)
                fetch(i * WK + wk, 0);
                wait_loads<0>();
                work(i, 0);
            }
        } else if constexpr (WR == 1) {
            if (wk < chunk) load(wk);
            for (uint32_t t = wk; t < chunk; t += WK) {
                store(0);
                if (t + WK < chunk) load(t + WK);
                work(t / WK, 0);
            }
        } else {
            load(wk);
            store(0);
            if (steps > 1) load(WK + wk);
            for (uint32_t i = 0; i < steps; ++i) {
                meet();
                if (i + 1 < steps) store((i + 1) & 1u);
                if (i + 2 < steps) load((i + 2) * WK + wk);
                work(i, i & 1u);
            }
        }
    }

    // ---- joining the groups of waves ----
#pragma unroll
    for (int w = 0; w < RW; ++w) sum[w] = over_query(sum[w], [](float x, float y) { return x + y; });
    const uint64_t row0 = static_cast<uint64_t>(req) * queries;        // first output row of the request
    if constexpr (WK > 1) {
        if (grp == 0) {
#pragma unroll
            for (int w = 0; w < RW; ++w) {
                stat[wave][w * 16 + col][0] = top[w];
                stat[wave][w * 16 + col][1] = sum[w];
            }
        }
        __syncthreads();
        // a group's output counts exp2(its maximum - the largest) times
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            float most = -INFINITY, all = 0.0f;
#pragma unroll
            for (int g = 0; g < WK; ++g) most = fmaxf(most, stat[g * WR + wr][w * 16 + col][0]);
            const float base = most == -INFINITY ? 0.0f : most;
#pragma unroll
            for (int g = 0; g < WK; ++g) {
                const float *x = stat[g * WR + wr][w * 16 + col];
                all += x[1] * __builtin_amdgcn_exp2f(x[0] - base);
            }
            // ... and, where this is all of it, over the sum
            const float whole = a.splits > 1 ? 1.0f : (all == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(all));
            if (grp == 0) weigh[wave][w * 16 + col] = __builtin_amdgcn_exp2f(top[w] - base) * whole;
            top[w] = most;
            sum[w] = all;
        }
        KVX_LDS float *join = (KVX_LDS float *)tiles;
#pragma unroll
        for (int round = 0; round < RW; ++round) {
#pragma unroll
            for (int d = 0; d < kJoinCols / 16; ++d) {
#pragma unroll
                for (int w = 0; w < RW; ++w) {
                    f32x4 &x = o[round * (kJoinCols / 16) + d][w];
                    keep_in_acc(x);
                    *reinterpret_cast<KVX_LDS f32x4 *>(join + (wave * kRows + w * 16 + col) * kJoinStride + d * 16 + grp * 4) = x;
                }
            }
            __syncthreads();
#pragma unroll
            for (int n = 0; n < WR * kRows * (kJoinCols / 4) / kThreads; ++n) {
                const uint32_t i = threadIdx.x + n * kThreads;
                const uint32_t c = i % (kJoinCols / 4), r = i / (kJoinCols / 4);
                f32x4 x = {};
#pragma unroll
                for (int g = 0; g < WK; ++g) {
                    x += *reinterpret_cast<const KVX_LDS f32x4 *>(join + (g * WR * kRows + r) * kJoinStride + c * 4) *
                         weigh[g * WR + r / kRows][r % kRows];
                }
                const uint32_t index = qt * WR * kRows + r;
                if (index < queries) {
                    if (a.splits == 1) {
                        KVX_GLB T *out = reinterpret_cast<KVX_GLB T *>(a.out) + (row0 + index) * kLatent + round * kJoinCols + c * 4;
                        *reinterpret_cast<KVX_GLB u32x2 *>(out) = u32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
                    } else {
                        KVX_GLB float *out = reinterpret_cast<KVX_GLB float *>(a.part) + ((static_cast<uint64_t>(req) * a.splits + split) * queries + index) * kLatent + round * kJoinCols + c * 4;
                        *reinterpret_cast<KVX_GLB f32x4 *>(out) = x;
                    }
                }
            }
            if (round + 1 < RW) __syncthreads();
        }
    } else {
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            if (query[w] >= queries) continue;
            if (a.splits == 1) {
                const float inv = sum[w] == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(sum[w]);
                KVX_GLB T *out = reinterpret_cast<KVX_GLB T *>(a.out) + (row0 + query[w]) * kLatent + grp * 4;
#pragma unroll
                for (int d = 0; d < kLatent / 16; ++d) {
                    keep_in_acc(o[d][w]);
                    *reinterpret_cast<KVX_GLB u32x2 *>(out + d * 16) =
                        u32x2{pack2<T>(o[d][w][0] * inv, o[d][w][1] * inv), pack2<T>(o[d][w][2] * inv, o[d][w][3] * inv)};
                }
            } else {
                KVX_GLB float *out = reinterpret_cast<KVX_GLB float *>(a.part) + ((static_cast<uint64_t>(req) * a.splits + split) * queries + query[w]) * kLatent + grp * 4;
#pragma unroll
                for (int d = 0; d < kLatent / 16; ++d) {
                    keep_in_acc(o[d][w]);
                    *reinterpret_cast<KVX_GLB f32x4 *>(out + d * 16) = o[d][w];
                }
            }
        }
    }
    if (wk == 0 && grp == 0) {
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            if (query[w] >= queries) continue;
            if (a.splits == 1) {
                if (a.lse != 0) {
                    reinterpret_cast<KVX_GLB float *>(a.lse)[row0 + query[w]] =
                        sum[w] == 0.0f ? -INFINITY : (top[w] + __builtin_amdgcn_logf(sum[w])) * 0.6931471805599453f;
                }
            } else {
                reinterpret_cast<KVX_GLB f32x2 *>(a.partStat)[(static_cast<uint64_t>(req) * a.splits + split) * queries + query[w]] = f32x2{top[w], sum[w]};
            }
        }
    }
}

// Joins the splits: one wave a query.
template <int DTYPE>
__global__ __launch_bounds__(kThreads) void kvx_tree_attention_join(AttnArgs a)
{
    typedef typename Elem<DTYPE>::T T;
    const uint32_t queries = a.draft * a.heads;
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (row >= static_cast<uint64_t>(a.reqs) * queries) return;
    const uint32_t lane = threadIdx.x & 63u;
    const uint64_t first = row / queries * a.splits * queries + row % queries;
    const KVX_GLB f32x2 *stats = reinterpret_cast<const KVX_GLB f32x2 *>(a.partStat) + first;
    float most = -INFINITY;
    for (uint32_t s = 0; s < a.splits; ++s) most = fmaxf(most, stats[static_cast<uint64_t>(s) * queries].x);
    const float base = most == -INFINITY ? 0.0f : most;
    float all = 0.0f;
    f32x4 x = {}, y = {};
    for (uint32_t s = 0; s < a.splits; ++s) {
        const uint64_t at = first + static_cast<uint64_t>(s) * queries;
        const f32x2 st = stats[static_cast<uint64_t>(s) * queries];
        const float keep = __builtin_amdgcn_exp2f(st.x - base);
        all += st.y * keep;
        const KVX_GLB f32x4 *v = reinterpret_cast<const KVX_GLB f32x4 *>(a.part) + at * (kLatent / 4) + lane * 2;
        x += v[0] * keep;
        y += v[1] * keep;
    }
    const float inv = all == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(all);
    *reinterpret_cast<KVX_GLB u32x4 *>(reinterpret_cast<KVX_GLB T *>(a.out) + row * kLatent + lane * 8) =
        u32x4{pack2<T>(x[0] * inv, x[1] * inv), pack2<T>(x[2] * inv, x[3] * inv), pack2<T>(y[0] * inv, y[1] * inv), pack2<T>(y[2] * inv, y[3] * inv)};
    if (lane == 0 && a.lse != 0) {
        reinterpret_cast<KVX_GLB float *>(a.lse)[row] = all == 0.0f ? -INFINITY : (most + __builtin_amdgcn_logf(all)) * 0.6931471805599453f;
    }
}

template <int DTYPE, int QUANT>
void launch(const AttnArgs &a, const AttnPlan &p, hipStream_t stream)
{
    auto *kernel = p.rows == 16   ? kvx_tree_attention<DTYPE, QUANT, 1, 1>
                   : p.rows == 32 ? kvx_tree_attention<DTYPE, QUANT, 2, 1>
                   : p.rows == 64 ? kvx_tree_attention<DTYPE, QUANT, 2, 2>
                                  : kvx_tree_attention<DTYPE, QUANT, 2, 4>;
    const uint32_t items = a.reqs * a.splits * a.queryTiles;
    hipLaunchKernelGGL(kernel, dim3((items + 7u) / 8u * 8u), dim3(kThreads), 0, stream, a);
    if (a.splits > 1) {
        const uint64_t rows = static_cast<uint64_t>(a.reqs) * a.draft * a.heads;
        hipLaunchKernelGGL(kvx_tree_attention_join<DTYPE>, dim3(static_cast<uint32_t>((rows + 3) / 4)), dim3(kThreads), 0,
                           stream, a);
    }
}

}  // namespace

AttnPlan plan_tree_attention(uint32_t reqs, uint32_t draft, uint32_t heads, uint32_t topK, bool drafted)
{
    AttnPlan p{};
    const uint32_t queries = draft * heads;
    p.rows = queries <= 16 ? 16 : (queries <= 32 ? 32 : (queries <= 64 ? 64 : 128));
    p.queryTiles = (queries + p.rows - 1) / p.rows;
    const uint32_t tiles = (topK + (drafted ? draft : 0u) + kTile - 1) / kTile;
    const uint32_t items = reqs * p.queryTiles;
    const uint32_t groups = p.rows <= 32 ? 4 : (p.rows == 64 ? 2 : 1);
    p.splits = std::max(1u, std::min(256u / std::max(items, 1u), tiles / (2 * groups)));
    if (p.splits > 1) p.floats = static_cast<uint64_t>(reqs) * p.splits * queries * (kLatent + 2);
    return p;
}

hipError_t launch_tree_attention(AttnArgs a, const AttnPlan &p, float *scratch, uint32_t dtype, uint32_t quant,
                                 hipStream_t stream)
{
    a.queryTiles = p.queryTiles;
    a.splits = p.splits;
    a.part = reinterpret_cast<uint64_t>(scratch);
    a.partStat = a.part + static_cast<uint64_t>(a.reqs) * p.splits * a.draft * a.heads * kLatent * sizeof(float);
    if (dtype == KVX_DTYPE_BF16) {
        if (quant == KVX_QUANT_NONE) launch<KVX_DTYPE_BF16, KVX_QUANT_NONE>(a, p, stream);
        else if (quant == KVX_QUANT_LATENT) launch<KVX_DTYPE_BF16, KVX_QUANT_LATENT>(a, p, stream);
        else launch<KVX_DTYPE_BF16, KVX_QUANT_ROW>(a, p, stream);
    } else {
        if (quant == KVX_QUANT_NONE) launch<KVX_DTYPE_FP16, KVX_QUANT_NONE>(a, p, stream);
        else if (quant == KVX_QUANT_LATENT) launch<KVX_DTYPE_FP16, KVX_QUANT_LATENT>(a, p, stream);
        else launch<KVX_DTYPE_FP16, KVX_QUANT_ROW>(a, p, stream);
    }
    return hipGetLastError();
}

}  // namespace kvx
