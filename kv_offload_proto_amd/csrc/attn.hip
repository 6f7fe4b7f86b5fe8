// Attention of drafted tokens over the hot buffer (kvx/kvx_attn.h).
//
// One workgroup of four waves takes 16 queries (node, head) of one request and
// walks the request's keys 64 at a time: the selected slots, then the drafted
// tokens' own.  Scores are held transposed, S^T = K Q^T (keys down, queries
// across the lanes), so that a lane's scores, its running maximum and its sum
// all belong to the query lane % 16; the output is O^T = V^T P^T, V being the
// first 512 columns of the same rows.  Each wave makes the scores of 16 keys of
// the tile and 128 columns of the output; the weights P go through LDS.
#include "row_format.h"

namespace kvx {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 64;                 // keys a tile
constexpr int kPanels = kDim / 64;        // a row in LDS: 9 panels of 64 values (128 bytes)
constexpr int kPanelBytes = kTile * 128;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <int DTYPE>
struct Elem;
template <>
struct Elem<KVX_DTYPE_BF16> {
    typedef __bf16 T;
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
};
template <>
struct Elem<KVX_DTYPE_FP16> {
    typedef _Float16 T;
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
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

// 8 values (columns 8c .. 8c+7) of a row as 16-bit ones.
template <int DTYPE, int QUANT>
__device__ __forceinline__ u32x4 load8(const uint8_t *row, int c)
{
    using F = RowForm<QUANT>;
    typedef typename Elem<DTYPE>::T T;
    if (c * 8 >= F::codes) return *reinterpret_cast<const u32x4 *>(row + F::codes + (c * 8 - F::codes) * 2);
    const u32x2 codes = *reinterpret_cast<const u32x2 *>(row + c * 8);
    const uint32_t byte = row[F::scaleAt + c / 4];
    const float scale = __uint_as_float(byte == 0 ? 0x00400000u : byte << 23);
    u32x4 out;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes[i]), false);
        const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes[i]), true);
        out[2 * i] = pack2<T>(lo[0] * scale, lo[1] * scale);
        out[2 * i + 1] = pack2<T>(hi[0] * scale, hi[1] * scale);
    }
    return out;
}

// Byte of the 16-byte chunk c (0..7) of row r in a panel: rows one after
// another are 128 bytes apart, so the chunks of 8 rows are permuted to spread a
// column over the banks.
__device__ __forceinline__ uint32_t chunk_at(uint32_t r, uint32_t c) { return r * 128u + ((c ^ (r & 7u)) << 4); }

template <int DTYPE, int QUANT>
__global__ __launch_bounds__(kThreads) void kvx_tree_attention(AttnArgs a)
{
    typedef Elem<DTYPE> E;
    typedef typename E::T T;
    __shared__ __align__(128) uint8_t tile[kPanels * kPanelBytes];
    __shared__ __align__(128) uint8_t weights[16 * 128];
    __shared__ int64_t keyRow[kTile];      // hot row of each key of the tile, -1: none
    __shared__ float part[4][16];          // the waves' maxima, then sums, of the 16 queries

    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t col = lane & 15u, grp = lane >> 4;
    const uint32_t queries = a.draft * a.heads;
    const uint32_t tiles = (queries + 15u) / 16u;
    const uint32_t req = blockIdx.x / tiles;
    const uint32_t query = (blockIdx.x % tiles) * 16u + col;      // this lane's
    const uint32_t node = query / a.heads, head = query % a.heads;
    const bool real = query < queries;

    u32x4 q[kDim / 32] = {};
    uint64_t sees = 0;                     // drafted tokens that the query sees
    if (real) {
        const uint64_t at = a.q + req * a.qStrideB + node * a.qStrideT + head * a.qStrideH;
#pragma unroll
        for (int s = 0; s < kDim / 32; ++s) q[s] = *reinterpret_cast<const u32x4 *>(at + s * 64 + grp * 16);
        sees = a.treeMask != 0 ? reinterpret_cast<const uint64_t *>(a.treeMask)[req * a.draft + node]
                               : ~0ull >> (63u - node);
    }
    const uint32_t drafted = a.draftSlots != 0 ? a.draft : 0u;
    const uint32_t keys = a.topK + drafted;
    float top = -INFINITY, total = 0.0f;
    f32x4 o[8] = {};

    for (uint32_t k0 = 0; k0 < keys; k0 += kTile) {
        __syncthreads();
        if (threadIdx.x < kTile) {
            const uint32_t k = k0 + threadIdx.x;
            int32_t slot = -1;
            if (k < a.topK) slot = reinterpret_cast<const int32_t *>(a.slots)[static_cast<uint64_t>(req) * a.topK + k];
            else if (k < keys) slot = reinterpret_cast<const int32_t *>(a.draftSlots)[static_cast<uint64_t>(req) * a.draft + k - a.topK];
            keyRow[threadIdx.x] = hot_row(slot, req, a.reqStride, a.hotRows, a.overflowSlot);
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < kTile * kPanels * 8; i += kThreads) {
            const uint32_t r = i / (kPanels * 8), c = i % (kPanels * 8);
            u32x4 v = {};
            if (keyRow[r] >= 0) {
                v = load8<DTYPE, QUANT>(reinterpret_cast<const uint8_t *>(a.hot) +
                                            static_cast<uint64_t>(keyRow[r]) * (QUANT == KVX_QUANT_NONE ? kDim * 2 : RowForm<QUANT>::bytes), c);
            }
            *reinterpret_cast<u32x4 *>(tile + (c >> 3) * kPanelBytes + chunk_at(r, c & 7u)) = v;
        }
        __syncthreads();

        // scores of keys 16 * wave + 4 * grp + i, in powers of two
        f32x4 s = {};
#pragma unroll
        for (int st = 0; st < kDim / 32; ++st) {
            const u32x4 k = *reinterpret_cast<const u32x4 *>(tile + (st >> 1) * kPanelBytes +
                                                             chunk_at(wave * 16 + col, (st & 1) * 4 + grp));
            s = E::mfma(k, q[st], s);
        }
        float most = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t r = wave * 16 + grp * 4 + i, k = k0 + r;
            const bool seen = keyRow[r] >= 0 && (k < a.topK || ((sees >> (k - a.topK)) & 1ull) != 0);
            s[i] = seen ? s[i] * a.scaleLog2 : -INFINITY;
            most = fmaxf(most, s[i]);   // (leaves a NaN out; its weight is one)
        }
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        if (grp == 0) part[wave][col] = most;
        __syncthreads();
        const float was = top;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, part[w][col]);
        const float base = top == -INFINITY ? 0.0f : top;
        const float keep = exp2f(was - base);
        total *= keep;
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            p[i] = exp2f(s[i] - base);
            total += p[i];
        }
        *reinterpret_cast<u32x2 *>(weights + chunk_at(col, wave * 2 + (grp >> 1)) + (grp & 1u) * 8u) =
            u32x2{pack2<T>(p[0], p[1]), pack2<T>(p[2], p[3])};
        // A drafted row that holds a NaN or an infinity must not reach the
        // queries that do not see it, whose weight 0 would turn it into a NaN;
        // those that see it have a score that is one already.
        if (k0 + kTile > a.topK) {
            for (uint32_t i = threadIdx.x; i < kTile * kLatent / 2; i += kThreads) {
                const uint32_t r = i / (kLatent / 2);
                if (k0 + r < a.topK) continue;
                const uint32_t c = i % (kLatent / 2);
                uint16_t *v = reinterpret_cast<uint16_t *>(tile + (c >> 5) * kPanelBytes + chunk_at(r, (c >> 2) & 7u) + (c & 3u) * 4u);
                constexpr uint16_t special = DTYPE == KVX_DTYPE_BF16 ? 0x7F80u : 0x7C00u;
                if ((v[0] & special) == special) v[0] = 0;
                if ((v[1] & special) == special) v[1] = 0;
            }
        }
        __syncthreads();
#pragma unroll
        for (int d = 0; d < 8; ++d) o[d] *= keep;
#pragma unroll
        for (int st = 0; st < kTile / 32; ++st) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(weights + chunk_at(col, st * 4 + grp));
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                // four keys by 16 columns a read: a lane gets its column's four keys
                const uint32_t r = st * 32 + grp * 8 + (col >> 2);
                const uint32_t c = (d & 3) * 2 + ((col & 3u) >> 1);
                const uint8_t *panel = tile + (wave * 2 + (d >> 2)) * kPanelBytes + (col & 1u) * 8u;
                typedef __attribute__((address_space(3))) s16x4 LVec;
                const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LVec *)(panel + chunk_at(r, c)));
                const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LVec *)(panel + chunk_at(r + 4, c)));
                o[d] = E::mfma(__builtin_bit_cast(u32x4, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7)), w, o[d]);
            }
        }
    }
    total += __shfl_xor(total, 16);
    total += __shfl_xor(total, 32);
    __syncthreads();
    if (grp == 0) part[wave][col] = total;
    __syncthreads();
    total = part[0][col] + part[1][col] + part[2][col] + part[3][col];
    if (!real) return;
    const uint64_t index = static_cast<uint64_t>(req) * queries + query;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    if (a.lse != 0 && wave == 0 && grp == 0) {
        reinterpret_cast<float *>(a.lse)[index] = total == 0.0f ? -INFINITY : (top + log2f(total)) * 0.6931471805599453f;
    }
    T *out = reinterpret_cast<T *>(a.out) + index * kLatent + wave * 128 + grp * 4;
#pragma unroll
    for (int d = 0; d < 8; ++d) {
        *reinterpret_cast<u32x2 *>(out + d * 16) = u32x2{pack2<T>(o[d][0] * inv, o[d][1] * inv), pack2<T>(o[d][2] * inv, o[d][3] * inv)};
    }
}

template <int DTYPE>
void launch(const AttnArgs &a, uint32_t quant, hipStream_t stream)
{
    auto *kernel = quant == KVX_QUANT_NONE     ? kvx_tree_attention<DTYPE, KVX_QUANT_NONE>
                   : quant == KVX_QUANT_LATENT ? kvx_tree_attention<DTYPE, KVX_QUANT_LATENT>
                                               : kvx_tree_attention<DTYPE, KVX_QUANT_ROW>;
    const uint32_t tiles = (a.draft * a.heads + 15u) / 16u;
    hipLaunchKernelGGL(kernel, dim3(a.reqs * tiles), dim3(kThreads), 0, stream, a);
}

}  // namespace

hipError_t launch_tree_attention(const AttnArgs &a, uint32_t dtype, uint32_t quant, hipStream_t stream)
{
    if (dtype == KVX_DTYPE_BF16) launch<KVX_DTYPE_BF16>(a, quant, stream);
    else launch<KVX_DTYPE_FP16>(a, quant, stream);
    return hipGetLastError();
}

}  // namespace kvx
