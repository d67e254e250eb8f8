// ts_prompt_attend: causal attention of packed prompts, grouped heads.
//
//   o_i = sum_{j <= i, same sequence} softmax_j(cap(scale q_i . k_j)) v_j
#include <limits.h>

#include "rope.cuh"
#include "umma.cuh"

namespace ts {
namespace {

constexpr int kPromptMaxBatch = 4096;

template <bool B> struct Flag { static constexpr bool value = B; };

struct PromptParams {
    const void* q;
    const void* k;
    const void* v;
    long long q_stride, k_stride, v_stride;
    const int* cu;
    void* out;
    int tokens, batch, hq, hkv, group;
    float sm_scale, logit_cap;
    int* status;
};

// Bounds that make no sense are reported and cut: a sequence lies in [0, tokens) and behind all before it, so no two of them share
// a token, and there are never more tiles than tokens and sequences allow.
__device__ __forceinline__ int bound_of(const PromptParams& p, int b) { return min(max(p.cu[b], 0), p.tokens); }
// Sequence b: first token and length; `floor`: the largest bound before it, and then with its own.
__device__ __forceinline__ int2 sequence_of(const PromptParams& p, int b, int& floor) {
    const int first = max(bound_of(p, b), floor), end = max(bound_of(p, b + 1), first);
    if (p.cu[b] != first || p.cu[b + 1] != end) report(p.status, TS_ERR_BAD_LENGTH);
    floor = end;
    return make_int2(first, end - first);
}
// The same for 32 sequences, a lane each (none behind the last).  All lanes call, for base = 0, 32, ... in turn.
__device__ __forceinline__ int2 sequences_of(const PromptParams& p, int base, int& floor) {
    const int lane = threadIdx.x & 31, b = base + lane;
    const bool in = b < p.batch;
    int first = in ? bound_of(p, b) : 0, end = in ? bound_of(p, b + 1) : 0;
    if (__any_sync(0xffffffffu, in && (first < floor || end < first))) {          // out of order
        int high = max(first, end);                            // of the bounds so far
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, high, off);
            if (lane >= off) high = max(high, t);
        }
        high = max(high, floor);
        const int before = __shfl_up_sync(0xffffffffu, high, 1);
        first = max(first, lane == 0 ? floor : before);
        end = high;
    }
    if (in && (p.cu[b] != first || p.cu[b + 1] != end)) report(p.status, TS_ERR_BAD_LENGTH);
    floor = __shfl_sync(0xffffffffu, end, 31);
    return make_int2(first, in ? end - first : 0);
}

// ------------------------------------------------------------------------------------------------
// CUDA cores: fp32
// ------------------------------------------------------------------------------------------------
// A CTA takes 32 query tokens of one head; keys and values pass through shared memory in tiles of 64, K of the next tile
// arriving under the second product and V under the first.  Thread (ty, tx) holds rows 4 ty .. 4 ty + 3 and, of S, columns
// tx + 16 j; of O, elements 4 tx + 64 j.  What bounds it: the multipliers (and, for few tokens, the CTA with the most keys,
// hence the small tile); products take two numbers an instruction, so that the loads of their operands find a place
// between them.
constexpr int kPpThreads = 128, kPpRows = 32, kPpTile = 64;

template <int D>
struct PromptPlainSmem {
    float q[kPpRows][D + 4];
    float k[kPpTile][D + 4];
    float v[kPpTile][D + 4];
    float p[kPpTile][kPpRows + 4];                             // [key][row]
    int tiles[kPpThreads];
    int found[3];                                              // first token, length, tile
};

// The tile'th tile of the packed sequences, the last tile of a sequence first (it has the most keys).  Returns false
// behind the last one.  All threads call.
template <int D>
__device__ __forceinline__ bool find_tile(const PromptParams& p, int tile, PromptPlainSmem<D>& sm) {
    const int per = (p.batch + kPpThreads - 1) / kPpThreads, b0 = threadIdx.x * per, b1 = min(b0 + per, p.batch);
    bool order = true;
    for (int b = b0; b < b1; ++b) order = order && p.cu[b] <= p.cu[b + 1];
    int floor0 = 0;                                            // largest bound before the thread's sequences, if it is above their first
    if (__syncthreads_or(!order)) {
        int high = 0;
        for (int b = b0; b < b1; ++b) high = max(high, max(bound_of(p, b), bound_of(p, b + 1)));
        sm.tiles[threadIdx.x] = high;
        __syncthreads();
        for (int i = 0; i < threadIdx.x; ++i) floor0 = max(floor0, sm.tiles[i]);
        __syncthreads();
    }
    int sum = 0, floor = floor0;
    for (int b = b0; b < b1; ++b) sum += (sequence_of(p, b, floor).y + kPpRows - 1) / kPpRows;
    sm.tiles[threadIdx.x] = sum;
    if (threadIdx.x == 0) sm.found[1] = 0;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < threadIdx.x; ++i) before += sm.tiles[i];
    if (tile >= before && tile < before + sum) {
        floor = floor0;
        for (int b = b0; b < b1; ++b) {
            const int2 s = sequence_of(p, b, floor);
            const int n = (s.y + kPpRows - 1) / kPpRows;
            if (tile < before + n) {
                sm.found[0] = s.x; sm.found[1] = s.y; sm.found[2] = n - 1 - (tile - before);
                break;
            }
            before += n;
        }
    }
    __syncthreads();
    return sm.found[1] > 0;
}

// Rows [row0, row0 + ROWS) of a [tokens, heads, D] tensor into shared memory; zeros from row `end` on.
template <int D, int ROWS>
__device__ __forceinline__ void request_rows(float (*dst)[D + 4], const float* src, long long stride, int row0, int end) {
    constexpr int kVecs = D / 4;
#pragma unroll 4
    for (int i = threadIdx.x; i < ROWS * kVecs; i += kPpThreads) {
        const int r = i / kVecs, c = i % kVecs * 4;
        const bool in = row0 + r < end;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(&dst[r][c])), "l"(src + (in ? (row0 + r) * stride + c : 0)), "r"(in ? 16 : 0) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void rows_here() {                  // all but the last N requests
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
    __syncthreads();
}

template <int D>
__global__ void __launch_bounds__(kPpThreads) prompt_plain_kernel(const PromptParams p) {
    extern __shared__ __align__(16) unsigned char dyn[];
    PromptPlainSmem<D>& sm = *reinterpret_cast<PromptPlainSmem<D>*>(dyn);
    constexpr int OJ = D / 64;
    const int h = blockIdx.y, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    wait_for_predecessor();
    if (!find_tile<D>(p, blockIdx.x, sm)) return;
    const int first = sm.found[0], len = sm.found[1], row0 = sm.found[2] * kPpRows;      // in the sequence
    const float* q = reinterpret_cast<const float*>(p.q) + (long long)first * p.q_stride + (long long)h * D;
    const float* k = reinterpret_cast<const float*>(p.k) + (long long)first * p.k_stride + (long long)(h / p.group) * D;
    const float* v = reinterpret_cast<const float*>(p.v) + (long long)first * p.v_stride + (long long)(h / p.group) * D;
    request_rows<D, kPpRows>(sm.q, q, p.q_stride, row0, len);
    request_rows<D, kPpTile>(sm.k, k, p.k_stride, 0, len);
    request_rows<D, kPpTile>(sm.v, v, p.v_stride, 0, len);
    const int end = min(row0 + kPpRows, len);                  // keys that the tile sees
    float m[4], l[4];
    uint64_t o[4][OJ][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int j = 0; j < OJ; ++j) o[i][j][0] = o[i][j][1] = 0ull;
    }
    for (int key0 = 0; key0 < end; key0 += kPpTile) {
        rows_here<1>();                                        // Q and K
        uint64_t s2[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s2[i][j] = 0ull;
#pragma unroll 4
        for (int d = 0; d < D; d += 4) {
            ulonglong2 a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const ulonglong2*>(&sm.q[4 * ty + i][d]);
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const ulonglong2*>(&sm.k[tx + 16 * j][d]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s2[i][j] = fma_f32x2(a[i].y, b[j].y, fma_f32x2(a[i].x, b[j].x, s2[i][j]));
        }
        __syncthreads();                                       // K has been read
        request_rows<D, kPpTile>(sm.k, k, p.k_stride, key0 + kPpTile, end);
        const bool diagonal = key0 + kPpTile > row0;
        float pe[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int lim = row0 + 4 * ty + i - key0;          // the row sees keys up to this one of the tile
            float s[4], mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float even, odd;
                unpack_f32x2(s2[i][j], even, odd);
                float x = (even + odd) * p.sm_scale;
                if (p.logit_cap > 0.f) x = p.logit_cap * tanhf(x / p.logit_cap);
                s[j] = diagonal && tx + 16 * j > lim ? -INFINITY : x * 1.4426950408889634f;
                mx = fmaxf(mx, s[j]);
            }
#pragma unroll
            for (int off = 1; off < 16; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            const float mn = fmaxf(m[i], mx), base = mn == -INFINITY ? 0.f : mn, corr = exp2f(m[i] - base);
            m[i] = mn;
            l[i] *= corr;                                      // this thread's columns; joined at the end
            const uint64_t corr2 = pack_f32x2(corr, corr);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                pe[j][i] = exp2f(s[j] - base);
                l[i] += pe[j][i];
            }
#pragma unroll
            for (int j = 0; j < OJ; ++j) {
                o[i][j][0] = mul_f32x2(o[i][j][0], corr2);
                o[i][j][1] = mul_f32x2(o[i][j][1], corr2);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<float4*>(&sm.p[tx + 16 * j][4 * ty]) = make_float4(pe[j][0], pe[j][1], pe[j][2], pe[j][3]);
        rows_here<1>();                                        // V; and P
        // On the diagonal a masked weight is 0, but 0 times a later token's infinity is not: those products are left out.
        const int keys = min(kPpTile, end - key0);
        auto products = [&](auto masked) {
#pragma unroll 4
            for (int c = 0; c < keys; ++c) {
                ulonglong2 b[OJ];
#pragma unroll
                for (int j = 0; j < OJ; ++j) b[j] = *reinterpret_cast<const ulonglong2*>(&sm.v[c][4 * tx + 64 * j]);
                const float4 a4 = *reinterpret_cast<const float4*>(&sm.p[c][4 * ty]);
                const float a[4] = {a4.x, a4.y, a4.z, a4.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (!decltype(masked)::value || key0 + c <= row0 + 4 * ty + i) {
                        const uint64_t a2 = pack_f32x2(a[i], a[i]);
#pragma unroll
                        for (int j = 0; j < OJ; ++j) {
                            o[i][j][0] = fma_f32x2(a2, b[j].x, o[i][j][0]);
                            o[i][j][1] = fma_f32x2(a2, b[j].y, o[i][j][1]);
                        }
                    }
                }
            }
        };
        if (diagonal) products(Flag<true>()); else products(Flag<false>());
        __syncthreads();                                       // V and P have been read
        request_rows<D, kPpTile>(sm.v, v, p.v_stride, key0 + kPpTile, end);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");       // (zeros, requested behind the last tile)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float sum = l[i];
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        const int row = row0 + 4 * ty + i;
        if (row >= len) continue;
        float* out = reinterpret_cast<float*>(p.out) + ((long long)(first + row) * p.hq + h) * D;
#pragma unroll
        for (int j = 0; j < OJ; ++j) {
            float x[4];
            unpack_f32x2(o[i][j][0], x[0], x[1]);
            unpack_f32x2(o[i][j][1], x[2], x[3]);
            *reinterpret_cast<float4*>(out + 4 * tx + 64 * j) = make_float4(x[0] / sum, x[1] / sum, x[2] / sum, x[3] / sum);
        }
    }
}

template <int D>
cudaError_t launch_prompt_plain(const PromptParams& p, cudaStream_t stream) {
    static SmemConfig configured = {};
    constexpr size_t kSmem = sizeof(PromptPlainSmem<D>);
    const cudaError_t e = ensure_dynamic_smem(prompt_plain_kernel<D>, kSmem, configured);
    if (e != cudaSuccess) return e;
    return launch_chained(prompt_plain_kernel<D>, dim3(p.tokens / kPpRows + p.batch, p.hq), dim3(kPpThreads), kSmem, stream, p);
}

// ------------------------------------------------------------------------------------------------
// Tensor cores: bf16
// ------------------------------------------------------------------------------------------------
// A CTA takes tiles of 256 query tokens of one head as two halves of 128 rows, keys in blocks of 128:
//   S_h (128 x 128 fp32)  = Q_h (shared memory, K-major) . K_b^T (shared memory, K-major)
//   O_h (128 x D fp32)   += P_h (tensor memory, packed bf16, in the place of S_h) . V_b (shared memory, MN-major)
// with S_0, S_1, O_0, O_1 in the 512 columns of tensor memory.  One thread issues every product, in the order
//   P.V of half 0, Q.K^T of half 0 for the next block, P.V of half 1, Q.K^T of half 1 for the next block, ...
// so the tensor pipe works on one half while 128 threads (one per row, so the row's maximum and sum need no exchange) turn
// the other half's S into P.  A half's Q.K^T may overwrite its P because the products of one thread run in order, and S
// complete means that every earlier P.V is: so those 128 threads also rescale O themselves.
//
// What bounds it, in this order as it was met (8192 tokens, 32 heads, 550 GFLOP):
//  * the operands of the issuing thread.  Behind `lane == 0` each product's descriptors were moved into uniform registers
//    anew, 80 cycles a product; behind elect.sync they are not (1091 -> 1190 TFLOP/s).
//  * the way from S to P.  The weights of a block are taken with the reference that the blocks before left, 32 columns at a
//    time as they arrive, instead of after the block's maximum: P in bf16 holds 2^127 as well as 1, so a maximum that grew
//    is caught up with, by rescaling O and the sum, before the next block, and only when it grew by more than 2^8.  (A jump of
//    more than 2^100 inside a block, which O might not hold, sends the row to the CUDA cores.)  P is handed over in two
//    parts.  One pair of columns in four takes its exponentials on the multipliers: the exponential unit alone would need as
//    long as the tensor pipe.  (1190 -> 1283; without the multipliers 1239, with one pair in three 1246, in eight 1230, P in
//    one part 1218.)
//  * now: that way still (the tensor pipe is busy for 65 % of the cycles, the exponential unit for 49 %), and the clock, which the
//    card's power limit takes from 1.965 to 1.58 GHz when the kernel runs on (435 us after a pause, 516 us then, whether on one
//    input or on changing ones).
//
// One thread requests tiles (tiled copies, 128-byte swizzle): Q, and K and V blocks through a ring of five.  It runs ahead
// into the CTA's next tile, of which it leaves the place in a two-entry queue.  Tiles are dealt out in the order of their
// last key, longest first, heads innermost (the heads that share K and V run side by side).
//
// What is not finite.  A masked weight is 0, but 0 times an infinity in V is not; the block on the diagonal holds the V of
// later tokens, and of the next sequence.  Only then does a row of O end up non-finite without cause, and mend_rows() has such
// rows computed again on the CUDA cores, from the keys that they see.  That is slow (150 cycles a key and warp), but few rows: one
// undefined value at the start of 16384 tokens, 8 heads, 1.0 ms in place of 0.45.  Rows whose logits jump by more than 2^100
// inside a block are not few where all logits are of that size (the same shape, logits of +-160: 83 ms), so while a warp is
// at work on rows the clock of its CTA's waits stands still.
constexpr int kPtRows = 128, kPtBlock = 128;                   // rows of a half, keys of a block
constexpr int kPtStages = 5, kPtThreads = 320;                 // two times four softmax warps, one that issues products, one that requests tiles
constexpr int kPtQueue = 2;
constexpr float kPtLowest = -3e38f;                            // reference of a row none of whose logits is above it

template <int D>
struct PromptTcSmem {
    unsigned char q[2][kPtRows * D * 2];                       // per half: D/64 parts of [128 rows][128 bytes]
    unsigned char kv[kPtStages][kPtBlock * D * 2];
    int4 queue[kPtQueue];                                      // first token, length, tile, head; length -1: no more
    uint64_t q_full, q_empty, kv_full[kPtStages], kv_empty[kPtStages], s_full[2], p_full[2][2], o_full[2], o_empty[2];
    uint64_t queue_full[kPtQueue], queue_empty[kPtQueue], drained;
    uint32_t tmem;
    int slow;                                                  // warps that compute rows again
    unsigned jumped[8];                                        // per softmax warp: rows of the tile whose logits jumped
};

// Blocks of keys that half h of a tile sees; 0 when the sequence ends before it.
__device__ __forceinline__ int blocks_of(int len, int tile, int h) {
    const int row0 = tile * 2 * kPtRows + h * kPtRows;
    return row0 < len ? min(row0 + kPtRows - 1, len - 1) / kPtBlock + 1 : 0;
}

// The warp that deals out tiles: positions 0, 1, ... name (sequence, tile) pairs by falling tile number, sequences in order
// within one.
struct TileOrder {
    int level, from;                                           // tiles of this number start at position `from`
};
__device__ __forceinline__ int tiles_of(int2 sequence) { return (sequence.y + 2 * kPtRows - 1) / (2 * kPtRows); }
__device__ int count_tiles(const PromptParams& p, int above) {     // sequences with more tiles than `above`; all lanes call
    int n = 0, floor = 0;
    for (int base = 0; base < p.batch; base += 32) n += __popc(__ballot_sync(0xffffffffu, tiles_of(sequences_of(p, base, floor)) > above));
    return n;
}
// The sequence (first token, length) at place `rank` among those with more tiles than `level`; all lanes call.
__device__ int2 sequence_at(const PromptParams& p, int level, int rank) {
    int floor = 0;
    for (int base = 0; base < p.batch; base += 32) {
        const int2 s = sequences_of(p, base, floor);
        const unsigned has = __ballot_sync(0xffffffffu, tiles_of(s) > level);
        const int n = __popc(has);
        if (rank < n) {
            const int from = __fns(has, 0, rank + 1);
            return make_int2(__shfl_sync(0xffffffffu, s.x, from), __shfl_sync(0xffffffffu, s.y, from));
        }
        rank -= n;
    }
    return make_int2(0, 0);
}

// Row `row` of a sequence for one head on the CUDA cores, by one warp: D/8 lanes hold a key's or a value's row, eight elements each,
// 32 keys a step, of which every lane then has one logit.
template <int D>
__device__ __noinline__ void prompt_row(const PromptParams& p, int first, int row, int h) {
    constexpr int kLanes = D / 8, kKeys = 32 / kLanes;         // keys of one load
    const int lane = threadIdx.x & 31, c = lane % kLanes, g = lane / kLanes;
    const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(p.q) + (long long)(first + row) * p.q_stride + (long long)h * D + 8 * c;
    const __nv_bfloat16* k = reinterpret_cast<const __nv_bfloat16*>(p.k) + (long long)first * p.k_stride + (long long)(h / p.group) * D + 8 * c;
    const __nv_bfloat16* v = reinterpret_cast<const __nv_bfloat16*>(p.v) + (long long)first * p.v_stride + (long long)(h / p.group) * D + 8 * c;
    auto floats = [](uint4 a, float (&x)[8]) {
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) { x[2 * e] = __uint_as_float(w[e] << 16); x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
    };
    float x[8], y[8], o[8], m = -INFINITY, l = 0.f;
    floats(*reinterpret_cast<const uint4*>(q), x);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = 0.f;
    for (int key0 = 0; key0 <= row; key0 += 32) {
        float s[kLanes];
#pragma unroll
        for (int i = 0; i < kLanes; ++i) {                     // (behind the row's own key: that one again)
            floats(*reinterpret_cast<const uint4*>(k + min(key0 + i * kKeys + g, row) * p.k_stride), y);
            s[i] = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) s[i] = fmaf(x[e], y[e], s[i]);
        }
        // lane (g, c) ends up with the whole sum of key key0 + c * kKeys + g
#pragma unroll
        for (int off = kLanes / 2; off >= 1; off >>= 1) {
            const bool up = (c & off) != 0;
#pragma unroll
            for (int i = 0; i < off; ++i) {
                const float keep = up ? s[i + off] : s[i], send = up ? s[i] : s[i + off];
                s[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
            }
        }
        float logit = s[0] * p.sm_scale;
        if (p.logit_cap > 0.f) logit = p.logit_cap * tanhf(logit / p.logit_cap);
        logit = key0 + c * kKeys + g <= row ? logit * 1.4426950408889634f : -INFINITY;
        float mn = fmaxf(m, logit);
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, off));
        const float base = mn == -INFINITY ? 0.f : mn, corr = exp2f(m - base), w = exp2f(logit - base);
        m = mn;
        l = l * corr + w;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] *= corr;
#pragma unroll
        for (int i = 0; i < kLanes; ++i) {
            const int key = key0 + i * kKeys + g;
            const float wi = __shfl_sync(0xffffffffu, w, g * kLanes + i);
            const uint4 raw = *reinterpret_cast<const uint4*>(v + min(key, row) * p.v_stride);
            floats(key <= row ? raw : make_uint4(0u, 0u, 0u, 0u), y);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = fmaf(wi, y[e], o[e]);
        }
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
#pragma unroll
    for (int off = 16; off >= kLanes; off >>= 1)
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] += __shfl_xor_sync(0xffffffffu, o[e], off);
    if (g == 0)
        *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.out) + ((long long)(first + row) * p.hq + h) * D + 8 * c) =
            make_uint4(pack_bf16x2(o[0] / l, o[1] / l), pack_bf16x2(o[2] / l, o[3] / l), pack_bf16x2(o[4] / l, o[5] / l), pack_bf16x2(o[6] / l, o[7] / l));
}

// Rows of 32 that came out non-finite (bits of `rows`; a lane's row is row0 + lane): which of them the tensor cores may have
// got wrong, and those again.
//
// A row whose logits jumped (bits of `jumped`) is one.  Of the others the products are right but for what masked values of
// the last block add, 0 times an infinity: a column of O that is not finite for another reason has met a value that is not
// finite in the blocks before, all of whose keys the row sees.  So a column that is finite there and is not in the result sends
// its row to be computed again, and the rest stays as it is.  That bounds the work: one undefined value early in a
// sequence makes every later row undefined, but only rows of the blocks in which a column first became so are computed
// again, at most 128 for each column.
template <int D>
__device__ __noinline__ void mend_rows(const PromptParams& p, int first, int row0, int before, int h, unsigned rows, unsigned jumped) {
    constexpr int kLanes = D / 8, kKeys = 32 / kLanes;
    const int lane = threadIdx.x & 31, c = lane % kLanes, g = lane / kLanes;
    uint32_t top[4] = {0u, 0u, 0u, 0u};                        // of the values before: largest magnitudes of the lane's eight columns
    if ((rows & ~jumped) != 0) {
        const __nv_bfloat16* v = reinterpret_cast<const __nv_bfloat16*>(p.v) + (long long)first * p.v_stride + (long long)(h / p.group) * D + 8 * c;
        for (int key0 = 0; key0 < before; key0 += 64) {        // (before: a multiple of 128)
#pragma unroll
            for (int i = 0; i < 64 / kKeys; ++i) {
                const uint4 x = *reinterpret_cast<const uint4*>(v + (key0 + i * kKeys + g) * p.v_stride);
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) top[e] = __vmaxu2(top[e], w[e] & 0x7fff7fffu);
            }
        }
#pragma unroll
        for (int off = 16; off >= kLanes; off >>= 1)
#pragma unroll
            for (int e = 0; e < 4; ++e) top[e] = __vmaxu2(top[e], __shfl_xor_sync(0xffffffffu, top[e], off));
    }
    for (; rows != 0; rows &= rows - 1) {
        const int i = __ffs(rows) - 1;
        bool again = (jumped >> i & 1) != 0;
        if (!again) {
            const uint4 x = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p.out) + ((long long)(first + row0 + i) * p.hq + h) * D + 8 * c);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                again = again || ((w[e] & 0x7f80u) == 0x7f80u && (top[e] & 0xffffu) < 0x7f80u) || ((w[e] & 0x7f800000u) == 0x7f800000u && top[e] < 0x7f800000u);
        }
        if (__any_sync(0xffffffffu, again)) prompt_row<D>(p, first, row0 + i, h);
    }
    __syncwarp();
}

// 2^x of two numbers on the multipliers, for x >= -125 (below, and for minus infinity and NaN, 2^-125): 2^n 2^f with n the
// nearest whole number and 2^f a polynomial of degree 3 (Remez exchange: 7.5e-5 relative on [-1/2, 1/2], a twentieth of the weight's rounding to bf16).
__device__ __forceinline__ uint64_t exp2_f32x2(uint64_t x) {
    float a, b;
    unpack_f32x2(x, a, b);
    x = pack_f32x2(fmaxf(a, -125.f), fmaxf(b, -125.f));
    const uint64_t magic = pack_f32x2(12582912.f, 12582912.f), minus = pack_f32x2(-12582912.f, -12582912.f);      // 1.5 * 2^23
    const uint64_t n = add_f32x2(x, magic);                    // the nearest whole number in the lowest bits
    const uint64_t f = fma_f32x2(add_f32x2(n, minus), pack_f32x2(-1.f, -1.f), x);
    uint64_t y = fma_f32x2(f, pack_f32x2(0.0551716691f, 0.0551716691f), pack_f32x2(0.2426111222f, 0.2426111222f));
    y = fma_f32x2(y, f, pack_f32x2(0.6932609855f, 0.6932609855f));
    y = fma_f32x2(y, f, pack_f32x2(0.9999280735f, 0.9999280735f));
    float ya, yb, na, nb;
    unpack_f32x2(y, ya, yb);
    unpack_f32x2(n, na, nb);
    return pack_f32x2(__int_as_float(__float_as_int(ya) + (__float_as_int(na) << 23)), __int_as_float(__float_as_int(yb) + (__float_as_int(nb) << 23)));
}

// The largest, and NaN where one of them is: what the multipliers make of an undefined logit is a number like any other, so the
// maximum is what remembers it.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// True for one lane of a converged warp.  (With `lane == 0` in its place the compiler does not know the code behind it to be
// uniform and moves every operand of every product into uniform registers anew.)
__device__ __forceinline__ bool elect_one() {
    uint32_t is;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
    return is != 0;
}

template <int D, bool CAP>
__global__ void __launch_bounds__(kPtThreads, 1) prompt_tc_kernel(const __grid_constant__ PromptParams p, const __grid_constant__ CUtensorMap map_q,
                                                                  const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    constexpr int kParts = D / 64;
    constexpr uint32_t kPart = kPtRows * 128, kTile = kPart * kParts;      // bytes of 128 rows of 64 elements; of a tile
    constexpr uint32_t kO = 256;                               // tensor memory: S_h at column 128 h, O_h at 256 + 128 h
    extern __shared__ unsigned char dyn[];
    PromptTcSmem<D>& sm = *reinterpret_cast<PromptTcSmem<D>*>(dyn + ((1024u - (smem_u32(dyn) & 1023u)) & 1023u));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        sm.slow = 0;
        for (int i = 0; i < 8; ++i) sm.jumped[i] = 0u;
        mbar_init(smem_u32(&sm.q_full), 1);
        mbar_init(smem_u32(&sm.q_empty), 1);
        mbar_init(smem_u32(&sm.drained), 1);
        for (int i = 0; i < kPtStages; ++i) { mbar_init(smem_u32(&sm.kv_full[i]), 1); mbar_init(smem_u32(&sm.kv_empty[i]), 1); }
        for (int h = 0; h < 2; ++h) {
            mbar_init(smem_u32(&sm.s_full[h]), 1);
            mbar_init(smem_u32(&sm.p_full[h][0]), 4);
            mbar_init(smem_u32(&sm.p_full[h][1]), 4);
            mbar_init(smem_u32(&sm.o_full[h]), 1);
            mbar_init(smem_u32(&sm.o_empty[h]), 4);
        }
        for (int i = 0; i < kPtQueue; ++i) { mbar_init(smem_u32(&sm.queue_full[i]), 1); mbar_init(smem_u32(&sm.queue_empty[i]), 9); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sm.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_before_sync();
    __syncthreads();
    tcgen05_after_sync();
    const uint32_t tmem = *(volatile uint32_t*)&sm.tmem;
    wait_for_predecessor();
    bool dead = false;
    // an entry of the queue; the last one says that there are no more
    int taken = 0;
    auto next_tile = [&]() {
        const int i = taken % kPtQueue;
        wait_phase(smem_u32(&sm.queue_full[i]), taken / kPtQueue & 1, p.status, dead, &sm.slow);
        dead = __any_sync(0xffffffffu, dead);                  // a warp gives up as one
        const int4 t = dead ? make_int4(0, -1, 0, 0) : sm.queue[i];
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.queue_empty[i]));
        ++taken;
        return t;
    };

    if (warp == 9) {
        // ---------------- requests ----------------
        TileOrder order = {0, 0};
        {
            int most = 0, floor = 0;
            for (int base = 0; base < p.batch; base += 32) most = max(most, tiles_of(sequences_of(p, base, floor)));
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, off));
            order.level = most - 1;
        }
        int here = order.level >= 0 ? count_tiles(p, order.level) : 0;     // tiles of this number
        int kv = 0, put = 0;                                   // blocks requested, entries left so far
        for (long long round = 0;; ++round, ++put) {
            // items in snake order, so that a CTA's long and short ones balance
            const long long item = round * gridDim.x + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
            const int pos = (int)min(item / p.hq, (long long)INT_MAX), head = (int)(item % p.hq);
            while (order.level >= 0 && pos - order.from >= here) {
                order.from += here;
                --order.level;
                here = order.level >= 0 ? count_tiles(p, order.level) : 0;
            }
            int4 t = make_int4(0, -1, 0, head);
            if (order.level >= 0 && !dead) {
                const int2 seq = sequence_at(p, order.level, pos - order.from);
                t = make_int4(seq.x, seq.y, order.level, head);
            }
            const int i = put % kPtQueue;
            wait_phase(smem_u32(&sm.queue_empty[i]), (put / kPtQueue & 1) ^ 1, p.status, dead, &sm.slow);
            dead = __any_sync(0xffffffffu, dead);
            if (dead) t.y = -1;
            __syncwarp();
            if (lane == 0) { sm.queue[i] = t; mbar_arrive(smem_u32(&sm.queue_full[i])); }
            if (t.y < 0) break;
            const int n0 = blocks_of(t.y, t.z, 0), n1 = blocks_of(t.y, t.z, 1), n = max(n0, n1);
            if (lane == 0) {
                wait_phase(smem_u32(&sm.q_empty), (put & 1) ^ 1, p.status, dead, &sm.slow);
                mbar_expect_tx(smem_u32(&sm.q_full), n1 > 0 ? 2 * kTile : kTile);
                for (int h = 0; h < (n1 > 0 ? 2 : 1); ++h)
                    for (int c = 0; c < kParts; ++c)
                        tile_g2s(smem_u32(sm.q[h]) + c * kPart, &map_q, 64 * c, t.w, t.x + t.z * 2 * kPtRows + h * kPtRows, smem_u32(&sm.q_full));
                for (int j = 0; j < 2 * n; ++j, ++kv) {        // K_0, V_0, K_1, ...
                    const int s = kv % kPtStages;
                    wait_phase(smem_u32(&sm.kv_empty[s]), (kv / kPtStages & 1) ^ 1, p.status, dead, &sm.slow);
                    mbar_expect_tx(smem_u32(&sm.kv_full[s]), kTile);
                    for (int c = 0; c < kParts; ++c)
                        tile_g2s(smem_u32(sm.kv[s]) + c * kPart, j & 1 ? &map_v : &map_k, 64 * c, t.w / p.group, t.x + (j >> 1) * kPtBlock, smem_u32(&sm.kv_full[s]));
                }
            }
            __syncwarp();
            kv = __shfl_sync(0xffffffffu, kv, 0);
        }
        if (lane == 0 && dead) {                               // given up: the copies still have to land (or time out)
            for (int i = max(kv - kPtStages, 0); i < kv; ++i) {
                bool gone = false;
                wait_phase(smem_u32(&sm.kv_full[i % kPtStages]), i / kPtStages & 1, p.status, gone, &sm.slow);
            }
            bool gone = false;
            if (put > 0) wait_phase(smem_u32(&sm.q_full), (put - 1) & 1, p.status, gone, &sm.slow);
        }
        __syncwarp();
    } else if (warp == 8) {
        // ---------------- products ----------------
        // instruction descriptors: fp32 accumulate, bf16 A and B, M = 128; N = 128 with K-major B, N = D with MN-major B
        constexpr uint32_t kIdescQK = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
        constexpr uint32_t kIdescPV = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (((uint32_t)D >> 3) << 17) | ((128u >> 4) << 24);
        int kv = 0, tiles = 0, p_count[2] = {0, 0}, o_count[2] = {0, 0};
        for (;;) {
            const int4 t = next_tile();
            const int len = __shfl_sync(0xffffffffu, t.y, 0), tile = __shfl_sync(0xffffffffu, t.z, 0);
            if (len < 0) break;
            const int n_of[2] = {blocks_of(len, tile, 0), blocks_of(len, tile, 1)}, n = max(n_of[0], n_of[1]);
            if (elect_one()) {
                auto wait_block = [&](int i) {                 // block i of the tile's K_0, V_0, K_1, ...
                    const int s = (kv + i) % kPtStages;
                    wait_phase(smem_u32(&sm.kv_full[s]), (kv + i) / kPtStages & 1, p.status, dead, &sm.slow);
                    tcgen05_after_sync();
                    return smem_u32(sm.kv[s]);
                };
                auto free_block = [&](int i) { mma_commit(smem_u32(&sm.kv_empty[(kv + i) % kPtStages])); };
                auto issue_qk = [&](int h, uint32_t k) {
                    const uint32_t q = smem_u32(sm.q[h]);
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) {
                        const uint32_t off = (ks >> 2) * kPart + (ks & 3) * 32u;
                        mma_ss(tmem + 128u * h, sw128_operand(q + off, 16, 1024), sw128_operand(k + off, 16, 1024), kIdescQK, ks > 0 ? 1u : 0u);
                    }
                    mma_commit(smem_u32(&sm.s_full[h]));
                };
                auto issue_pv = [&](int h, uint32_t v, bool first) {
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {           // 16 keys a step: 8 columns of P, which comes in two parts
                        if (ks % 4 == 0) {
                            wait_phase(smem_u32(&sm.p_full[h][ks / 4]), p_count[h] & 1, p.status, dead, &sm.slow);
                            tcgen05_after_sync();
                        }
                        mma_ts(tmem + kO + 128u * h, tmem + 128u * h + 8u * ks, sw128_operand(v + ks * 2048u, kPart, 1024), kIdescPV, !first || ks > 0 ? 1u : 0u);
                    }
                    ++p_count[h];
                };
                wait_phase(smem_u32(&sm.q_full), tiles & 1, p.status, dead, &sm.slow);
                uint32_t k = wait_block(0);
                issue_qk(0, k);
                if (n_of[1] > 0) issue_qk(1, k);
                free_block(0);
                if (n == 1) mma_commit(smem_u32(&sm.q_empty));
                for (int j = 0; j < n; ++j) {
                    const uint32_t v = wait_block(2 * j + 1);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (j < n_of[h]) {
                            if (j == 0) {                      // the half's last result has been read
                                wait_phase(smem_u32(&sm.o_empty[h]), (o_count[h] & 1) ^ 1, p.status, dead, &sm.slow);
                                ++o_count[h];
                            }
                            issue_pv(h, v, j == 0);
                            if (j + 1 == n_of[h]) mma_commit(smem_u32(&sm.o_full[h]));
                        }
                        if (j + 1 < n_of[h]) issue_qk(h, wait_block(2 * j + 2));
                    }
                    free_block(2 * j + 1);
                    if (j + 1 < n) free_block(2 * j + 2);
                    if (j + 2 == n) mma_commit(smem_u32(&sm.q_empty));
                }
            }
            __syncwarp();
            kv += 2 * n;
            ++tiles;
        }
        if (lane == 0 && dead) {                               // given up: the products still have to end (or time out)
            bool gone = false;
            mma_commit(smem_u32(&sm.drained));
            wait_phase(smem_u32(&sm.drained), 0, p.status, gone, &sm.slow);
        }
        __syncwarp();
    } else {
        // ---------------- softmax: half h, row r of it ----------------
        const int h = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t at_s = tmem + ((uint32_t)(warp & 3) << 21) + 128u * h, at_o = at_s + kO;
        const float cap = p.logit_cap, mul = CAP ? 1.f : p.sm_scale * 1.4426950408889634f;      // x * mul: base-2 units
        int s_count = 0, o_count = 0;
        for (;;) {
            const int4 t = next_tile();
            if (t.y < 0) break;
            const int n = blocks_of(t.y, t.z, h);
            if (n == 0) continue;
            const int row = t.z * 2 * kPtRows + h * kPtRows + r;                  // in the sequence
            float ref = 0.f, top_x = 0.f;                      // the row's reference; its largest logit so far
            uint64_t sums[2] = {0ull, 0ull};                   // relative to the reference
            bool fresh = true;
            auto block = [&](auto last) {
                constexpr bool diagonal = decltype(last)::value;
                float x[2][32];
                tmem_load32(at_s, x[0]);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float (&y32)[32] = x[c & 1];
                    tmem_loads_done();
                    if (c < 3) tmem_load32(at_s + 32u * (c + 1), x[(c + 1) & 1]);
                    if (CAP) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) y32[e] = cap * tanhf(y32[e] * p.sm_scale / cap) * 1.4426950408889634f;
                    }
                    if (diagonal) {                            // the last block; keys behind the sequence's end lie behind every row too
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (32 * c + e > r) y32[e] = -INFINITY;
                    }
                    float m4[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        m4[i] = max_nan(y32[i], y32[4 + i], y32[8 + i]);
                        m4[i] = max_nan(m4[i], y32[12 + i], y32[16 + i]);
                        m4[i] = max_nan(m4[i], y32[20 + i], y32[24 + i]);
                        m4[i] = max_nan(m4[i], y32[28 + i]);
                    }
                    const float mx = max_nan(max_nan(m4[0], m4[1], m4[2]), m4[3]) * mul;
                    if (fresh) {                               // any number near the maximum will do: that of the first 32 keys
                        ref = fmaxf(mx, kPtLowest);
                        top_x = ref;
                        fresh = false;
                    }
                    top_x = max_nan(top_x, mx);
                    const uint64_t mul2 = pack_f32x2(mul, mul), ref2 = pack_f32x2(-ref, -ref);
                    uint32_t w[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        uint64_t y = fma_f32x2(pack_f32x2(y32[2 * e], y32[2 * e + 1]), mul2, ref2);
                        float p0, p1;
                        if (!diagonal && (e & 3) == 3) {       // (a masked weight has to be exactly 0)
                            y = exp2_f32x2(y);
                            unpack_f32x2(y, p0, p1);
                        } else {
                            unpack_f32x2(y, p0, p1);
                            asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(p0));
                            asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(p1));
                            y = pack_f32x2(p0, p1);
                        }
                        sums[e & 1] = add_f32x2(sums[e & 1], y);
                        w[e] = pack_bf16x2(p0, p1);
                    }
                    tmem_store16(at_s + 16u * c, w);           // into columns that have been read
                    if (c & 1) {
                        tmem_stores_done();
                        tcgen05_before_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&sm.p_full[h][c >> 1]));
                    }
                }
            };
            for (int j = 0; j < n; ++j) {
                wait_phase(smem_u32(&sm.s_full[h]), s_count & 1, p.status, dead, &sm.slow);
                ++s_count;
                tcgen05_after_sync();
                // The blocks before raised a row's maximum by more than 2^8: O (every P.V so far is complete) and the sum follow.
                if (__any_sync(0xffffffffu, top_x > ref + 8.f)) {
                    const bool grown = top_x > ref + 8.f;
                    const float corr = grown ? exp2f(ref - top_x) : 1.f;
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        float o[32];
                        tmem_load32(at_o + 32u * c, o);
                        tmem_loads_done();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] *= corr;
                        tmem_store32(at_o + 32u * c, reinterpret_cast<const uint32_t*>(o));
                    }
                    const uint64_t corr2 = pack_f32x2(corr, corr);
                    sums[0] = mul_f32x2(sums[0], corr2);
                    sums[1] = mul_f32x2(sums[1], corr2);
                    // a jump that P, up to 2^127 in bf16, or O would not hold: the row is computed again at the end
                    const unsigned far = __ballot_sync(0xffffffffu, row < t.y && top_x > ref + 100.f);
                    if (far != 0) {
                        if (top_x > ref + 100.f) sums[0] = pack_f32x2(__int_as_float(0x7fc00000), 0.f);
                        if (lane == 0) sm.jumped[warp] |= far;
                    }
                    if (grown) ref = top_x;
                }
                if (j == n - 1) block(Flag<true>()); else block(Flag<false>());
            }
            float sum, sum1;
            unpack_f32x2(add_f32x2(sums[0], sums[1]), sum, sum1);
            sum += sum1;
            // (an undefined or infinite logit makes the row undefined, and so do logits that are minus infinity without exception)
            const bool defined = top_x > kPtLowest && top_x <= 3.4028235e38f;
            if (!(defined && top_x <= ref + 100.f)) sum = __int_as_float(0x7fc00000);
            // the result
            wait_phase(smem_u32(&sm.o_full[h]), o_count & 1, p.status, dead, &sm.slow);
            ++o_count;
            tcgen05_after_sync();
            const float inv = 1.f / sum;
            __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(p.out) + ((long long)(t.x + row) * p.hq + t.w) * D;
            uint32_t top = 0;                                  // largest magnitude, NaN counting as the largest
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                float o[32];
                tmem_load32(at_o + 32u * c, o);
                tmem_loads_done();
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    o[e] *= inv;
                    top = max(top, __float_as_uint(o[e]) & 0x7fffffffu);
                }
                if (row < t.y) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
                        *reinterpret_cast<uint4*>(out + 32 * c + e) = make_uint4(pack_bf16x2(o[e], o[e + 1]), pack_bf16x2(o[e + 2], o[e + 3]),
                                                                                 pack_bf16x2(o[e + 4], o[e + 5]), pack_bf16x2(o[e + 6], o[e + 7]));
                }
            }
            tcgen05_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sm.o_empty[h]));
            if (__any_sync(0xffffffffu, row < t.y && top >= 0x7f800000u)) {      // rows that are not finite
                const unsigned jumped = (sm.jumped[warp] | __ballot_sync(0xffffffffu, top_x > ref + 100.f)) & __ballot_sync(0xffffffffu, defined);
                const bool mine = jumped >> lane & 1;
                // (a row whose sum is undefined without a jump is undefined with cause, in every column)
                const unsigned rows = __ballot_sync(0xffffffffu, row < t.y && top >= 0x7f800000u && (sum == sum || mine));
                __syncwarp();
                if (lane == 0) sm.jumped[warp] = 0u;
                if (rows != 0) {                               // (row by row: the other warps' waits have to be patient)
                    if (lane == 0) atomicAdd(&sm.slow, 1);
                    mend_rows<D>(p, t.x, row - lane, (n - 1) * kPtBlock, t.w, rows, jumped);
                    if (lane == 0) atomicSub(&sm.slow, 1);
                }
            }
        }
    }
    tcgen05_before_sync();
    __syncthreads();
    if (warp == 8) {
        tcgen05_after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled f = [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
            ptr = nullptr;
        return reinterpret_cast<EncodeTiled>(ptr);
    }();
    return f;
}
// [tokens][heads][D] bf16, boxes of 128 tokens x one head x 64 elements, 128-byte swizzle, zeros outside.
bool tensor_map(CUtensorMap& m, const void* base, int d, int heads, int tokens, long long stride) {
    const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)tokens}, strides[2] = {(cuuint64_t)d * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64, 1, kPtBlock}, step[3] = {1, 1, 1};
    return encode_tiled()(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool CAP>
cudaError_t launch_prompt_tc(const PromptParams& p, int sms, cudaStream_t stream) {
    static SmemConfig configured = {};
    constexpr size_t kSmem = sizeof(PromptTcSmem<D>) + 1024;
    static_assert(kSmem <= 232448, "the kernel's shared memory must fit one CTA's maximum");
    const cudaError_t e = ensure_dynamic_smem(prompt_tc_kernel<D, CAP>, kSmem, configured);
    if (e != cudaSuccess) return e;
    CUtensorMap q, k, v;
    if (!encode_tiled() || !tensor_map(q, p.q, D, p.hq, p.tokens, p.q_stride) || !tensor_map(k, p.k, D, p.hkv, p.tokens, p.k_stride) ||
        !tensor_map(v, p.v, D, p.hkv, p.tokens, p.v_stride))
        return cudaErrorInvalidValue;
    const long long items = ((long long)p.tokens / (2 * kPtRows) + p.batch) * p.hq;       // at most
    return launch_chained(prompt_tc_kernel<D, CAP>, dim3((unsigned)(items < sms ? items : sms)), dim3(kPtThreads), kSmem, stream, p, q, k, v);
}

}  // namespace
}  // namespace ts

extern "C" int ts_prompt_attend(const ts_prompt_args* a) {
    using namespace ts;
    if (!a || a->struct_size != sizeof(ts_prompt_args)) return TS_ERR_INVALID_ARG;
    if (a->dtype != TS_DTYPE_BF16 && a->dtype != TS_DTYPE_F32) return TS_ERR_UNSUPPORTED;
    if (a->head_dim != 64 && a->head_dim != 128) return TS_ERR_UNSUPPORTED;
    if (a->tokens < 0 || a->batch < 0 || a->batch > kPromptMaxBatch || a->hq < 1 || a->hkv < 1 || a->hq > 8192 || a->hq % a->hkv != 0) return TS_ERR_INVALID_ARG;
    if (a->q_stride < (int64_t)a->hq * a->head_dim || a->k_stride < (int64_t)a->hkv * a->head_dim || a->v_stride < (int64_t)a->hkv * a->head_dim) return TS_ERR_INVALID_ARG;
    if (!positive(a->sm_scale) || !isfinite(a->logit_cap)) return TS_ERR_INVALID_ARG;
    if (a->tokens == 0 || a->batch == 0) return TS_OK;
    if (!a->q || !a->k || !a->v || !a->cu_seqlens || !a->out) return TS_ERR_INVALID_ARG;
    const int es = a->dtype == TS_DTYPE_BF16 ? 2 : 4;
    const uintptr_t bits = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v) |
                           reinterpret_cast<uintptr_t>(a->out) | (uintptr_t)((a->q_stride | a->k_stride | a->v_stride) * es);
    if (bits % 16 != 0) return TS_ERR_INVALID_ARG;
    {
        const uint64_t n = (uint64_t)a->tokens, qb = (uint64_t)a->hq * a->head_dim * es, kb = (uint64_t)a->hkv * a->head_dim * es;
        const Extent out(a->out, qb * n);
        if (overlap(out, Extent(a->q, qb, a->q_stride * es, n)) || overlap(out, Extent(a->k, kb, a->k_stride * es, n)) ||
            overlap(out, Extent(a->v, kb, a->v_stride * es, n)) || overlap(out, Extent(a->cu_seqlens, 4 * ((uint64_t)a->batch + 1))))
            return TS_ERR_INVALID_ARG;
    }
    const DeviceScope scope(a->device);
    if (!scope.ok) return TS_ERR_CUDA;
    PromptParams p;
    p.q = a->q; p.k = a->k; p.v = a->v; p.q_stride = a->q_stride; p.k_stride = a->k_stride; p.v_stride = a->v_stride;
    p.cu = a->cu_seqlens; p.out = a->out;
    p.tokens = a->tokens; p.batch = a->batch; p.hq = a->hq; p.hkv = a->hkv; p.group = a->hq / a->hkv;
    p.sm_scale = a->sm_scale; p.logit_cap = a->logit_cap; p.status = a->status;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(a->stream);
    cudaError_t e;
    const int sms = sms_of(a->device);
    if (sms <= 0) return TS_ERR_CUDA;
    const bool cap = a->logit_cap > 0.f;
    if (a->dtype == TS_DTYPE_F32) e = a->head_dim == 128 ? launch_prompt_plain<128>(p, s) : launch_prompt_plain<64>(p, s);
    else if (a->head_dim == 128) e = cap ? launch_prompt_tc<128, true>(p, sms, s) : launch_prompt_tc<128, false>(p, sms, s);
    else e = cap ? launch_prompt_tc<64, true>(p, sms, s) : launch_prompt_tc<64, false>(p, sms, s);
    return e == cudaSuccess ? TS_OK : TS_ERR_CUDA;
}
