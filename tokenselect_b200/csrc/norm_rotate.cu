// ts_norm_rotate: RMS norm of every query and key head and the rotation of both in one pass.
//
//   y = x * rsqrt(mean(x^2) + eps) * w,   (y_i, y_{i+D/2}) -> (y_i cos - y_{i+D/2} sin, y_{i+D/2} cos + y_i sin)
//
// What bounds it: HBM (a row is read once, written once, a key row twice) and, for a few tokens, the launch.  Eight lanes
// hold the rows of two (D = 64: four) neighbouring heads of a token: lane l the elements [P l, P l + P) of both halves of each
// (P = D/16), that is both members of its rotation pairs, so the rotation exchanges nothing and the norm three shuffles, and
// the angles (an integer product each, rope.cuh, and in bf16 the fast sine and cosine, whose 2^-20 is far below the output's
// 2^-9) are evaluated once for them.  All rows are requested before the first is used.  In fp32 it runs at 95 % of the copy
// rate; in bf16, with half the bytes for the same arithmetic, the instructions come close, and pairs of numbers halve them.
#include "ptx.cuh"
#include "rope.cuh"

namespace ts {
namespace {

constexpr int kNormThreads = 256;
constexpr int kNormLanes = 8;                                  // lanes a row
// Rows of a group of lanes: 32 elements a thread (8192 tokens, 32 + 8 heads of 128 in bf16: 40.2 us with four rows a thread,
// 36.4 with two, 62 with one; heads of 64: 18.6 with four, 19.9 with two).
template <int D> constexpr int kNormHeads = 256 / D;

struct NormParams {
    const void* q;
    const void* k;
    long long q_stride, k_stride;
    const int* positions;
    const void* q_weight;
    const void* k_weight;
    void* q_out;
    void* k_out;
    void* k_plain;
    int hq, hkv;
    unsigned groups_q, per_token;                              // groups of kNormHeads heads: of the queries, of a token
    unsigned long long groups;
    float eps;
    TurnFreqs freqs;
};

// P consecutive elements; WIDE: every row and every pointer is aligned to them.
template <typename T, int P, bool WIDE>
__device__ __forceinline__ void load_row(const T* src, float (&x)[P]) {
    if constexpr (WIDE) {
        constexpr int kBytes = P * (int)sizeof(T);
        constexpr int kStep = kBytes < 16 ? kBytes : 16, kPer = kStep / (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < kBytes / kStep; ++i) {
            alignas(16) T raw[kPer];
            if constexpr (kStep == 16) *reinterpret_cast<uint4*>(raw) = *reinterpret_cast<const uint4*>(src + i * kPer);
            else *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(src + i * kPer);
#pragma unroll
            for (int e = 0; e < kPer; ++e) x[i * kPer + e] = to_f32<T>(raw[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < P; ++e) x[e] = to_f32<T>(src[e]);
    }
}
template <typename T, int P, bool WIDE>
__device__ __forceinline__ void store_row(T* dst, const float (&x)[P]) {
    if constexpr (WIDE) {
        constexpr int kBytes = P * (int)sizeof(T);
        constexpr int kStep = kBytes < 16 ? kBytes : 16, kPer = kStep / (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < kBytes / kStep; ++i) {
            alignas(16) T raw[kPer];
#pragma unroll
            for (int e = 0; e < kPer; ++e) raw[e] = from_f32<T>(x[i * kPer + e]);
            if constexpr (kStep == 16) *reinterpret_cast<uint4*>(dst + i * kPer) = *reinterpret_cast<const uint4*>(raw);
            else *reinterpret_cast<uint2*>(dst + i * kPer) = *reinterpret_cast<const uint2*>(raw);
        }
    } else {
#pragma unroll
        for (int e = 0; e < P; ++e) dst[e] = from_f32<T>(x[e]);
    }
}

template <typename T, int D, bool WIDE>
__global__ void __launch_bounds__(kNormThreads) norm_rotate_kernel(const __grid_constant__ NormParams p) {
    constexpr int P = D / 2 / kNormLanes, R = kNormHeads<D>;
    __shared__ unsigned long long freqs[D / 2];                // (lanes read different ones: the parameters' bank would serve them one by one)
    if (threadIdx.x < D / 2) freqs[threadIdx.x] = p.freqs.f[threadIdx.x];
    __syncthreads();
    const int lane = threadIdx.x % kNormLanes;
    const unsigned long long group = (unsigned long long)blockIdx.x * (kNormThreads / kNormLanes) + threadIdx.x / kNormLanes;
    const bool mine = group < p.groups;                        // the others keep their warp's shuffles company
    const unsigned long long t64 = mine ? group / p.per_token : 0;
    const long long t = (long long)t64;
    const unsigned part = mine ? (unsigned)(group - t64 * p.per_token) : 0u;
    const bool is_q = part < p.groups_q;
    const int h0 = (int)(is_q ? part : part - p.groups_q) * R, count = min(R, (is_q ? p.hq : p.hkv) - h0);
    const T* src = (is_q ? reinterpret_cast<const T*>(p.q) + t * p.q_stride : reinterpret_cast<const T*>(p.k) + t * p.k_stride) + h0 * D + P * lane;
    const T* w = reinterpret_cast<const T*>(is_q ? p.q_weight : p.k_weight);
    wait_for_predecessor();
    float lo[R][P], hi[R][P];
#pragma unroll
    for (int i = 0; i < R; ++i) {                     // behind the last head: that one again
        load_row<T, P, WIDE>(src + min(i, count - 1) * D, lo[i]);
        load_row<T, P, WIDE>(src + min(i, count - 1) * D + D / 2, hi[i]);
    }
    if (p.q_weight != nullptr || p.k_weight != nullptr) {      // uniform: whether any row of the launch is normed
        float a[P], b[P];
        if (w != nullptr) {
            load_row<T, P, WIDE>(w + P * lane, a);
            load_row<T, P, WIDE>(w + D / 2 + P * lane, b);
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            uint64_t squares = 0ull;
#pragma unroll
            for (int e = 0; e < P; e += 2) {
                const uint64_t x = pack_f32x2(lo[i][e], lo[i][e + 1]), y = pack_f32x2(hi[i][e], hi[i][e + 1]);
                squares = fma_f32x2(y, y, fma_f32x2(x, x, squares));
            }
            float sum, odd;
            unpack_f32x2(squares, sum, odd);
            sum += odd;
#pragma unroll
            for (int off = 1; off < kNormLanes; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            if (w != nullptr) {
                const float r = rsqrtf(sum * (1.f / D) + p.eps);
                const uint64_t r2 = pack_f32x2(r, r);
#pragma unroll
                for (int e = 0; e < P; e += 2) {
                    unpack_f32x2(mul_f32x2(mul_f32x2(pack_f32x2(lo[i][e], lo[i][e + 1]), r2), pack_f32x2(a[e], a[e + 1])), lo[i][e], lo[i][e + 1]);
                    unpack_f32x2(mul_f32x2(mul_f32x2(pack_f32x2(hi[i][e], hi[i][e + 1]), r2), pack_f32x2(b[e], b[e + 1])), hi[i][e], hi[i][e + 1]);
                }
            }
        }
    }
    if (!mine) return;
    const long long at = (t * (is_q ? p.hq : p.hkv) + h0) * D + P * lane;
    if (!is_q && p.k_plain != nullptr) {
        T* plain = reinterpret_cast<T*>(p.k_plain) + at;
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (i < count) {
                store_row<T, P, WIDE>(plain + i * D, lo[i]);
                store_row<T, P, WIDE>(plain + i * D + D / 2, hi[i]);
            }
    }
    if (p.positions != nullptr) {
        const long long pos = p.positions[t];
#pragma unroll
        for (int e = 0; e < P; e += 2) {
            const unsigned long long f0 = freqs[P * lane + e], f1 = freqs[P * lane + e + 1];
            const float2 cs0 = sizeof(T) == 2 ? cos_sin_fast(pos, f0) : cos_sin(pos, f0), cs1 = sizeof(T) == 2 ? cos_sin_fast(pos, f1) : cos_sin(pos, f1);
            const uint64_t c = pack_f32x2(cs0.x, cs1.x), s = pack_f32x2(cs0.y, cs1.y), minus_s = pack_f32x2(-cs0.y, -cs1.y);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const uint64_t x = pack_f32x2(lo[i][e], lo[i][e + 1]), y = pack_f32x2(hi[i][e], hi[i][e + 1]);
                unpack_f32x2(fma_f32x2(y, minus_s, mul_f32x2(x, c)), lo[i][e], lo[i][e + 1]);
                unpack_f32x2(fma_f32x2(x, s, mul_f32x2(y, c)), hi[i][e], hi[i][e + 1]);
            }
        }
    }
    T* out = reinterpret_cast<T*>(is_q ? p.q_out : p.k_out) + at;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (i < count) {
            store_row<T, P, WIDE>(out + i * D, lo[i]);
            store_row<T, P, WIDE>(out + i * D + D / 2, hi[i]);
        }
}

template <typename T, int D>
cudaError_t launch_norm_rotate(const NormParams& p, cudaStream_t stream) {
    constexpr int kAlign = (D / 16) * (int)sizeof(T) < 16 ? (D / 16) * (int)sizeof(T) : 16;
    const uintptr_t bits = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.q_weight) |
                           reinterpret_cast<uintptr_t>(p.k_weight) | reinterpret_cast<uintptr_t>(p.q_out) | reinterpret_cast<uintptr_t>(p.k_out) |
                           reinterpret_cast<uintptr_t>(p.k_plain) | (uintptr_t)(p.q_stride * sizeof(T)) | (uintptr_t)(p.k_stride * sizeof(T));
    const dim3 grid((unsigned)((p.groups * kNormLanes + kNormThreads - 1) / kNormThreads));
    return bits % kAlign == 0 ? launch_chained(norm_rotate_kernel<T, D, true>, grid, dim3(kNormThreads), 0, stream, p)
                              : launch_chained(norm_rotate_kernel<T, D, false>, grid, dim3(kNormThreads), 0, stream, p);
}

}  // namespace
}  // namespace ts

extern "C" int ts_norm_rotate(const ts_norm_rotate_args* a) {
    using namespace ts;
    if (!a || a->struct_size != sizeof(ts_norm_rotate_args)) return TS_ERR_INVALID_ARG;
    if (a->dtype != TS_DTYPE_BF16 && a->dtype != TS_DTYPE_F32) return TS_ERR_UNSUPPORTED;
    if (a->head_dim != 64 && a->head_dim != 128) return TS_ERR_UNSUPPORTED;
    if (a->tokens < 0 || a->hq < 1 || a->hkv < 1 || a->hq > 1024 || a->hkv > 1024) return TS_ERR_INVALID_ARG;
    if (a->q_stride < (int64_t)a->hq * a->head_dim || a->k_stride < (int64_t)a->hkv * a->head_dim) return TS_ERR_INVALID_ARG;
    if (!(a->eps >= 0.f)) return TS_ERR_INVALID_ARG;
    if (a->positions && (!positive(a->rope_base) || !positive(a->rope_scale))) return TS_ERR_INVALID_ARG;
    if (a->tokens == 0) return TS_OK;
    if (!a->q || !a->k || !a->q_out || !a->k_out) return TS_ERR_INVALID_ARG;
    {
        // A token's rows are read by others than those that write them, so an output is an input's whole place or no part of it.
        const uint64_t es = a->dtype == TS_DTYPE_BF16 ? 2 : 4, n = (uint64_t)a->tokens, qb = (uint64_t)a->hq * a->head_dim * es, kb = (uint64_t)a->hkv * a->head_dim * es;
        const Extent q(a->q, qb, a->q_stride * es, n), k(a->k, kb, a->k_stride * es, n);
        const Extent small[3] = {{a->positions, 4 * n}, {a->q_weight, a->head_dim * es}, {a->k_weight, a->head_dim * es}};
        const Extent outs[3] = {{a->q_out, qb * n}, {a->k_out, kb * n}, {a->k_plain, kb * n}};
        for (int i = 0; i < 3; ++i) {
            const Extent &own = i == 0 ? q : k, &other = i == 0 ? k : q;
            const bool in_place = outs[i].at == own.at && own.n == 1;
            if ((!in_place && overlap(outs[i], own)) || overlap(outs[i], other) || overlap(outs[i], outs[(i + 1) % 3])) return TS_ERR_INVALID_ARG;
            for (const Extent& s : small)
                if (overlap(outs[i], s)) return TS_ERR_INVALID_ARG;
        }
    }
    const DeviceScope scope(a->device);
    if (!scope.ok) return TS_ERR_CUDA;
    NormParams p;
    p.q = a->q; p.k = a->k; p.q_stride = a->q_stride; p.k_stride = a->k_stride;
    p.positions = a->positions; p.q_weight = a->q_weight; p.k_weight = a->k_weight;
    p.q_out = a->q_out; p.k_out = a->k_out; p.k_plain = a->k_plain;
    p.hq = a->hq; p.hkv = a->hkv; p.eps = a->eps;
    const int heads = a->head_dim == 128 ? kNormHeads<128> : kNormHeads<64>;
    p.groups_q = (a->hq + heads - 1) / heads;
    p.per_token = p.groups_q + (a->hkv + heads - 1) / heads;
    p.groups = (unsigned long long)a->tokens * p.per_token;
    if (p.groups > ((1ull << 31) - 1) * (kNormThreads / kNormLanes)) return TS_ERR_CAPACITY;      // blocks of one launch
    if (a->positions) p.freqs = turn_freqs(a->rope_base, a->rope_scale, a->head_dim);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(a->stream);
    cudaError_t e;
    if (a->dtype == TS_DTYPE_BF16) e = a->head_dim == 128 ? launch_norm_rotate<__nv_bfloat16, 128>(p, s) : launch_norm_rotate<__nv_bfloat16, 64>(p, s);
    else e = a->head_dim == 128 ? launch_norm_rotate<float, 128>(p, s) : launch_norm_rotate<float, 64>(p, s);
    return e == cudaSuccess ? TS_OK : TS_ERR_CUDA;
}
