// ts_prompt_attend: causal attention of packed prompts, grouped heads.
//
//   o_i = sum_{j <= i, same sequence} softmax_j(cap(scale q_i . k_j)) v_j
#include "ptx.cuh"
#include "rope.cuh"

namespace ts {
namespace {

constexpr int kPromptMaxBatch = 4096;

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

// Sequence b: first token and length.  Bounds that make no sense are reported and cut.
__device__ __forceinline__ int2 sequence_of(const PromptParams& p, int b) {
    const int a = p.cu[b], e = p.cu[b + 1];
    const int first = min(max(a, 0), p.tokens), end = min(max(e, first), p.tokens);
    if (a != first || e != end) report(p.status, TS_ERR_BAD_LENGTH);
    return make_int2(first, end - first);
}

// ------------------------------------------------------------------------------------------------
// CUDA cores
// ------------------------------------------------------------------------------------------------
// A CTA takes 64 query tokens of one head, key tiles of 64 pass through shared memory in fp32.  Thread (ty, tx) holds
// rows 4 ty .. 4 ty + 3 and, of S, columns tx + 16 j; of O, elements 4 tx + 64 j.
constexpr int kPpThreads = 256, kPpTile = 64;

template <int D>
struct PromptPlainSmem {
    float q[kPpTile][D + 4];
    float kv[kPpTile][D + 4];                                  // the tile's keys, then its values
    float p[kPpTile][kPpTile + 4];
    int tiles[kPpThreads];
    int found[3];                                              // first token, length, tile
};

// The tile'th tile of the packed sequences, the last tile of a sequence first (it has the most keys).  Returns false
// behind the last one.  All threads call.
template <int D>
__device__ __forceinline__ bool find_tile(const PromptParams& p, int tile, PromptPlainSmem<D>& sm) {
    const int per = (p.batch + kPpThreads - 1) / kPpThreads, b0 = threadIdx.x * per, b1 = min(b0 + per, p.batch);
    int sum = 0;
    for (int b = b0; b < b1; ++b) sum += (sequence_of(p, b).y + kPpTile - 1) / kPpTile;
    sm.tiles[threadIdx.x] = sum;
    if (threadIdx.x == 0) sm.found[1] = 0;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < threadIdx.x; ++i) before += sm.tiles[i];
    if (tile >= before && tile < before + sum) {
        for (int b = b0; b < b1; ++b) {
            const int2 s = sequence_of(p, b);
            const int n = (s.y + kPpTile - 1) / kPpTile;
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

// Rows [row0, row0 + 64) of a [tokens, heads, D] tensor into shared memory; zeros from row `end` on.
template <typename T, int D>
__device__ __forceinline__ void stage_rows(float (*dst)[D + 4], const T* src, long long stride, int row0, int end) {
    constexpr int kPer = 16 / (int)sizeof(T), kVecs = D / kPer;
    for (int i = threadIdx.x; i < kPpTile * kVecs; i += kPpThreads) {
        const int r = i / kVecs, c = i % kVecs * kPer;
        alignas(16) T raw[kPer];
        *reinterpret_cast<uint4*>(raw) = row0 + r < end ? *reinterpret_cast<const uint4*>(src + (row0 + r) * stride + c) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int e = 0; e < kPer; ++e) dst[r][c + e] = to_f32<T>(raw[e]);
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kPpThreads) prompt_plain_kernel(const PromptParams p) {
    extern __shared__ __align__(16) unsigned char dyn[];
    PromptPlainSmem<D>& sm = *reinterpret_cast<PromptPlainSmem<D>*>(dyn);
    constexpr int OJ = D / 64;
    const int h = blockIdx.y, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    wait_for_predecessor();
    if (!find_tile<D>(p, blockIdx.x, sm)) return;
    const int first = sm.found[0], len = sm.found[1], row0 = sm.found[2] * kPpTile;      // in the sequence
    const T* q = reinterpret_cast<const T*>(p.q) + (long long)first * p.q_stride + (long long)h * D;
    const T* k = reinterpret_cast<const T*>(p.k) + (long long)first * p.k_stride + (long long)(h / p.group) * D;
    const T* v = reinterpret_cast<const T*>(p.v) + (long long)first * p.v_stride + (long long)(h / p.group) * D;
    stage_rows<T, D>(sm.q, q, p.q_stride, row0, len);
    float m[4], l[4], o[4][OJ][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int j = 0; j < OJ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][j][e] = 0.f;
    }
    for (int key0 = 0; key0 <= row0; key0 += kPpTile) {
        __syncthreads();
        stage_rows<T, D>(sm.kv, k, p.k_stride, key0, len);
        __syncthreads();
        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
        for (int d = 0; d < D; d += 4) {
            float4 a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(&sm.q[4 * ty + i][d]);
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const float4*>(&sm.kv[tx + 16 * j][d]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[i][j] += a[i].x * b[j].x + a[i].y * b[j].y + a[i].z * b[j].z + a[i].w * b[j].w;
        }
        const bool diagonal = key0 == row0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float x = s[i][j] * p.sm_scale;
                if (p.logit_cap > 0.f) x = p.logit_cap * tanhf(x / p.logit_cap);
                s[i][j] = diagonal && tx + 16 * j > 4 * ty + i ? -INFINITY : x * 1.4426950408889634f;
                mx = fmaxf(mx, s[i][j]);
            }
#pragma unroll
            for (int off = 1; off < 16; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            const float mn = fmaxf(m[i], mx), base = mn == -INFINITY ? 0.f : mn, corr = exp2f(m[i] - base);
            m[i] = mn;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float pe = exp2f(s[i][j] - base);
                sum += pe;
                sm.p[4 * ty + i][tx + 16 * j] = pe;
            }
            l[i] = l[i] * corr + sum;                          // this thread's columns; joined at the end
#pragma unroll
            for (int j = 0; j < OJ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][j][e] *= corr;
        }
        __syncthreads();
        stage_rows<T, D>(sm.kv, v, p.v_stride, key0, len);
        __syncthreads();
        // On the diagonal a masked weight is 0, but 0 times a later token's infinity is not: those products are left out.
        const int keys = diagonal ? min(kPpTile, len - key0) : kPpTile;
        for (int c = 0; c < keys; ++c) {
            float4 b[OJ];
#pragma unroll
            for (int j = 0; j < OJ; ++j) b[j] = *reinterpret_cast<const float4*>(&sm.kv[c][4 * tx + 64 * j]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = sm.p[4 * ty + i][c];
                if (!diagonal || c <= 4 * ty + i) {
#pragma unroll
                    for (int j = 0; j < OJ; ++j) {
                        o[i][j][0] += a * b[j].x; o[i][j][1] += a * b[j].y; o[i][j][2] += a * b[j].z; o[i][j][3] += a * b[j].w;
                    }
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float sum = l[i];
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        const int row = row0 + 4 * ty + i;
        if (row >= len) continue;
        T* out = reinterpret_cast<T*>(p.out) + ((long long)(first + row) * p.hq + h) * D;
#pragma unroll
        for (int j = 0; j < OJ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) out[4 * tx + 64 * j + e] = from_f32<T>(o[i][j][e] / sum);
    }
}

template <typename T, int D>
cudaError_t launch_prompt_plain(const PromptParams& p, cudaStream_t stream) {
    static SmemConfig configured = {};
    constexpr size_t kSmem = sizeof(PromptPlainSmem<D>);
    const cudaError_t e = ensure_dynamic_smem(prompt_plain_kernel<T, D>, kSmem, configured);
    if (e != cudaSuccess) return e;
    return launch_chained(prompt_plain_kernel<T, D>, dim3(p.tokens / kPpTile + p.batch, p.hq), dim3(kPpThreads), kSmem, stream, p);
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
    if (!(a->sm_scale > 0.f) || !isfinite(a->sm_scale)) return TS_ERR_INVALID_ARG;
    if (a->tokens == 0 || a->batch == 0) return TS_OK;
    if (!a->q || !a->k || !a->v || !a->cu_seqlens || !a->out) return TS_ERR_INVALID_ARG;
    const int es = a->dtype == TS_DTYPE_BF16 ? 2 : 4;
    const uintptr_t bits = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v) |
                           reinterpret_cast<uintptr_t>(a->out) | (uintptr_t)((a->q_stride | a->k_stride | a->v_stride) * es);
    if (bits % 16 != 0) return TS_ERR_INVALID_ARG;
    const DeviceScope scope(a->device);
    if (!scope.ok) return TS_ERR_CUDA;
    PromptParams p;
    p.q = a->q; p.k = a->k; p.v = a->v; p.q_stride = a->q_stride; p.k_stride = a->k_stride; p.v_stride = a->v_stride;
    p.cu = a->cu_seqlens; p.out = a->out;
    p.tokens = a->tokens; p.batch = a->batch; p.hq = a->hq; p.hkv = a->hkv; p.group = a->hq / a->hkv;
    p.sm_scale = a->sm_scale; p.logit_cap = a->logit_cap; p.status = a->status;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(a->stream);
    cudaError_t e;
    if (a->dtype == TS_DTYPE_BF16) e = a->head_dim == 128 ? launch_prompt_plain<__nv_bfloat16, 128>(p, s) : launch_prompt_plain<__nv_bfloat16, 64>(p, s);
    else e = a->head_dim == 128 ? launch_prompt_plain<float, 128>(p, s) : launch_prompt_plain<float, 64>(p, s);
    return e == cudaSuccess ? TS_OK : TS_ERR_CUDA;
}
