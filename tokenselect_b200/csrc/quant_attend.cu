// ts_quant_attend: decode attention of a ragged batch over pool rows held in 4 bits.
//
//   o = sum_j softmax_j(cap(scale * R(n-1) q . R(j) k_j)) v_j,   R(j): rotation by position j
//
// The rows of all requests form one sequence of units of sixteen rows (no unit spans two requests).  CTA c of G owns the
// units [U c / G, U (c+1) / G), whatever the lengths; it keeps a running maximum and sum per head and leaves one partial
// result per request it meets, in slot c + request (unique, because both grow along the sequence).  A second kernel joins
// them.  Every kernel derives the pieces from the lengths alone: nothing is planned on the host, which does not know them.
#include "quant.cuh"
#include "rope.cuh"

namespace ts {
namespace {

constexpr int kQaMaxBatch = 1024;
constexpr int kUnit = 16;                                      // rows
constexpr float kLog2e = 1.4426950408889634f;

struct QuantAttendParams {
    const void* q;
    const unsigned char* pool;
    long long pool_rows;
    const int* rtt;
    long long rtt_stride, max_ctx;
    const int* req_pool_indices;
    const int* seq_lens;
    void* out;
    float* part_o;                                             // [slots][hq][d] unnormalised
    float2* part_ml;                                           // [slots][hq] (maximum in base-2 units, sum)
    int batch, hq, hkv, group, max_reqs, pieces;
    float sm_scale, logit_cap, v_scale;                        // sm_scale includes the pool's scale of K
    int* status;
    TurnFreqs freqs;
};

// Length of request b, 0 where the call's numbers make no sense.
__device__ __forceinline__ int checked_length(const QuantAttendParams& p, int b) {
    const int n = p.seq_lens[b], req = p.req_pool_indices[b];
    if (n < 0 || n > p.max_ctx || req < 0 || req >= p.max_reqs) { report(p.status, TS_ERR_BAD_LENGTH); return 0; }
    return n;
}

// start[b]: first unit of request b; start[batch]: their number.  All threads call; ends with a barrier.
__device__ __forceinline__ void count_units(const QuantAttendParams& p, int* start) {
    for (int b = threadIdx.x; b < p.batch; b += blockDim.x) start[b + 1] = (checked_length(p, b) + kUnit - 1) / kUnit;
    if (threadIdx.x == 0) start[0] = 0;
    __syncthreads();
    if (threadIdx.x < 32 && p.batch > 1) {
        int carry = 0;
        for (int base = 0; base < p.batch; base += 32) {
            const int b = base + threadIdx.x;
            int v = b < p.batch ? start[b + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, v, o);
                if ((int)threadIdx.x >= o) v += t;
            }
            v += carry;
            __syncwarp();
            if (b < p.batch) start[b + 1] = v;
            carry = __shfl_sync(0xffffffffu, v, 31);
        }
    }
    __syncthreads();
}
// Pieces in use: no piece is empty, so every slot between a request's first and last one is written.
__device__ __forceinline__ int used_pieces(int units, int pieces) { return min(units, pieces); }
__device__ __forceinline__ int piece_start(int units, int piece, int pieces) { return (int)((long long)units * piece / pieces); }
// The piece that owns unit u: the last one that starts at or before it.
__device__ __forceinline__ int piece_of(int u, int units, int pieces) { return (int)(((long long)(u + 1) * pieces - 1) / units); }
// The request that holds unit u (start[] ascending, start[batch] > u).
__device__ __forceinline__ int request_of(const int* start, int batch, int u) {
    int lo = 0, hi = batch;                                    // start[lo] <= u < start[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= u) lo = mid; else hi = mid;
    }
    return lo;
}

// ------------------------------------------------------------------------------------------------
// CUDA cores: fp32
// ------------------------------------------------------------------------------------------------
// A warp takes one KV head and up to four of its query heads, eight rows at a time; lane l holds elements
// [P l, P l + P) of both halves of a row, both members of each rotation pair.  The angles of a unit's rows are evaluated
// once per CTA and shared by its eight warps.
constexpr int kQpThreads = 256;
constexpr int kQpHeads = 4;                                    // query heads per warp
constexpr int kQpRows = 8;                                     // rows per step of a warp

template <typename T, int D>
__global__ void __launch_bounds__(kQpThreads) quant_attend_plain_kernel(const __grid_constant__ QuantAttendParams p) {
    using Row = QuantRow<D>;
    constexpr int P = D / 64, HALF = D / 2;
    __shared__ int start[kQaMaxBatch + 1];
    __shared__ float2 sm_cs[kUnit][HALF];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    wait_for_predecessor();
    count_units(p, start);
    const int units = start[p.batch];
    const int pieces = used_pieces(units, p.pieces);
    if ((int)blockIdx.x >= pieces) return;
    const int u_end = piece_start(units, blockIdx.x + 1, pieces);
    int u = piece_start(units, blockIdx.x, pieces);
    const int nsub = (p.group + kQpHeads - 1) / kQpHeads;
    const int mine = blockIdx.y * (kQpThreads / 32) + warp;
    const bool busy = mine < p.hkv * nsub;
    const int kv = busy ? mine / nsub : 0, g0 = busy ? (mine - kv * nsub) * kQpHeads : 0;
    const int ng = min(kQpHeads, p.group - g0), h0 = kv * p.group + g0;
    while (u < u_end) {
        const int b = request_of(start, p.batch, u);
        const int n = p.seq_lens[b];
        const int last = min(u_end, start[b + 1]);             // this CTA's units of the request end here
        const int* table = p.rtt + (long long)p.req_pool_indices[b] * p.rtt_stride;
        float q1[kQpHeads][P], q2[kQpHeads][P];
        float m = -INFINITY, l = 0.f, o1[kQpHeads][P], o2[kQpHeads][P];
#pragma unroll
        for (int e = 0; e < P; ++e) {
            const float2 cs = cos_sin(n - 1, p.freqs.f[P * lane + e]);
#pragma unroll
            for (int g = 0; g < kQpHeads; ++g) {
                const T* qh = reinterpret_cast<const T*>(p.q) + ((long long)b * p.hq + h0 + min(g, ng - 1)) * D + P * lane + e;
                const float x = to_f32<T>(qh[0]), y = to_f32<T>(qh[HALF]);
                q1[g][e] = x * cs.x - y * cs.y;
                q2[g][e] = y * cs.x + x * cs.y;
                o1[g][e] = 0.f;
                o2[g][e] = 0.f;
            }
        }
        for (; u < last; ++u) {
            const int row0 = (u - start[b]) * kUnit, cnt = min(kUnit, n - row0);
            __syncthreads();                                   // the unit before has been read
            for (int i = threadIdx.x; i < cnt * HALF; i += kQpThreads) sm_cs[i / HALF][i % HALF] = cos_sin(row0 + i / HALF, p.freqs.f[i % HALF]);
            __syncthreads();
            if (!busy) continue;
            for (int r0 = 0; r0 < cnt; r0 += kQpRows) {
                int my_row = -1;
                if (lane < kQpRows && r0 + lane < cnt) {
                    my_row = table[row0 + r0 + lane];
                    if (my_row < 0 || my_row >= p.pool_rows) { report(p.status, TS_ERR_BAD_SLOT); my_row = -1; }
                }
                float s[kQpRows * kQpHeads], v1[kQpRows][P], v2[kQpRows][P];
#pragma unroll
                for (int r = 0; r < kQpRows; ++r) {
                    const int row = __shfl_sync(0xffffffffu, my_row, r);
                    float k1[P], k2[P];
#pragma unroll
                    for (int e = 0; e < P; ++e) { k1[e] = 0.f; k2[e] = 0.f; v1[r][e] = 0.f; v2[r][e] = 0.f; }
                    if (row >= 0) {                            // warp-uniform
                        const unsigned char* at = p.pool + ((long long)row * p.hkv + kv) * Row::kBytes;
                        auto element = [&](int codes, int scales, int d) {
                            return e2m1_to_f32(at[codes + d / 2] >> (4 * (d & 1))) * e4m3_to_f32(at[scales + d / kQuantBlock]);
                        };
#pragma unroll
                        for (int e = 0; e < P; ++e) {
                            k1[e] = element(0, Row::kKScales, P * lane + e);
                            k2[e] = element(0, Row::kKScales, HALF + P * lane + e);
                            v1[r][e] = element(Row::kV, Row::kVScales, P * lane + e);
                            v2[r][e] = element(Row::kV, Row::kVScales, HALF + P * lane + e);
                        }
                    }
                    float acc[kQpHeads] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int e = 0; e < P; ++e) {
                        const float2 cs = sm_cs[min(r0 + r, cnt - 1)][P * lane + e];
                        const float y1 = k1[e] * cs.x - k2[e] * cs.y, y2 = k2[e] * cs.x + k1[e] * cs.y;
#pragma unroll
                        for (int g = 0; g < kQpHeads; ++g) acc[g] += q1[g][e] * y1 + q2[g][e] * y2;
                    }
#pragma unroll
                    for (int g = 0; g < kQpHeads; ++g) s[r * kQpHeads + g] = acc[g];
                }
                // lane r*4 + g ends up with the whole sum of (row r, head g)
#pragma unroll
                for (int off = 16; off >= 1; off >>= 1) {
                    const bool up = (lane & off) != 0;
#pragma unroll
                    for (int i = 0; i < off; ++i) {
                        const float keep = up ? s[i + off] : s[i], send = up ? s[i] : s[i + off];
                        s[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
                    }
                }
                float x = s[0] * p.sm_scale;
                if (p.logit_cap > 0.f) x = p.logit_cap * tanhf(x / p.logit_cap);
                x = (r0 + (lane >> 2) < cnt) ? x * kLog2e : -INFINITY;
                float mn = fmaxf(m, x);
#pragma unroll
                for (int off = 4; off <= 16; off <<= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, off));
                const float base = mn == -INFINITY ? 0.f : mn;  // every logit so far -infinity
                const float pe = exp2f(x - base), sc = exp2f(m - base);
                float sum = pe;
#pragma unroll
                for (int off = 4; off <= 16; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                l = l * sc + sum;
                m = mn;
#pragma unroll
                for (int g = 0; g < kQpHeads; ++g) {
                    const float scg = __shfl_sync(0xffffffffu, sc, g);
#pragma unroll
                    for (int e = 0; e < P; ++e) { o1[g][e] *= scg; o2[g][e] *= scg; }
                }
#pragma unroll
                for (int r = 0; r < kQpRows; ++r) {
                    if (r0 + r >= cnt) break;                  // warp-uniform
#pragma unroll
                    for (int g = 0; g < kQpHeads; ++g) {
                        const float pg = __shfl_sync(0xffffffffu, pe, r * kQpHeads + g);
#pragma unroll
                        for (int e = 0; e < P; ++e) { o1[g][e] += pg * v1[r][e]; o2[g][e] += pg * v2[r][e]; }
                    }
                }
            }
        }
        if (busy) {
            const long long slot = blockIdx.x + b;
#pragma unroll
            for (int g = 0; g < kQpHeads; ++g)
                if (g < ng) {
                    float* dst = p.part_o + (slot * p.hq + h0 + g) * D + P * lane;
#pragma unroll
                    for (int e = 0; e < P; ++e) { dst[e] = o1[g][e]; dst[HALF + e] = o2[g][e]; }
                }
            if (lane < ng) p.part_ml[slot * p.hq + h0 + lane] = make_float2(m, l);
        }
    }
}

// ------------------------------------------------------------------------------------------------
// Join the partial results: grid (hq, batch), one warp per partial in flight
// ------------------------------------------------------------------------------------------------
constexpr int kQmThreads = 256;
template <typename T, int D>
__global__ void __launch_bounds__(kQmThreads) quant_merge_kernel(const __grid_constant__ QuantAttendParams p) {
    constexpr int VEC = D / 32, NW = kQmThreads / 32, kAhead = 4;
    __shared__ int start[kQaMaxBatch + 1];
    __shared__ float s_acc[NW][D];
    __shared__ float2 s_ml[NW];
    const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    wait_for_predecessor();
    count_units(p, start);
    const int units = start[p.batch], pieces = used_pieces(units, p.pieces);
    float m = -INFINITY, l = 0.f, acc[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) acc[v] = 0.f;
    if (start[b] < start[b + 1]) {
        const int c_end = piece_of(start[b + 1] - 1, units, pieces);
        for (int c0 = piece_of(start[b], units, pieces) + warp; c0 <= c_end; c0 += NW * kAhead) {
            float x[kAhead][VEC];
            float2 ml[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int c = c0 + NW * i;
                ml[i] = make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int v = 0; v < VEC; ++v) x[i][v] = 0.f;
                if (c <= c_end) {
                    const long long at = (long long)(c + b) * p.hq + h;
                    ml[i] = __ldcg(p.part_ml + at);
                    const float* src = p.part_o + at * D + VEC * lane;
                    if constexpr (VEC == 4) {
                        const float4 t = __ldcg(reinterpret_cast<const float4*>(src));
                        x[i][0] = t.x; x[i][1] = t.y; x[i][2] = t.z; x[i][3] = t.w;
                    } else {
                        const float2 t = __ldcg(reinterpret_cast<const float2*>(src));
                        x[i][0] = t.x; x[i][1] = t.y;
                    }
                }
            }
            float mn = m;
#pragma unroll
            for (int i = 0; i < kAhead; ++i) mn = fmaxf(mn, ml[i].x);
            const float base = mn == -INFINITY ? 0.f : mn;
            const float sc = exp2f(m - base);
            l *= sc;
#pragma unroll
            for (int v = 0; v < VEC; ++v) acc[v] *= sc;
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const float w = exp2f(ml[i].x - base);
                l += ml[i].y * w;
#pragma unroll
                for (int v = 0; v < VEC; ++v) acc[v] += x[i][v] * w;
            }
            m = mn;
        }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) s_acc[warp][VEC * lane + v] = acc[v];
    if (lane == 0) s_ml[warp] = make_float2(m, l);
    __syncthreads();
    for (int e = threadIdx.x; e < D; e += kQmThreads) {
        float mm = -INFINITY, r = 0.f, ll = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) mm = fmaxf(mm, s_ml[w].x);
        const float base = mm == -INFINITY ? 0.f : mm;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float wgt = exp2f(s_ml[w].x - base);
            r += s_acc[w][e] * wgt;
            ll += s_ml[w].y * wgt;
        }
        // an empty request: no row, sum 0, zeros
        reinterpret_cast<T*>(p.out)[((long long)b * p.hq + h) * D + e] = from_f32<T>(start[b] < start[b + 1] ? r / ll * p.v_scale : 0.f);
    }
}

// Pieces the sequence of units is cut into.
int plain_pieces(int sms) { return 4 * sms; }

size_t partial_bytes(int pieces, int batch, int hq, int d) { return (size_t)(pieces + batch) * hq * (d + 2) * sizeof(float); }

template <typename T, int D>
cudaError_t launch_attend_plain(const QuantAttendParams& p, cudaStream_t stream) {
    const int nsub = (p.group + kQpHeads - 1) / kQpHeads, per_cta = kQpThreads / 32;
    cudaError_t e = launch_chained(quant_attend_plain_kernel<T, D>, dim3(p.pieces, (p.hkv * nsub + per_cta - 1) / per_cta), dim3(kQpThreads), 0, stream, p);
    if (e != cudaSuccess) return e;
    return launch_chained(quant_merge_kernel<T, D>, dim3(p.hq, p.batch), dim3(kQmThreads), 0, stream, p);
}

}  // namespace
}  // namespace ts

extern "C" int ts_quant_attend_workspace(int32_t device, int32_t batch, int32_t hq, int32_t head_dim, size_t* bytes) {
    using namespace ts;
    if (!bytes || batch < 0 || batch > kQaMaxBatch || hq < 1 || hq > 8192) return TS_ERR_INVALID_ARG;
    if (head_dim != 64 && head_dim != 128) return TS_ERR_UNSUPPORTED;
    const int sms = sms_of(device);
    if (sms <= 0) return TS_ERR_CUDA;
    *bytes = partial_bytes(plain_pieces(sms), batch, hq, head_dim);
    return TS_OK;
}

extern "C" int ts_quant_attend(const ts_quant_attend_args* a) {
    using namespace ts;
    if (!a || a->struct_size != sizeof(ts_quant_attend_args)) return TS_ERR_INVALID_ARG;
    if (a->dtype != TS_DTYPE_BF16 && a->dtype != TS_DTYPE_F32) return TS_ERR_UNSUPPORTED;
    if (a->head_dim != 64 && a->head_dim != 128) return TS_ERR_UNSUPPORTED;
    if (a->batch < 0 || a->batch > kQaMaxBatch || a->hq < 1 || a->hkv < 1 || a->hkv > 1024 || a->hq % a->hkv != 0) return TS_ERR_INVALID_ARG;
    if (a->hq / a->hkv > 8) return TS_ERR_UNSUPPORTED;
    if (!(a->rope_base > 0.0) || !(a->rope_scale > 0.0) || !power_of_two(a->k_scale) || !power_of_two(a->v_scale)) return TS_ERR_INVALID_ARG;
    if (a->max_reqs < 1 || a->max_ctx < 0 || a->req_to_token_stride < 0 || a->pool_rows < 1) return TS_ERR_INVALID_ARG;
    if (a->max_ctx > (1ll << 31) - kUnit || (a->max_ctx + kUnit - 1) / kUnit * a->batch >= (1ll << 31)) return TS_ERR_INVALID_ARG;   // units are counted in 32 bits
    if (!(a->sm_scale > 0.f) || !isfinite(a->sm_scale)) return TS_ERR_INVALID_ARG;
    if (a->batch == 0) return TS_OK;
    if (!a->q || !a->pool || !a->req_to_token || !a->req_pool_indices || !a->seq_lens || !a->out || !a->workspace) return TS_ERR_INVALID_ARG;
    if (reinterpret_cast<uintptr_t>(a->pool) % 16 != 0 || reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0) return TS_ERR_INVALID_ARG;
    const int sms = sms_of(a->device);
    if (sms <= 0) return TS_ERR_CUDA;
    const int pieces = plain_pieces(sms);
    if (a->workspace_bytes < partial_bytes(pieces, a->batch, a->hq, a->head_dim)) return TS_ERR_CAPACITY;
    const DeviceScope scope(a->device);
    if (!scope.ok) return TS_ERR_CUDA;
    QuantAttendParams p;
    p.q = a->q; p.pool = static_cast<const unsigned char*>(a->pool); p.pool_rows = a->pool_rows;
    p.rtt = a->req_to_token; p.rtt_stride = a->req_to_token_stride; p.max_ctx = a->max_ctx;
    p.req_pool_indices = a->req_pool_indices; p.seq_lens = a->seq_lens; p.out = a->out;
    p.part_o = static_cast<float*>(a->workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + (size_t)(pieces + a->batch) * a->hq * a->head_dim);
    p.batch = a->batch; p.hq = a->hq; p.hkv = a->hkv; p.group = a->hq / a->hkv; p.max_reqs = a->max_reqs; p.pieces = pieces;
    p.sm_scale = a->sm_scale * a->k_scale; p.logit_cap = a->logit_cap; p.v_scale = a->v_scale;
    p.status = a->status;
    p.freqs = turn_freqs(a->rope_base, a->rope_scale, a->head_dim);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(a->stream);
    cudaError_t e;
    if (a->dtype == TS_DTYPE_BF16) e = a->head_dim == 128 ? launch_attend_plain<__nv_bfloat16, 128>(p, s) : launch_attend_plain<__nv_bfloat16, 64>(p, s);
    else e = a->head_dim == 128 ? launch_attend_plain<float, 128>(p, s) : launch_attend_plain<float, 64>(p, s);
    return e == cudaSuccess ? TS_OK : TS_ERR_CUDA;
}
