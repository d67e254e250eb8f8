// ts_quant_attend: decode attention of a ragged batch over pool rows held in 4 bits.
//
//   o = sum_j softmax_j(cap(scale * R(n-1) q . R(j) k_j)) v_j,   R(j): rotation by position j
//
// The rows of all requests form one sequence of units of sixteen rows (no unit spans two requests).  CTA c of G owns the
// units [U c / G, U (c+1) / G), whatever the lengths; it keeps a running maximum and sum per head and leaves one partial
// result per request it meets, in slot c + request (unique, because both grow along the sequence).  A second kernel joins
// them.  Every kernel derives the pieces from the lengths alone: nothing is planned on the host, which does not know them.
#include <limits.h>

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
    int step_units, share;                                     // units that a CTA takes in one step; partial results of a slot
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
// Pieces in use: no piece is empty, so every slot between a request's first and last one is written.  And none is shorter than
// what a CTA's warps take in their first step anyway: fewer partial results then cost nothing.
__device__ __forceinline__ int used_pieces(const QuantAttendParams& p, int units) { return min((units + p.step_units - 1) / p.step_units, p.pieces); }
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
    const int pieces = used_pieces(p, units);
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
// Tensor cores: bf16
// ------------------------------------------------------------------------------------------------
// What bounds it: the instructions that turn 4-bit codes into operands.  A unit of sixteen rows of one head is 2304 bytes, at
// the copy rate 395 cycles of a scheduler; its 128 conversions, scalings and turns a lane, 16 products and the rest are 506
// instructions, and take about 750 (2.7 TB/s of 6.55: 4 requests of 100000..262144 tokens, 28 heads over 4).  So the layout
// spares instructions.  (On the way, the same case: rows in 16-byte cp.async pieces by the computing warps 175 us, bulk copies by
// one requesting warp 420, by four in turn 166; a partial result per warp instead of per CTA 158; shared memory free of bank
// conflicts 150.)
//
// A warp takes one KV head; its up to eight query heads are the N of m16n8k16 products in fp16.  S^T = K Q^T has sixteen
// keys as M: a key row's codes, read eight bytes at a time, ARE the A fragments of a thread once converted, because a
// product over d does not mind in which order it meets the d's -- thread t of a quad simply owns elements [16 t, 16 t + 16) of
// both halves of the head (both members of its rotation pairs, and two scales in all).  O^T = V^T P^T has sixteen d as M:
// thread g owns the d of one scale block, and two keys' codes are interleaved as 4-bit fields (four instructions for sixteen
// elements) so that one conversion gives the pair (key, key + 1) that a fragment register holds.  S^T becomes the B
// fragment of the second product with one movmatrix per eight keys.
//
// Rotation.  R(n-1) q . R(j0 + i) k = (R(n-1-j0) q) . (R(i) k): per macro tile of 128 keys the query is turned in fp32 by its
// exact distance to the tile's first key, and a key only by its place i in the tile, from a table of 128 rows of cosines and
// sines in fp16 that stays in shared memory.  No table grows with the context, and the far angles stay exact.
//
// Rows arrive through rings in shared memory: the warps that take the same units (one per KV head) share one.  Warps of
// their own request the units in turn, all heads of the CTA at once.  With three heads or more that is one bulk copy a row,
// sixteen by one instruction, which holds its warp for a microsecond whatever their number and size (measured, random rows, four
// warps: 6.4 TB/s in rows of 1152 bytes, 4.2 in rows of 576, but 1.1 in rows of 144).  Narrower rows, and rows of D = 64 that
// lie off the copies' 16-byte grid, come in cp.async pieces.  (1.2 million rows of one head: pieces 107 us, bulk 192; 300000
// rows of two: 51 and 64; 800000 rows of four: 187 and 174.)  A row takes 16 bytes modulo 128 in shared memory, and the order in
// which the sixteen keys are given to the sixteen M rows then makes every read of eight-byte fragments free of bank conflicts.
// Eight computing warps with their operands in registers do as well as sixteen with some of them spilled, and better than twelve
// in 152 registers (4 x 200000, 28 heads over 4: 173 and 184 us).
constexpr int kQtWarps = 8;
constexpr int kQtBulkBytes = 400;                              // bulk copies for rows of at least this many
constexpr int kQtLoadRegs = 56;
// Requesting warps, and registers: those they give up are the computing ones'.  Four for bulk copies; eight for rows in pieces, of
// which a warp has few in flight (1.2 million rows of one head: 153 us with four, 106 with eight; bulk rows of eight heads 123 and
// 133, because the computing warps then get 200 registers).
template <int PIECE>
struct QtLaunch {
    static constexpr int kLoaders = PIECE == 0 ? 4 : 8, kThreads = 32 * (kQtWarps + kLoaders);
    static constexpr int kComputeRegs = PIECE == 0 ? 224 : 200;        // 2 * 224 + 56 = 3 * 168; 2 * 200 + 2 * 56 = 4 * 128 a thread
};
constexpr int kQtMacro = 8;                                    // units of a macro tile
// Weights enter the second product in fp16, whose smallest number is 2^-24 and largest below 2^16.  They are taken 2^7 times as
// large as their reference says (in the sum too), so that what a warp loses of many small weights beside a large one is
// at most 2^-32 of it each, and not 2^-25.
constexpr float kQtLift = 7.f;
// Stages of a ring: a step holds two while the two behind it arrive, so fewer than four would wait for themselves.  And never
// fewer than warps that fill it in turn: a warp asks for the stage's release before last with the same parity, and knows that one
// to have happened because it filled a stage that many units ago.
constexpr int kQtMinStages = 4, kQtMaxStages = 8, kQtBytes = 232448;          // (dynamic shared memory)

template <int D>
struct QuantTcSmem {                                           // behind it: the rings
    uint4 turn[kQtMacro * kUnit][D / 8];                       // per key of a macro tile: cosines, sines of the pairs, fp16
    float2 base[kQtWarps][D / 2];                              // per warp: (cos, sin) of the query's distance to the tile
    uint4 q[kQtWarps][D / 32][32];                             // per warp and lane: its pairs of its head's query, bf16
    uint64_t full[kQtWarps][kQtMaxStages], empty[kQtWarps][kQtMaxStages];
    int start[kQaMaxBatch + 1];
    int pad[3];
};
// Bytes between the rows of `heads` heads in shared memory: 16 modulo 128.
template <int D>
__host__ __device__ __forceinline__ int row_pitch(int heads) {
    const int bytes = heads * QuantRow<D>::kBytes;
    return bytes + ((16 - bytes) & 127);
}

template <int D>
__host__ __device__ __forceinline__ int ring_space() { return kQtBytes - (int)sizeof(QuantTcSmem<D>); }
// Warps that share a head's units.
template <int D>
__host__ __device__ __forceinline__ int shares_of(int heads) {
    const int most = ring_space<D>() / (kQtMinStages * kUnit * row_pitch<D>(heads));
    return kQtWarps / heads < most ? kQtWarps / heads : most;
}
template <int D>
constexpr bool rings_fit() {
    for (int heads = 1; heads <= kQtWarps; ++heads) {
        const int bytes = heads * QuantRow<D>::kBytes, pitch = bytes + ((16 - bytes) & 127);
        if (kQtBytes - (int)sizeof(QuantTcSmem<D>) < kQtMinStages * kUnit * pitch) return false;
    }
    return true;
}
static_assert(rings_fit<128>() && rings_fit<64>(), "four stages for one warp of every head count");

// Key of a stage that M row m of a fragment stands for: rows 0..7 the even keys, 8..15 the odd ones, in an order in which
// the four rows of a half-warp's read lie 32 bytes apart modulo 128, for K (rows g) and for V (rows 2t and 2t + 1) alike.
__device__ __forceinline__ int key_of(int m) { return ((m & 4) ? 8 + (((m & 3) * 2) ^ 2) : (m & 3) * 2) + (m >> 3); }

__device__ __forceinline__ __half2 as_half2(uint32_t a) { return *reinterpret_cast<const __half2*>(&a); }
__device__ __forceinline__ uint32_t as_bits(__half2 a) { return *reinterpret_cast<const uint32_t*>(&a); }
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) { return as_bits(__hmul2(as_half2(a), as_half2(b))); }
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) { return as_bits(__hfma2(as_half2(a), as_half2(b), as_half2(c))); }
__device__ __forceinline__ uint32_t fnma2(uint32_t a, uint32_t b, uint32_t c) { return as_bits(__hfma2(__hneg2(as_half2(a)), as_half2(b), as_half2(c))); }
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int BYTES>
__device__ __forceinline__ void copy_piece(uint32_t dst, const unsigned char* src, int bytes) {      // zeros behind `bytes`
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// A thread's eight (D = 64: four) bytes of a row's codes.
template <int D>
__device__ __forceinline__ void load_words(const unsigned char* src, uint32_t (&w)[D / 64]) {
    if constexpr (D == 128) { const uint2 x = *reinterpret_cast<const uint2*>(src); w[0] = x.x; w[1] = x.y; }
    else w[0] = *reinterpret_cast<const uint32_t*>(src);
}

// What a CTA takes of one request: units [u0, u1), dealt out to the warps of a head in macro tiles of `per` units.
struct Segment {
    int b, n, first, u1, per;                                  // request, its length and first unit
    const int* table;
    __device__ __forceinline__ int units_of(int u0, int w, int share) const {      // of share w
        const int round = share * per, whole = (u1 - u0) / round, rest = u1 - u0 - whole * round;
        return whole * per + min(per, max(0, rest - w * per));
    }
};
__device__ __forceinline__ Segment segment_at(const QuantAttendParams& p, const int* start, int u0, int u_end, int share) {
    Segment s;
    s.b = request_of(start, p.batch, u0);
    s.n = p.seq_lens[s.b];
    s.first = start[s.b];
    s.u1 = min(u_end, start[s.b + 1]);
    s.table = p.rtt + (long long)p.req_pool_indices[s.b] * p.rtt_stride;
    const int units = s.u1 - u0, rounds = (units + share * kQtMacro - 1) / (share * kQtMacro);
    s.per = (units + share * rounds - 1) / (share * rounds);
    return s;
}

// PIECE: 0, rows by bulk copies; 16 or 8, by pieces of that many bytes.
template <int D, bool CAP, int PIECE>
__global__ void __launch_bounds__(QtLaunch<PIECE>::kThreads, 1) quant_attend_tc_kernel(const __grid_constant__ QuantAttendParams p) {
    using Row = QuantRow<D>;
    using Launch = QtLaunch<PIECE>;
    constexpr int HALF = D / 2, NW = D / 64, MT = D / 16;      // words a half, M tiles of O
    extern __shared__ __align__(16) unsigned char dyn[];
    QuantTcSmem<D>& sm = *reinterpret_cast<QuantTcSmem<D>*>(dyn);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

    // The turns of a macro tile's keys.  16-byte unit 4 c + t (c: cosines' then sines' words) holds what thread t reads; the units
    // of every other pair of keys are exchanged by fours so that a read of two keys by eight lanes meets eight different bank
    // groups (key_of).
    {
        const int pair = threadIdx.x % HALF, owner = pair / (D / 8), r = pair % (D / 8);
        const unsigned long long f = p.freqs.f[pair];
        for (int i = threadIdx.x / HALF; i < kQtMacro * kUnit; i += Launch::kThreads / HALF) {
            const float2 cs = cos_sin_fast(i, f);
            __half* row = reinterpret_cast<__half*>(sm.turn[i]);
            const int swap = (i & 2) * 2;
            // D = 128: a thread's 16 pairs are two units of cosines and two of sines; D = 64: its 8 pairs one of each
            const int uc = ((r >> 3) * 4 + owner) ^ swap, us = ((NW + (r >> 3)) * 4 + owner) ^ swap;
            row[uc * 8 + (r & 7)] = __float2half_rn(cs.x);
            row[us * 8 + (r & 7)] = __float2half_rn(cs.y);
        }
    }
    const int hpc = (p.hkv + gridDim.y - 1) / gridDim.y;       // KV heads of a CTA
    const int head0 = blockIdx.y * hpc, heads = min(hpc, p.hkv - head0);
    const int pitch = row_pitch<D>(hpc), stage_bytes = kUnit * pitch;
    const int share = p.share;                                 // warps of a head
    unsigned char* rings = dyn + sizeof(QuantTcSmem<D>);
    const int stages = min(kQtMaxStages, ring_space<D>() / (share * stage_bytes));
    const bool requests = warp >= kQtWarps;
    const int my_head = warp % hpc, kv = head0 + my_head, my_share = warp / hpc;
    const bool busy = !requests && my_share < share && my_head < heads;
    if (threadIdx.x < share * stages) {
        const int r = threadIdx.x / stages, i = threadIdx.x % stages;
        mbar_init(smem_u32(&sm.full[r][i]), PIECE == 0 ? 1 : 32);
        mbar_init(smem_u32(&sm.empty[r][i]), heads);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    wait_for_predecessor();
    count_units(p, sm.start);                                  // ends with a barrier: the table and the barriers are complete too
    const int units = sm.start[p.batch], pieces = used_pieces(p, units);
    if ((int)blockIdx.x >= pieces) return;
    const int u_end = piece_start(units, blockIdx.x + 1, pieces);
    const unsigned char* head_pool = p.pool + (long long)head0 * Row::kBytes;
    const long long row_bytes = (long long)p.hkv * Row::kBytes;
    const int width = heads * Row::kBytes;                     // bytes of a row that this CTA takes
    unsigned char* ring = rings + min(my_share, share - 1) * stages * stage_bytes;
    const uint32_t full = smem_u32(sm.full[min(my_share, share - 1)]), empty = smem_u32(sm.empty[min(my_share, share - 1)]);
    bool dead = false;
    const unsigned long long f0 = p.freqs.f[lane], f1 = D == 128 ? p.freqs.f[(lane + 32) % HALF] : 0ull;

    int u0 = piece_start(units, blockIdx.x, pieces);
    if (requests) {
        // ---------------- requests ----------------
        // (these warps leave their registers to the computing ones)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kQtLoadRegs));
        static_assert(kQtMinStages >= QtLaunch<0>::kLoaders, "stages for the warps of bulk copies");
        const int turns = PIECE == 0 ? Launch::kLoaders : min(Launch::kLoaders, stages), my_turn = warp - kQtWarps;
        if (my_turn >= turns) return;
        int before = 0;                                        // lane w: units of share w in the segments so far
        while (u0 < u_end) {
            const Segment seg = segment_at(p, sm.start, u0, u_end, share);
            const int b = seg.b, n = seg.n, first = seg.first, u1 = seg.u1, per = seg.per;
            const int* table = seg.table;
            auto units_of = [&](int w) { return seg.units_of(u0, w, share); };
            // Lane w keeps the place of share w: unit `at` of its units, counted over all requests, goes into stage at % stages and is
            // requested by warp at % turns of these.  Lanes 16 (w & 1) + r of ahead[w / 2] hold the number of row r of this warp's next
            // unit (or none), read when the one before was requested.
            const int end = before + (lane < share ? units_of(lane) : 0);
            int at = before + (my_turn + turns - before % turns) % turns, ahead[kQtWarps / 2];
            auto unit_of = [&]() { const int k = at - before, m = k / per; return u0 + (m * share + lane) * per + k - m * per; };
            auto read_ahead = [&](int w, int unit) {
                const int r = (unit - first) * kUnit + (lane & 15);
                const bool mine = lane >> 4 == (w & 1), some = unit < u1 && r < n;
#pragma unroll
                for (int i = 0; i < kQtWarps / 2; ++i)
                    if (mine && w >> 1 == i) {
                        if (some) ahead[i] = __ldcg(table + r); else ahead[i] = INT_MIN;
                    }
            };
            {
                const int unit = unit_of();
                for (int w = 0; w < share; ++w) read_ahead(w, __shfl_sync(0xffffffffu, unit, w));
            }
            long long idle_since = clock64();
            while (__any_sync(0xffffffffu, at < end)) {
                const int stage_in = at % stages;
                const bool ready = at < end && (dead || test_phase(smem_u32(&sm.empty[lane % kQtWarps][stage_in]), (at / stages & 1) ^ 1));
                unsigned todo = __ballot_sync(0xffffffffu, ready);
                if (todo == 0) {
                    __nanosleep(100);                          // (leaves the issue slots to the computing warps)
                    if (clock64() - idle_since > kWaitCycles) { report(p.status, TS_ERR_DEVICE_TIMEOUT); dead = true; }
                    dead = __any_sync(0xffffffffu, dead);
                    continue;
                }
                for (; todo != 0; todo &= todo - 1) {
                    const int w = __ffs(todo) - 1, to = __shfl_sync(0xffffffffu, stage_in, w);
                    int pair = ahead[0];
#pragma unroll
                    for (int i = 1; i < kQtWarps / 2; ++i) pair = w >> 1 == i ? ahead[i] : pair;
                    const int r = lane & 15, id = __shfl_sync(0xffffffffu, pair, (w & 1) * 16 + r);
                    unsigned char* dst = rings + (w * stages + to) * stage_bytes;
                    const uint32_t bar = smem_u32(&sm.full[w][to]);
                    const bool bad = id != INT_MIN && (id < 0 || id >= p.pool_rows);
                    if (bad) report(p.status, TS_ERR_BAD_SLOT);
                    const bool some = !bad && id != INT_MIN;
                    const unsigned char* src = head_pool + (some ? id * row_bytes : 0);
                    if constexpr (PIECE == 0) {
                        const unsigned rows = __ballot_sync(0xffffffffu, some) & 0xffffu;
                        if (rows != 0xffffu) {                 // zeros where no row comes
                            for (int i = 0; i < kUnit; ++i)
                                if (!(rows >> i & 1))
                                    for (int j = lane; j < width / 8; j += 32) reinterpret_cast<uint2*>(dst + i * pitch)[j] = make_uint2(0u, 0u);
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // a later copy into the stage comes behind them
                            __syncwarp();
                        }
                        if (lane == 0) mbar_expect_tx(bar, __popc(rows) * width);
                        __syncwarp();
                        if (lane < 16 && some) bulk_g2s(smem_u32(dst + r * pitch), src, width, bar);
                    } else {
                        // two lanes a row, two neighbouring pieces at a time
                        for (int j = (lane >> 4) * PIECE; j < width; j += 2 * PIECE) copy_piece<PIECE>(smem_u32(dst + r * pitch + j), src + (some ? j : 0), some ? PIECE : 0);
                        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
                    }
                    if (lane == w) at += turns;
                    const int unit = unit_of();
                    read_ahead(w, __shfl_sync(0xffffffffu, unit, w));
                }
                idle_since = clock64();
            }
            before = end;
            u0 = u1;
        }
        if (__any_sync(0xffffffffu, dead) && lane < share)     // given up: the copies still have to land (or time out)
            for (int i = max(before - stages, 0); i < before; ++i) {
                bool gone = false;
                wait_phase(smem_u32(&sm.full[lane][i % stages]), i / stages & 1, p.status, gone);
            }
        return;
    }
    // ---------------- products ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Launch::kComputeRegs));
    int stage = 0;                                             // next stage to read
    uint32_t phase = 0;                                        // parity of its barrier
    while (u0 < u_end) {
        const Segment seg = segment_at(p, sm.start, u0, u_end, share);
        const int b = seg.b, n = seg.n, first = seg.first, u1 = seg.u1, per = seg.per;
        const int* table = seg.table;
        const int steps = busy ? seg.units_of(u0, my_share, share) : 0, skip = (share - 1) * per;
        float o[MT][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
        if (steps > 0) {
            // the query of head g, of which a quad's thread turns its own pairs; scaled by a power of two to below 2
            const bool real = g < p.group;
            const __nv_bfloat16* qh = reinterpret_cast<const __nv_bfloat16*>(p.q) + ((long long)b * p.hq + kv * p.group + (real ? g : 0)) * D + t * (D / 8);
            const bool aligned = (reinterpret_cast<uintptr_t>(p.q) & 3) == 0;
            float unit_scale;
            {
                uint32_t x[4 * NW], y[4 * NW], top = 0;
#pragma unroll
                for (int i = 0; i < 4 * NW; ++i) {
                    x[i] = real ? load_bf16_pair(qh + 2 * i, aligned) : 0u;           // heads beyond the group: zeros
                    y[i] = real ? load_bf16_pair(qh + HALF + 2 * i, aligned) : 0u;
                    top = max(top, max(max(x[i] & 0x7fffu, (x[i] >> 16) & 0x7fffu), max(y[i] & 0x7fffu, (y[i] >> 16) & 0x7fffu)));
                }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const uint32_t ex = min(max(top >> 7, 1u), 253u);             // biased exponent of the largest element
                const float down = __uint_as_float((254u - ex) << 23);
                // (never 0, which a masked row's minus infinity is multiplied by: smaller logits than these are all alike)
                unit_scale = fmaxf(__uint_as_float(ex << 23) * p.sm_scale, 1.17549435e-38f);
#pragma unroll
                for (int i = 0; i < 4 * NW; ++i) {
                    x[i] = pack_bf16x2(__uint_as_float(x[i] << 16) * down, __uint_as_float(x[i] & 0xffff0000u) * down);
                    y[i] = pack_bf16x2(__uint_as_float(y[i] << 16) * down, __uint_as_float(y[i] & 0xffff0000u) * down);
                }
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    sm.q[warp][w][lane] = make_uint4(x[4 * w], x[4 * w + 1], x[4 * w + 2], x[4 * w + 3]);
                    sm.q[warp][NW + w][lane] = make_uint4(y[4 * w], y[4 * w + 1], y[4 * w + 2], y[4 * w + 3]);
                }
            }
            // a column of S^T is a query head: this thread's columns are heads 2t and 2t + 1
            const float per_log = CAP ? 1.f : kLog2e;
            const float mul0 = __shfl_sync(0xffffffffu, unit_scale, 8 * t) * per_log, mul1 = __shfl_sync(0xffffffffu, unit_scale, 8 * t + 4) * per_log;

            uint32_t qa[4 * NW], qb[4 * NW];
            const int swap = (key_of(g) & 2) * 2;
            const uint32_t blk_k = t * (D / 8) / kQuantBlock, pick = blk_k | (blk_k + 4) << 4;      // bytes of the row's K scales
            int in_macro = 0, unit = u0 + my_share * per;      // units of the macro tile done; the next one

            for (int s = 0; s < steps;) {
                const int cnt = min(min(2, per - in_macro), steps - s);
                const int row0 = (unit - first) * kUnit;       // first key of this step
                if (in_macro == 0) {
                    // the query, turned by its distance to the tile's first key
                    __syncwarp();
                    const int slot = lane / (D / 8) * (D / 8) + (((lane % (D / 8)) / 2 ^ ((lane / (D / 8)) * 2)) % (D / 16)) * 2 + (lane & 1);
                    sm.base[warp][slot] = cos_sin_fast(n - 1 - row0, f0);
                    if (D == 128) {
                        const int l2 = lane + 32, slot2 = l2 / 16 * 16 + (((l2 % 16) / 2 ^ ((l2 / 16) * 2)) % 8) * 2 + (l2 & 1);
                        sm.base[warp][slot2] = cos_sin_fast(n - 1 - row0, f1);
                    }
                    __syncwarp();
#pragma unroll
                    for (int w = 0; w < NW; ++w) {
                        const uint4 x4 = sm.q[warp][w][lane], y4 = sm.q[warp][NW + w][lane];
                        const uint32_t x[4] = {x4.x, x4.y, x4.z, x4.w}, y[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int i = 4 * w + e;
                            const float4 cs = *reinterpret_cast<const float4*>(&sm.base[warp][t * (D / 8) + ((i ^ (t * 2)) % (D / 16)) * 2]);
                            const float x0 = __uint_as_float(x[e] << 16), x1 = __uint_as_float(x[e] & 0xffff0000u);
                            const float y0 = __uint_as_float(y[e] << 16), y1 = __uint_as_float(y[e] & 0xffff0000u);
                            qa[i] = pack2(x0 * cs.x - y0 * cs.y, x1 * cs.z - y1 * cs.w);
                            qb[i] = pack2(y0 * cs.x + x0 * cs.y, y1 * cs.z + x1 * cs.w);
                        }
                    }
                }
                const int stage1 = stage + 1 == stages ? 0 : stage + 1;
                wait_phase(full + 8 * stage, phase, p.status, dead);
                if (cnt == 2) wait_phase(full + 8 * stage1, phase ^ (stage1 == 0), p.status, dead);

                // S^T of the step's two units side by side (of a step with one unit, the second is whatever its stage holds, masked
                // below): the products of one run while the other's operands are made
                float sc[2][4];
                const unsigned char* st[2] = {ring + stage * stage_bytes + my_head * Row::kBytes, ring + stage1 * stage_bytes + my_head * Row::kBytes};
                uint32_t s_lo[2][2], s_hi[2][2];               // scales of the thread's two blocks, [unit][parity of the key]
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        // all scales of the key's row at once; of them the thread's two
                        const unsigned char* row = st[j] + key_of(g + 8 * r) * pitch + Row::kKScales;
                        uint32_t lo, hi;
                        if constexpr (D == 128) { const uint2 x = *reinterpret_cast<const uint2*>(row); lo = x.x; hi = x.y; }
                        else { lo = *reinterpret_cast<const uint32_t*>(row); hi = lo >> 16; }
                        const uint32_t two = e4m3x2_to_f16(__byte_perm(lo, hi, pick));
                        s_lo[j][r] = __byte_perm(two, two, 0x1010);
                        s_hi[j][r] = __byte_perm(two, two, 0x3232);
                        sc[j][2 * r] = 0.f;
                        sc[j][2 * r + 1] = 0.f;
                    }
                const int in_second = min(in_macro + 1, kQtMacro - 1);
                uint32_t k_lo[2][2][NW], k_hi[2][2][NW];
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const unsigned char* row = st[j] + key_of(g + 8 * r) * pitch + t * 4 * NW;
                        load_words<D>(row, k_lo[j][r]);
                        load_words<D>(row + D / 4, k_hi[j][r]);
                    }
#pragma unroll
                for (int w = 0; w < NW; ++w)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint32_t a_lo[2][4], a_hi[2][4];
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const uint4* turn = sm.turn[(j == 0 ? in_macro : in_second) * kUnit + key_of(g + 8 * r)];
                            const uint4 c4 = turn[(4 * w + t) ^ swap], s4 = turn[(4 * (NW + w) + t) ^ swap];
                            const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w}, sn[4] = {s4.x, s4.y, s4.z, s4.w};
                            uint32_t x[4], y[4];
                            e2m1x8_to_f16(k_lo[j][r][w], x);
                            e2m1x8_to_f16(k_hi[j][r][w], y);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t xs = mul2(x[e], s_lo[j][r]), ys = mul2(y[e], s_hi[j][r]);
                                a_lo[r][e] = fnma2(ys, sn[e], mul2(xs, c[e]));
                                a_hi[r][e] = fma2(xs, sn[e], mul2(ys, c[e]));
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t a[4] = {a_lo[0][e], a_lo[1][e], a_hi[0][e], a_hi[1][e]};
                            mma_f16_16816(sc[j], a, qa[4 * w + e], qb[4 * w + e]);
                        }
                    }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int left = j < cnt ? n - (row0 + j * kUnit) : 0;
                    if (left < kUnit) {                        // the request's last unit, or none
#pragma unroll
                        for (int r = 0; r < 2; ++r)
                            if (key_of(g + 8 * r) >= left) { sc[j][2 * r] = -INFINITY; sc[j][2 * r + 1] = -INFINITY; }
                    }
                    if (CAP) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = sc[j][e] * ((e & 1) ? mul1 : mul0);
                            sc[j][e] = x == -INFINITY ? x : p.logit_cap * tanhf(x / p.logit_cap) * kLog2e;
                        }
                    }
                }
                const float k0 = CAP ? 1.f : mul0, k1 = CAP ? 1.f : mul1;
                float x0 = fmaxf(fmaxf(sc[0][0], sc[0][2]), fmaxf(sc[1][0], sc[1][2])) * k0;
                float x1 = fmaxf(fmaxf(sc[0][1], sc[0][3]), fmaxf(sc[1][1], sc[1][3])) * k1;
#pragma unroll
                for (int off = 4; off <= 16; off <<= 1) {
                    x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, off));
                    x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, off));
                }
                // the reference maximum moves only when a row grew by more than 2^8: weights stay below 2^(8 + kQtLift)
                if (__any_sync(0xffffffffu, x0 > m0 + 8.f || x1 > m1 + 8.f)) {
                    const float n0 = fmaxf(fmaxf(m0, x0), -1e30f), n1 = fmaxf(fmaxf(m1, x1), -1e30f);
                    const float c0 = exp2_fast(m0 - n0), c1 = exp2_fast(m1 - n1);
                    m0 = n0, m1 = n1;
                    l0 *= c0, l1 *= c1;
#pragma unroll
                    for (int i = 0; i < MT; ++i) { o[i][0] *= c0; o[i][1] *= c1; o[i][2] *= c0; o[i][3] *= c1; }
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if (j >= cnt) break;
                    float pe[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) pe[e] = exp2_fast(fmaf(sc[j][e], (e & 1) ? k1 : k0, kQtLift - ((e & 1) ? m1 : m0)));
                    l0 += pe[0] + pe[2];
                    l1 += pe[1] + pe[3];
                    const uint32_t b0 = transpose8(pack2(pe[0], pe[1])), b1 = transpose8(pack2(pe[2], pe[3]));
                    const unsigned char* ra = st[j] + key_of(2 * t) * pitch;           // keys of the fragment's columns 2t, 2t+1,
                    const unsigned char* rb = st[j] + key_of(2 * t + 1) * pitch;       // and one row further on 2t+8, 2t+9
                    const int blk = g * (D / 8) / kQuantBlock;
                    uint32_t a[2][MT], h[2][MT];               // even and odd d of the thread's block; keys (2t, 2t+1), (2t+8, 2t+9)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        uint32_t wa[NW], wb[NW];
                        load_words<D>(ra + r * pitch + Row::kV + g * 4 * NW, wa);
                        load_words<D>(rb + r * pitch + Row::kV + g * 4 * NW, wb);
                        const uint32_t s2 = e4m3x2_to_f16(ra[r * pitch + Row::kVScales + blk] | (uint32_t)rb[r * pitch + Row::kVScales + blk] << 8);
#pragma unroll
                        for (int w = 0; w < NW; ++w) {
                            uint32_t x[4], y[4];
                            e2m1x8_to_f16((wa[w] & 0x0f0f0f0fu) | ((wb[w] << 4) & 0xf0f0f0f0u), x);
                            e2m1x8_to_f16(((wa[w] >> 4) & 0x0f0f0f0fu) | (wb[w] & 0xf0f0f0f0u), y);
#pragma unroll
                            for (int e = 0; e < 4; ++e) { a[r][4 * w + e] = mul2(x[e], s2); h[r][4 * w + e] = mul2(y[e], s2); }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const uint32_t f[4] = {a[0][i], h[0][i], a[1][i], h[1][i]};
                        mma_f16_16816(o[i], f, b0, b1);
                    }
                }
                __syncwarp();                                  // every lane has read the stages
                if (lane == 0) {
                    mbar_arrive(empty + 8 * stage);
                    if (cnt == 2) mbar_arrive(empty + 8 * stage1);
                }
                if (cnt == 2) {
                    stage = stage1;
                    phase ^= stage1 == 0;
                }
                if (++stage == stages) { stage = 0; phase ^= 1; }
                s += cnt;
                in_macro += cnt;
                unit += cnt;
                if (in_macro == per) { in_macro = 0; unit += skip; }
            }
#pragma unroll
            for (int off = 4; off <= 16; off <<= 1) {
                l0 += __shfl_xor_sync(0xffffffffu, l0, off);
                l1 += __shfl_xor_sync(0xffffffffu, l1, off);
            }
        }
        // This warp's partial result.  Elements of a head in the order in which the lanes hold them, so that eight lanes'
        // pairs are 64 bytes side by side; the join puts them back.
        if (busy) {
            const long long slot = (long long)(blockIdx.x + b) * share + my_share;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int head = 2 * t + k;
                if (head < p.group) {
                    const long long at = slot * p.hq + kv * p.group + head;
                    if (steps > 0) {
#pragma unroll
                        for (int i = 0; i < MT; ++i) *reinterpret_cast<float2*>(p.part_o + at * D + 16 * i + 2 * g) = make_float2(o[i][k], o[i][2 + k]);
                    }
                    if (g == 0) p.part_ml[at] = k == 0 ? make_float2(m0, l0) : make_float2(m1, l1);
                }
            }
        }
        u0 = u1;
    }
}

// ------------------------------------------------------------------------------------------------
// Join the partial results: grid (hq, batch)
// ------------------------------------------------------------------------------------------------
// LANES: elements in the order of the tensor-core kernel's lanes.  WARPS, AHEAD: partial results in flight, so that a request's
// are one round trip: 16 x 10 where a request has many (1 x 131072, 32 heads, the whole call: 61.4 us, 64.5 with 8 x 8), 8 x 8
// where it has 64 at most on average (16 x 1000..32000, 28 heads: 46.1 us; 52.0 with 16 x 10, whose one CTA per SM makes the 448
// of them four rounds; 47.6 with 4 x 8).
template <typename T, int D, bool LANES, int WARPS, int AHEAD>
__global__ void __launch_bounds__(32 * WARPS) quant_merge_kernel(const __grid_constant__ QuantAttendParams p) {
    constexpr int VEC = D / 32, NW = WARPS, kAhead = AHEAD;
    __shared__ int start[kQaMaxBatch + 1];
    __shared__ float s_acc[NW][D];
    __shared__ float2 s_ml[NW];
    const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    wait_for_predecessor();
    count_units(p, start);
    const int units = start[p.batch], pieces = used_pieces(p, units);
    float m = -INFINITY, l = 0.f, acc[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) acc[v] = 0.f;
    if (start[b] < start[b + 1]) {
        const int c_first = piece_of(start[b], units, pieces), count = (piece_of(start[b + 1] - 1, units, pieces) - c_first + 1) * p.share;
        const long long first = (long long)(c_first + b) * p.share;
        for (int c0 = warp; c0 < count; c0 += NW * kAhead) {
            float x[kAhead][VEC];
            float2 ml[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int c = c0 + NW * i;
                ml[i] = make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int v = 0; v < VEC; ++v) x[i][v] = 0.f;
                if (c < count) {
                    const long long at = (first + c) * p.hq + h;
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
                for (int v = 0; v < VEC; ++v) acc[v] += w > 0.f || w != w ? x[i][v] * w : 0.f;     // (a warp without units leaves no elements)
            }
            m = mn;
        }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) s_acc[warp][VEC * lane + v] = acc[v];
    if (lane == 0) s_ml[warp] = make_float2(m, l);
    __syncthreads();
    for (int e = threadIdx.x; e < D; e += 32 * WARPS) {
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
        const int d = LANES ? (e & 15) / 2 * (D / 8) + e / 16 * 2 + (e & 1) : e;
        // an empty request: no row, sum 0, zeros
        reinterpret_cast<T*>(p.out)[((long long)b * p.hq + h) * D + d] = from_f32<T>(start[b] < start[b + 1] ? r / ll * p.v_scale : 0.f);
    }
}

// Pieces the sequence of units is cut into: for the tensor cores one CTA per SM, eight warps over at most eight KV heads
// each; for the CUDA cores what fits an SM.  (With three or more blocks of heads the CTAs may be a few more than the SMs: 24 heads
// make 3 x 50, 40 heads 5 x 30, and the last two run behind the others.)
int tc_head_blocks(int hkv) { return (hkv + kQtWarps - 1) / kQtWarps; }
int attend_pieces(int dtype, int hkv, int sms) {
    return dtype == TS_DTYPE_BF16 ? (sms + tc_head_blocks(hkv) - 1) / tc_head_blocks(hkv) : 4 * sms;
}

// At most (a KV head serves up to eight query heads, a CTA's warps are shared out over its KV heads).
size_t partial_slots(int sms, int batch, int hq) {
    const int hkv = (hq + 7) / 8, share = hkv < kQtWarps ? kQtWarps / hkv : 1;
    const size_t tc = (size_t)(sms + batch) * share, plain = 4 * sms + batch;
    return tc > plain ? tc : plain;
}
size_t partial_bytes(int sms, int batch, int hq, int d) { return partial_slots(sms, batch, hq) * hq * (d + 2) * sizeof(float); }

template <typename T, int D, bool LANES>
cudaError_t launch_merge(const QuantAttendParams& p, cudaStream_t stream) {
    const dim3 grid(p.hq, p.batch);
    return p.pieces * p.share / p.batch > 64 ? launch_chained(quant_merge_kernel<T, D, LANES, 16, 10>, grid, dim3(512), 0, stream, p)
                                             : launch_chained(quant_merge_kernel<T, D, LANES, 8, 8>, grid, dim3(256), 0, stream, p);
}
template <int D>
cudaError_t launch_attend_plain(const QuantAttendParams& p, cudaStream_t stream) {
    const int nsub = (p.group + kQpHeads - 1) / kQpHeads, per_cta = kQpThreads / 32;
    const cudaError_t e = launch_chained(quant_attend_plain_kernel<float, D>, dim3(p.pieces, (p.hkv * nsub + per_cta - 1) / per_cta), dim3(kQpThreads), 0, stream, p);
    if (e != cudaSuccess) return e;
    return launch_merge<float, D, false>(p, stream);
}
template <int D, bool CAP, int PIECE>
cudaError_t launch_attend_tc(QuantAttendParams p, cudaStream_t stream) {
    using Launch = QtLaunch<PIECE>;
    static SmemConfig configured = {};
    p.share = shares_of<D>((p.hkv + tc_head_blocks(p.hkv) - 1) / tc_head_blocks(p.hkv));
    p.step_units = 2 * p.share;
    // The computing warpgroups wait for registers that the launch has to have brought along: never launch without them.
    static const bool enough = [] {
        cudaFuncAttributes attr;
        return cudaFuncGetAttributes(&attr, quant_attend_tc_kernel<D, CAP, PIECE>) == cudaSuccess &&
               attr.numRegs * Launch::kThreads >= Launch::kComputeRegs * 32 * kQtWarps + kQtLoadRegs * 32 * Launch::kLoaders;
    }();
    if (!enough) return cudaErrorInvalidDeviceFunction;
    cudaError_t e = ensure_dynamic_smem(quant_attend_tc_kernel<D, CAP, PIECE>, kQtBytes, configured);
    if (e != cudaSuccess) return e;
    e = launch_chained(quant_attend_tc_kernel<D, CAP, PIECE>, dim3(p.pieces, tc_head_blocks(p.hkv)), dim3(Launch::kThreads), kQtBytes, stream, p);
    if (e != cudaSuccess) return e;
    return launch_merge<__nv_bfloat16, D, true>(p, stream);
}
template <int D, bool CAP>
cudaError_t launch_attend_bf16(const QuantAttendParams& p, cudaStream_t stream) {
    // Bulk copies and 16-byte pieces need rows, and a CTA's heads in them, that start on multiples of 16 bytes.
    const int hpc = (p.hkv + tc_head_blocks(p.hkv) - 1) / tc_head_blocks(p.hkv);
    const bool grid16 = p.hkv * QuantRow<D>::kBytes % 16 == 0 && (hpc == p.hkv || hpc * QuantRow<D>::kBytes % 16 == 0);
    if (!grid16) return launch_attend_tc<D, CAP, 8>(p, stream);
    return hpc * QuantRow<D>::kBytes < kQtBulkBytes ? launch_attend_tc<D, CAP, 16>(p, stream) : launch_attend_tc<D, CAP, 0>(p, stream);
}

}  // namespace
}  // namespace ts

extern "C" int ts_quant_attend_workspace(int32_t device, int32_t batch, int32_t hq, int32_t head_dim, size_t* bytes) {
    using namespace ts;
    if (!bytes || batch < 0 || batch > kQaMaxBatch || hq < 1 || hq > 8192) return TS_ERR_INVALID_ARG;
    if (head_dim != 64 && head_dim != 128) return TS_ERR_UNSUPPORTED;
    const int sms = sms_of(device);
    if (sms <= 0) return TS_ERR_CUDA;
    *bytes = partial_bytes(sms, batch, hq, head_dim);          // whatever the type and the number of KV heads
    return TS_OK;
}

extern "C" int ts_quant_attend(const ts_quant_attend_args* a) {
    using namespace ts;
    if (!a || a->struct_size != sizeof(ts_quant_attend_args)) return TS_ERR_INVALID_ARG;
    if (a->dtype != TS_DTYPE_BF16 && a->dtype != TS_DTYPE_F32) return TS_ERR_UNSUPPORTED;
    if (a->head_dim != 64 && a->head_dim != 128) return TS_ERR_UNSUPPORTED;
    if (a->batch < 0 || a->batch > kQaMaxBatch || a->hq < 1 || a->hkv < 1 || a->hkv > 1024 || a->hq % a->hkv != 0) return TS_ERR_INVALID_ARG;
    if (a->hq / a->hkv > 8) return TS_ERR_UNSUPPORTED;
    if (!positive(a->rope_base) || !positive(a->rope_scale) || !power_of_two(a->k_scale) || !power_of_two(a->v_scale)) return TS_ERR_INVALID_ARG;
    if (a->max_reqs < 1 || a->max_ctx < 0 || a->req_to_token_stride < 0 || a->pool_rows < 1) return TS_ERR_INVALID_ARG;
    if (a->max_ctx > (1ll << 31) - kUnit || (a->max_ctx + kUnit - 1) / kUnit * a->batch >= (1ll << 31)) return TS_ERR_INVALID_ARG;   // units are counted in 32 bits
    if (!positive(a->sm_scale) || !isfinite(a->logit_cap)) return TS_ERR_INVALID_ARG;
    if (a->batch == 0) return TS_OK;
    if (!a->q || !a->pool || !a->req_to_token || !a->req_pool_indices || !a->seq_lens || !a->out || !a->workspace) return TS_ERR_INVALID_ARG;
    if (reinterpret_cast<uintptr_t>(a->pool) % 16 != 0 || reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0) return TS_ERR_INVALID_ARG;
    // (`out` may be `q`: it is written when all queries have been read.)
    const uint64_t heads = (uint64_t)a->batch * a->hq * a->head_dim * (a->dtype == TS_DTYPE_BF16 ? 2 : 4);
    const Extent out(a->out, heads), q(a->q, heads), pool(a->pool, (uint64_t)a->pool_rows * a->hkv * (a->head_dim * 9 / 8));
    const Extent table(a->req_to_token, 4 * (uint64_t)a->max_ctx, 4 * (uint64_t)a->req_to_token_stride, a->max_reqs);
    const Extent slots(a->req_pool_indices, 4 * (uint64_t)a->batch), lens(a->seq_lens, 4 * (uint64_t)a->batch);
    if (overlap(out, pool) || overlap(out, table) || overlap(out, slots) || overlap(out, lens)) return TS_ERR_INVALID_ARG;
    const int sms = sms_of(a->device);
    if (sms <= 0) return TS_ERR_CUDA;
    const int pieces = attend_pieces(a->dtype, a->hkv, sms);
    if (a->workspace_bytes < partial_bytes(sms, a->batch, a->hq, a->head_dim)) return TS_ERR_CAPACITY;
    const Extent work(a->workspace, partial_bytes(sms, a->batch, a->hq, a->head_dim));
    if (overlap(work, out) || overlap(work, q) || overlap(work, pool) || overlap(work, table) || overlap(work, slots) || overlap(work, lens)) return TS_ERR_INVALID_ARG;
    const DeviceScope scope(a->device);
    if (!scope.ok) return TS_ERR_CUDA;
    QuantAttendParams p;
    p.q = a->q; p.pool = static_cast<const unsigned char*>(a->pool); p.pool_rows = a->pool_rows;
    p.rtt = a->req_to_token; p.rtt_stride = a->req_to_token_stride; p.max_ctx = a->max_ctx;
    p.req_pool_indices = a->req_pool_indices; p.seq_lens = a->seq_lens; p.out = a->out;
    p.part_o = static_cast<float*>(a->workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + partial_slots(sms, a->batch, a->hq) * a->hq * a->head_dim);
    p.batch = a->batch; p.hq = a->hq; p.hkv = a->hkv; p.group = a->hq / a->hkv; p.max_reqs = a->max_reqs; p.pieces = pieces;
    p.sm_scale = a->sm_scale * a->k_scale; p.logit_cap = a->logit_cap; p.v_scale = a->v_scale;
    p.status = a->status; p.step_units = 1; p.share = 1;
    p.freqs = turn_freqs(a->rope_base, a->rope_scale, a->head_dim);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(a->stream);
    cudaError_t e;
    if (a->dtype == TS_DTYPE_F32) e = a->head_dim == 128 ? launch_attend_plain<128>(p, s) : launch_attend_plain<64>(p, s);
    else if (a->head_dim == 128) e = a->logit_cap > 0.f ? launch_attend_bf16<128, true>(p, s) : launch_attend_bf16<128, false>(p, s);
    else e = a->logit_cap > 0.f ? launch_attend_bf16<64, true>(p, s) : launch_attend_bf16<64, false>(p, s);
    return e == cudaSuccess ? TS_OK : TS_ERR_CUDA;
}
