// ts_quant_write, ts_quant_read: rows of a cache held in 4 bits, quantised as they are written and read back.
//
// Per block of sixteen elements x: scale = E4M3(min(max|x| / (6 g), 448)), code = E2M1(x / (g scale)), value = code scale g.
//
// What bounds both: HBM (a bf16 row of 2 KB at eight heads becomes 1152 bytes with its V) and, as they are, instructions and the
// waits for loads (16385 rows of eight heads: writing 25 us, issue slots 67 % busy, reading 18 us, 64 %; 13 us of bytes each); for
// the rows of a decode step the launch.  One thread takes one block: 32 bytes of bf16 or 64 of fp32 on one side, eight bytes of codes and one
// scale on the other, so the maximum needs no exchange and neighbouring lanes touch neighbouring bytes on both sides.
//
// Rounding is decided exactly.  g is a power of two, so x / g is exact; max|x| / 6 is IEEE-divided, and a quotient that
// lies beside a border of E4M3 does not round onto it (a border has five significant bits, so the dividend beside six times
// it is at least two thirds of a unit of the quotient's last place away).  Borders of E2M1 times a scale have at most
// seven significant bits: x either is on one, and then the quotient is exact, or at least 0.53 units of its last place off.
#include "quant.cuh"
#include "rope.cuh"

namespace ts {
namespace {

constexpr int kRowsThreads = 256;

struct QuantRowsParams {
    void* k;
    void* v;
    long long k_stride, v_stride;
    const int* rows;
    unsigned char* pool;
    long long pool_rows;
    unsigned blocks;                                           // count * hkv * 2 * head_dim/16
    int hkv;
    float k_scale, v_scale;
    int* status;
};

template <typename T, bool WIDE>
__device__ __forceinline__ void load_block(const T* src, T (&x)[kQuantBlock]) {
    if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(x) / 16; ++i) reinterpret_cast<uint4*>(x)[i] = reinterpret_cast<const uint4*>(src)[i];
    } else {
#pragma unroll
        for (int e = 0; e < kQuantBlock; ++e) x[e] = src[e];
    }
}

// Bits of the largest magnitude; an infinity or a NaN counts as the largest.
template <typename T>
__device__ __forceinline__ uint32_t largest(const T (&x)[kQuantBlock]) {
    if constexpr (sizeof(T) == 2) {                            // two at a time
        const uint32_t* w = reinterpret_cast<const uint32_t*>(x);
        uint32_t top = w[0] & 0x7fff7fffu;
#pragma unroll
        for (int e = 1; e < kQuantBlock / 2; ++e) top = __vmaxu2(top, w[e] & 0x7fff7fffu);
        return max(top & 0xffffu, top >> 16) << 16;
    } else {
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < kQuantBlock; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
        return top;
    }
}

// The block's codes in `w`; returns its scale.
template <typename T>
__device__ __forceinline__ uint32_t quantise_block(const T (&x)[kQuantBlock], float g, uint2& w) {
    const uint32_t top = largest<T>(x);
    w = make_uint2(0u, 0u);
    if (top >= 0x7f800000u) return 0x7fu;                      // an infinity or a NaN: the scale is NaN
    const float most = __uint_as_float(top) * (1.f / g);
    const uint32_t scale = f32_to_e4m3(fminf(__fdiv_rn(most, 6.f), 448.f));
    if (scale == 0) return 0;
    const float s = e4m3_to_f32(scale) * g;
    float y[2][8];
    if (most < 1e30f) {
        // Sixteen quotients by one divisor: Markstein's correction (1990) of the product with the rounded reciprocal gives the
        // rounded quotient in three operations.  (With the remainder's sign the other way round a zero keeps its own: -0 would
        // become +0, and a row read back and written again change.)
        const float inv_s = __fdiv_rn(1.f, s);
#pragma unroll
        for (int e = 0; e < kQuantBlock; ++e) {
            const float v = to_f32<T>(x[e]), q = v * inv_s;
            y[e >> 3][e & 7] = fmaf(-fmaf(q, s, -v), inv_s, q);
        }
    } else {                                                   // far beyond what the scale can hold: the quotient may be infinite
#pragma unroll
        for (int e = 0; e < kQuantBlock; ++e) y[e >> 3][e & 7] = __fdiv_rn(to_f32<T>(x[e]), s);
    }
    w = make_uint2(f32x8_to_e2m1(y[0]), f32x8_to_e2m1(y[1]));
    return scale;
}

struct BlockPlace { int i, head, part; bool is_v; };           // row of the call, head, block of the head
template <int D>
__device__ __forceinline__ BlockPlace block_place(unsigned b, unsigned hkv) {
    constexpr unsigned kParts = D / kQuantBlock;
    BlockPlace r;
    r.part = (int)(b % kParts);
    const unsigned u = b / kParts, w = u / hkv;                // (row, K or V, head)
    r.head = (int)(u - w * hkv);
    r.is_v = (w & 1) != 0;
    r.i = (int)(w >> 1);
    return r;
}

template <typename T, int D, bool WIDE>
__global__ void __launch_bounds__(kRowsThreads) quant_write_kernel(const QuantRowsParams p) {
    using Row = QuantRow<D>;
    const unsigned b = blockIdx.x * kRowsThreads + threadIdx.x;
    wait_for_predecessor();
    if (b >= p.blocks) return;
    const BlockPlace at = block_place<D>(b, p.hkv);
    const int row = p.rows[at.i];
    if (row < 0 || row >= p.pool_rows) { report(p.status, TS_ERR_BAD_SLOT); return; }
    const T* src = at.is_v ? reinterpret_cast<const T*>(p.v) + at.i * p.v_stride : reinterpret_cast<const T*>(p.k) + at.i * p.k_stride;
    alignas(16) T x[kQuantBlock];
    load_block<T, WIDE>(src + at.head * D + at.part * kQuantBlock, x);
    uint2 w;
    const uint32_t scale = quantise_block<T>(x, at.is_v ? p.v_scale : p.k_scale, w);
    unsigned char* dst = p.pool + ((long long)row * p.hkv + at.head) * Row::kBytes;
    *reinterpret_cast<uint2*>(dst + (at.is_v ? Row::kV : 0) + at.part * 8) = w;
    dst[(at.is_v ? Row::kVScales : Row::kKScales) + at.part] = (unsigned char)scale;
}

// Two threads share two neighbouring blocks, half of each for either: what the two store at a time lies side by side (with a
// block a thread, a store fills 16 of every 32 bytes).
template <typename T, int D, bool WIDE>
__global__ void __launch_bounds__(kRowsThreads) quant_read_kernel(const QuantRowsParams p) {
    using Row = QuantRow<D>;
    const unsigned b = blockIdx.x * kRowsThreads + threadIdx.x;
    wait_for_predecessor();
    if (b >= p.blocks) return;
    BlockPlace at = block_place<D>(b, p.hkv);
    const int half = at.part & 1;
    at.part &= ~1;
    const int row = p.rows[at.i];
    uint32_t w[2] = {0u, 0u}, scale[2] = {0u, 0u};
    if (row >= 0 && row < p.pool_rows) {
        const unsigned char* src = p.pool + ((long long)row * p.hkv + at.head) * Row::kBytes;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            w[i] = *reinterpret_cast<const uint32_t*>(src + (at.is_v ? Row::kV : 0) + (at.part + i) * 8 + half * 4);
            scale[i] = src[(at.is_v ? Row::kVScales : Row::kKScales) + at.part + i];
        }
    } else {
        report(p.status, TS_ERR_BAD_SLOT);
    }
    T* dst = (at.is_v ? reinterpret_cast<T*>(p.v) + at.i * p.v_stride : reinterpret_cast<T*>(p.k) + at.i * p.k_stride) +
             at.head * D + at.part * kQuantBlock + half * 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float s = e4m3_to_f32(scale[i]) * (at.is_v ? p.v_scale : p.k_scale);
        uint32_t h[4];
        e2m1x8_to_f16(w[i], h);
        alignas(16) T out[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = half2_to_float2(h[e]);
            out[2 * e] = from_f32<T>(f.x * s);
            out[2 * e + 1] = from_f32<T>(f.y * s);
        }
        if constexpr (WIDE) {
#pragma unroll
            for (int j = 0; j < (int)sizeof(out) / 16; ++j) reinterpret_cast<uint4*>(dst + i * kQuantBlock)[j] = reinterpret_cast<const uint4*>(out)[j];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) dst[i * kQuantBlock + e] = out[e];
        }
    }
}

template <typename T, int D>
cudaError_t launch_rows_t(const QuantRowsParams& p, bool write, cudaStream_t stream) {
    const uintptr_t bits = reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) | (uintptr_t)(p.k_stride * sizeof(T)) |
                           (uintptr_t)(p.v_stride * sizeof(T));
    const bool wide = bits % 16 == 0;
    const dim3 grid((p.blocks + kRowsThreads - 1) / kRowsThreads), block(kRowsThreads);
    if (write) return wide ? launch_chained(quant_write_kernel<T, D, true>, grid, block, 0, stream, p)
                           : launch_chained(quant_write_kernel<T, D, false>, grid, block, 0, stream, p);
    return wide ? launch_chained(quant_read_kernel<T, D, true>, grid, block, 0, stream, p)
                : launch_chained(quant_read_kernel<T, D, false>, grid, block, 0, stream, p);
}

int quant_rows(const ts_quant_rows_args* a, bool write) {
    if (!a || a->struct_size != sizeof(ts_quant_rows_args)) return TS_ERR_INVALID_ARG;
    if (a->dtype != TS_DTYPE_BF16 && a->dtype != TS_DTYPE_F32) return TS_ERR_UNSUPPORTED;
    if (a->head_dim != 64 && a->head_dim != 128) return TS_ERR_UNSUPPORTED;
    if (a->hkv < 1 || a->hkv > 1024 || a->count < 0 || a->pool_rows < 1) return TS_ERR_INVALID_ARG;
    if (a->k_stride < (int64_t)a->hkv * a->head_dim || a->v_stride < (int64_t)a->hkv * a->head_dim) return TS_ERR_INVALID_ARG;
    if (!power_of_two(a->k_scale) || !power_of_two(a->v_scale)) return TS_ERR_INVALID_ARG;
    if (a->count == 0) return TS_OK;
    if (!a->k || !a->v || !a->rows || !a->pool || reinterpret_cast<uintptr_t>(a->pool) % 16 != 0) return TS_ERR_INVALID_ARG;
    {
        const uint64_t es = a->dtype == TS_DTYPE_BF16 ? 2 : 4, n = (uint64_t)a->count, row = (uint64_t)a->hkv * a->head_dim * es;
        const Extent k(a->k, row, a->k_stride * es, n), v(a->v, row, a->v_stride * es, n), rows(a->rows, 4 * n);
        const Extent pool(a->pool, (uint64_t)a->pool_rows * a->hkv * (a->head_dim * 9 / 8));
        if (overlap(k, pool) || overlap(v, pool) || overlap(rows, pool)) return TS_ERR_INVALID_ARG;
        if (!write && (overlap(k, v) || overlap(k, rows) || overlap(v, rows))) return TS_ERR_INVALID_ARG;
    }
    const DeviceScope scope(a->device);
    if (!scope.ok) return TS_ERR_CUDA;
    QuantRowsParams p;
    p.k = a->k; p.v = a->v; p.k_stride = a->k_stride; p.v_stride = a->v_stride; p.rows = a->rows;
    p.pool = static_cast<unsigned char*>(a->pool); p.pool_rows = a->pool_rows; p.hkv = a->hkv;
    const long long blocks = (long long)a->count * a->hkv * 2 * (a->head_dim / kQuantBlock);
    if (blocks >= (1ll << 32) - kRowsThreads) return TS_ERR_CAPACITY;         // blocks are counted in 32 bits
    p.blocks = (unsigned)blocks;
    p.k_scale = a->k_scale; p.v_scale = a->v_scale; p.status = a->status;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(a->stream);
    cudaError_t e;
    if (a->dtype == TS_DTYPE_BF16) e = a->head_dim == 128 ? launch_rows_t<__nv_bfloat16, 128>(p, write, s) : launch_rows_t<__nv_bfloat16, 64>(p, write, s);
    else e = a->head_dim == 128 ? launch_rows_t<float, 128>(p, write, s) : launch_rows_t<float, 64>(p, write, s);
    return e == cudaSuccess ? TS_OK : TS_ERR_CUDA;
}

}  // namespace
}  // namespace ts

extern "C" int ts_quant_write(const ts_quant_rows_args* a) { return ts::quant_rows(a, true); }
extern "C" int ts_quant_read(const ts_quant_rows_args* a) { return ts::quant_rows(a, false); }
