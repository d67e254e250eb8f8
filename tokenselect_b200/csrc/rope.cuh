// Angles of the rotary positions for the calls that keep no tables, and what those calls share on the host.
#pragma once
#include <math.h>

#include "extent.h"
#include "ptx.cuh"

namespace ts {

// A rotation angle is position * frequency, and only its part behind the last whole turn counts.  The frequency is held
// in turns as a 64-bit binary fraction, so the product with a whole position, taken modulo 2^64, IS that part: one integer
// multiplication, no reduction, and an error of position * 2^-56 turns (the frequency's own 53 bits) instead of the
// position * 2^-24 radians of a product in fp32, which at a million tokens is several degrees.
struct TurnFreqs {
    unsigned long long f[64];      // f[i]: base^(-2i/d) / (scale * 2 pi) modulo 1, times 2^64
};

// The last table of this thread is kept: it depends on the three numbers alone, and evaluating it takes 3 us.
inline const TurnFreqs& turn_freqs(double base, double scale, int d) {
    static thread_local struct { double base, scale; int d; TurnFreqs t; } last = {0.0, 0.0, 0, {}};
    if (last.base != base || last.scale != scale || last.d != d) {
        for (int i = 0; i < d / 2; ++i) {
            double turns = exp2(-log2(base) * (2.0 * i / d)) / (scale * 6.283185307179586476925286766559);
            turns -= floor(turns);
            last.t.f[i] = (unsigned long long)ldexp(turns < 1.0 ? turns : 0.0, 64);
        }
        last.base = base, last.scale = scale, last.d = d;
    }
    return last.t;
}

// The angle in units of pi, in [-1, 1).
__device__ __forceinline__ float half_turns(long long pos, unsigned long long f) {
    return (float)(int)((unsigned long long)(pos * (long long)f) >> 32) * 4.656612873077392578125e-10f;   // 2^-31
}
// cos and sin: to fp32's last bits, and to 2^-20 absolute (enough where the result is rounded to 16 bits).
__device__ __forceinline__ float2 cos_sin(long long pos, unsigned long long f) {
    float s, c;
    sincospif(half_turns(pos, f), &s, &c);
    return make_float2(c, s);
}
__device__ __forceinline__ float2 cos_sin_fast(long long pos, unsigned long long f) {
    const float a = half_turns(pos, f) * 3.14159265358979f;
    return make_float2(__cosf(a), __sinf(a));
}

// Makes `device` current for the life of the object: the handle-less calls take tensors of any device.
struct DeviceScope {
    int before = -1;
    bool ok = true;
    explicit DeviceScope(int device) {
        int now = -1;
        if (cudaGetDevice(&now) != cudaSuccess) { ok = false; return; }
        if (now == device) return;
        if (cudaSetDevice(device) != cudaSuccess) { ok = false; return; }
        before = now;
    }
    ~DeviceScope() { if (before >= 0) cudaSetDevice(before); }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
};

inline int sms_of(int device) {
    static int known[64] = {0};        // written with the same value whoever comes first
    if (device < 0 || device >= 64) return 0;
    if (known[device] == 0) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return 0;
        known[device] = n;
    }
    return known[device];
}

// Launch with programmatic stream serialization: the kernel may start while its predecessor drains and must not touch
// global memory before griddepcontrol.wait.
template <typename... Params, typename... Args>
inline cudaError_t launch_chained(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Two fp32 numbers an instruction.
__device__ __forceinline__ uint64_t pack_f32x2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ void wait_for_predecessor() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ void report(int* status, int code) {
    if (status != nullptr) atomicCAS(status, 0, code);
}

// Whether a phase is complete, without waiting for it (try_wait may suspend the warp for a while).
__device__ __forceinline__ bool test_phase(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// A wait of at most about a second; then the call's status says so, and the waits that follow give up at once.  While
// *`slow` is not 0 (a warp of the CTA is at work that may take long) the time does not run.
__device__ __forceinline__ void wait_phase(uint32_t bar, uint32_t parity, int* status, bool& dead, const volatile int* slow = nullptr) {
    if (mbar_try_wait(bar, parity) || dead) return;
    long long t0 = clock64();
    while (!mbar_try_wait(bar, parity)) {
        if (slow != nullptr && *slow != 0) t0 = clock64();
        if (clock64() - t0 > kWaitCycles) { report(status, TS_ERR_DEVICE_TIMEOUT); dead = true; return; }
    }
}

inline bool positive(double x) { return x > 0.0 && isfinite(x); }
inline bool power_of_two(float g) {
    int e;
    return g >= 2.3283064365386963e-10f && g <= 4294967296.f && frexpf(g, &e) == 0.5f;
}

}  // namespace ts
