// Internal interface between the shared-prefix attention's entry point and its prefix kernel.
#pragma once
#include <atomic>
#include <type_traits>

#include "common.cuh"

namespace vq {

// Partial softmax records in the workspace: of output row r and split j of n_splits,
//   o  [(r * n_splits + j) * D + d]  sum over the split's slots of 2^(score - m) * v
//   ml [(r * n_splits + j) * 2]      m (maximum score in the base-2 domain, -inf: nothing seen) and l
struct SharedPartials {
    float *o, *ml;
    int n_splits;  // prefix splits, then own splits
};

// The tcgen05 kernel (shared_tiles_tc5.cu): the splits it uses for the parts it takes, each `units` x `rows`
// query rows against a store (st NULL: not that part; `wanted` > 0: so many for the prefix; `beside`: what else
// there is to do meanwhile, in SM microseconds); its launch for the prefix (prefix_splits > 0, records from 0)
// and the own tokens (own_splits > 0, records from own_record0), one record a split; its "a bounded wait gave
// up" flag.
struct Tc5Part {
    const vq_kivi_rows *st;
    int64_t units, rows;
};
void shared_tiles_tc5_splits(const Tc5Part &prefix, const Tc5Part &own, int D, int wanted, double beside, const DeviceInfo &di, int *prefix_splits, int *own_splits);
int32_t shared_tiles_tc5_launch(const vq_shared_attend_args &a, const SharedPartials &parts, int prefix_splits, int own_splits, int own_record0,
                                cudaStream_t stream);
int32_t shared_tiles_tc5_take_timeout(int *flag);

// Opts a kernel into `bytes` of dynamic shared memory, once per device (`done`: one bit a device).
template <typename K>
int32_t allow_shared_memory(K *kernel, int bytes, std::atomic<uint64_t> &done) {
    int dev = 0;
    VQ_CHECK_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_acquire) & bit) return VQ_OK;
    VQ_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_release);
    return VQ_OK;
}

// Launch as a programmatic dependent of the kernel before it on the stream: its blocks may be placed while
// that kernel's last blocks finish, and must pass wait_for_previous() before they touch what it writes.
template <typename... P, typename... A>
int32_t launch_dependent(void (*kernel)(P...), const char *name, unsigned blocks, int threads, int smem, cudaStream_t st, bool dependent, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, P(args)...);
    if (e != cudaSuccess) return fail(VQ_ERR_CUDA, "launch of %s failed: %s", name, cudaGetErrorString(e));
    return VQ_OK;
}
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- packed codes to numbers ------------------------------------------------------------------
// A code c becomes the float BASE + c by placing its byte into the mantissa of BASE (one byte
// permutation), and code*scale + zero becomes one fused multiply-add against zero - BASE*scale.
// That difference is rounded once: an error of at most 2^-24 * BASE * scale, 2^-17 (2- and 4-bit
// codes) or 2^-9 (8-bit) of the quantization step.
template <int SB>
struct Codes {
    static constexpr float kBase = SB == 8 ? 32768.f : 128.f;
    static constexpr int kPerWord = 32 / SB;
    // plane k of a word: its codes k, k + 8/SB, k + 2 * 8/SB, ..., each alone in its byte
    __device__ static __forceinline__ uint32_t plane(uint32_t w, int k) {
        if constexpr (SB == 8) return w;
        else return (w >> (SB * k)) & (SB == 4 ? 0x0f0f0f0fu : 0x03030303u);
    }
    // BASE + the code in byte `b` of a plane
    __device__ static __forceinline__ float place(uint32_t plane, int b) {
        if constexpr (SB == 8) return __uint_as_float(__byte_perm(plane, 0x47000000u, 0x7404u | ((uint32_t)b << 4)));
        else return __uint_as_float(__byte_perm(plane, 0x43000000u, 0x7044u | ((uint32_t)b << 8)));
    }
    // code i of word w (i a compile-time constant after unrolling)
    __device__ static __forceinline__ float get(uint32_t w, int i) { return place(plane(w, i % (8 / SB)), i / (8 / SB)); }
};

__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}

// Codes to numbers in half precision, two at a time, for bfloat16 data and codes of 2 or 4 bits: a code beside
// the exponent of 1024 is the half 1024 + code * 2^bit, one half FMA makes it the code, exactly, and another
// one the value: 13 instructions instead of 20 a word of eight. Scale and zero are rounded to halves too, so a value is off by
// up to 2^-11 (code scale + |zero| + |value|) instead of 2^-11 |value|, and, where scale, zero or value lie below
// half's normal range, by (code + 2) 2^-25 more instead of 2^-25. Chosen for its time, with this error: calls of 16
// requests behind 8K tokens 24.4 us instead of 26.6, 64 behind 32K 72 instead of 82, prompts 377 instead of 428;
// relative rms error of outputs at 4 bits 0.0018 for values around 1 and 0.01 (float32 form 0.0017, which is
// bfloat16's own rounding), 0.0023 / 0.013 / 0.14 around 1e-4 / 1e-5 / 1e-6 (0.0017 / 0.0022 / 0.018). The contract in
// vqb200.h says so. float16 data keeps the float32 form: there the three roundings would show (its own is 0.0002).
// `w8` is w >> 8; pair i (0..3) is the codes in bits SB*i of the two halves of w.
template <int SB, typename T>
constexpr bool kHalfDecode = std::is_same<T, __nv_bfloat16>::value && SB != 8;
template <int SB>
__device__ __forceinline__ uint32_t half_codes(uint32_t w, uint32_t w8, int i) {
    const int bit = SB == 2 ? 2 * i : 4 * (i & 1);
    const uint32_t mask = (SB == 2 ? 0x00030003u : 0x000f000fu) << bit;
    const uint32_t x = ((SB == 4 && i >= 2 ? w8 : w) & mask) | 0x64006400u;
    // code = x * 2^-bit - 1024 * 2^-bit
    return hfma2(x, 0x3c003c00u - (uint32_t)bit * 0x04000400u, 0xe400e400u - (uint32_t)bit * 0x04000400u);
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Two float32 operations in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 8 halves as they come, or, where codes are decoded in pairs (i, i + 4), in the order 0 4 1 5 2 6 3 7
template <bool SPREAD>
__device__ __forceinline__ uint4 in_order(uint4 v) {
    if constexpr (!SPREAD) return v;
    return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
}

// Two neighbouring 16-bit floats as packed halves (bfloat16 goes through float32: exact inside
// half's normal range)
template <typename T>
__device__ __forceinline__ uint32_t as_f16x2(uint32_t raw);
template <>
__device__ __forceinline__ uint32_t as_f16x2<__half>(uint32_t raw) { return raw; }
template <>
__device__ __forceinline__ uint32_t as_f16x2<__nv_bfloat16>(uint32_t raw) {
    return pack_f16(__uint_as_float(raw << 16), __uint_as_float(raw & 0xffff0000u));
}

}  // namespace vq
