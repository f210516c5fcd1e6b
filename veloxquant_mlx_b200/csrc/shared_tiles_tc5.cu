// Shared-prefix attention on the fifth-generation tensor cores: all B * H_q/H_kv * S_q query rows of a
// kv head against ONE copy of the packed prefix, and, where each request brings many query rows (its own
// prompt), those rows against the request's own tokens.
//
// Per 128 query rows and 128 tokens: S = Q K^T (tcgen05.mma, float16 in, float32 in tensor memory),
// P = 2^(S scale - m) (float16, back into tensor memory over S), O += P V (A operand from tensor
// memory). Each CTA keeps two such streams in flight so that the softmax of one runs under the MMAs
// of the other:
//   more than 128 rows: two row tiles share every decoded token tile;
//   up to 128 rows:     one row tile, the streams take token tiles in turn and are joined at the end.
// Roles: warps 0-3 and 4-7 the softmax of stream 0 and 1 (a thread owns a row: no exchange between
// lanes), warps 8-11 decode keys, 12-15 values, warp 16 issues the MMAs. Codes go from global memory to
// registers one tile ahead (a register is refilled as soon as its code is used), through one fused
// multiply-add and one rounding into 128-byte-swizzled operand tiles, two stages each. Decoding once for
// 128 or 256 rows is what makes dense float16 operands affordable (the decode kernel for a few rows folds
// the scales into its queries instead).
//
// The reference maximum m of a row moves only when one of 64 scores exceeds it by more than 2^8: O, with the weights of
// the tokens before, is then rescaled by the row's own thread. Weights are held times 2^7: up to 2^15, which float16
// holds, and down to 2^-32 of 2^m before its smallest step (2^-25 without the factor, and then the tail behind one
// token that outweighs all others is lost: 4096 tokens of 2^-26 each came out as 0). The factor costs nothing: it is in
// the exponent (m itself is held 7 lower, so that rescaling stays exact). That S of step i + 1 is complete implies that P V of step i is (MMAs of one thread
// complete in order), so only the second half of a tile waits for more (P V of the first).
//
// Measured at 4 bits in bfloat16: 256 query rows of each of 8 kv heads behind 32K tokens, 13 splits (104 CTAs, beside
// the own tokens' kernel), 56-60 us; 8192 rows behind 8K tokens, 337 us = 0.83 PFLOP/s, 50 % of the measured bfloat16 rate. A pair of row tiles takes
// about 4300 clocks a token tile, against 2048 for the MMAs, 2048 for the exponentials (16 a clock), 1000 for
// HBM and about 2400 of instruction issue: what bounds it is the chain of one stream (1000 until scores are
// there: the last half of P V 256, Q K 700; weights 3350, of which about 2000 beside the other stream's), of
// which two run side by side.
//
// Every wait is bounded; a role that gives up raises a flag (reported by vq_kivi_attend_status), leaves its
// loop, and the CTA still waits (bounded) for its MMAs and frees its tensor memory.
#include <algorithm>
#include <type_traits>

#include "shared_attend.h"

namespace vq {
namespace {

constexpr int kTile = 128;         // query rows of a stream = tensor-memory lanes; tokens of a tile
constexpr int kGroup = 32;
constexpr int kThreads = 17 * 32;
constexpr uint32_t kSpin = 1u << 20;
constexpr float kLazy = 8.f;       // log2 of how far a maximum may rise before O is rescaled
constexpr float kLift = 7.f;       // log2 of the factor on weights: kLazy + kLift = 15, below float16's 2^16
constexpr float kFar = 1 << 20;    // scores (base 2) from here on are spaced by 2^-3 and more

__device__ int g_shared_timeout = 0;
std::atomic<uint64_t> g_launched{0};  // one bit a device that the kernel was ever launched on (or captured for)
uint64_t device_bit(int dev) { return 1ull << (dev & 63); }

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, uint32_t limit = kSpin) {
    for (uint32_t i = 0; i < limit; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
    }
    return false;
}

// Shared-memory matrix descriptor with the 128-byte swizzle (tiles start on 1024-byte boundaries).
// K-major: rows of 64 channels, 8-row groups `sbo` apart. MN-major: 64 channels of 8 tokens are one
// 1024-byte block, token groups `sbo` apart, channel halves `lbo` apart.
__device__ __forceinline__ uint64_t make_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    uint64_t d = 0;
    d |= (uint64_t)((addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)((lbo >> 4) & 0x3FFFu) << 16;
    d |= (uint64_t)((sbo >> 4) & 0x3FFFu) << 32;
    d |= 1ull << 46;  // descriptor version of this architecture
    d |= 2ull << 61;  // 128-byte swizzle
    return d;
}
// kind::f16, float16 operands, float32 accumulator, M = 128; B K-major or MN-major
__device__ __forceinline__ constexpr uint32_t make_idesc(int N, bool b_mn_major) {
    return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
                 "l"(b), "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a),
                 "l"(b), "r"(idesc), "r"(accumulate)
                 : "memory");
}
// true in one lane of the (converged) warp, always the same one
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// The loaded values are threaded through the wait so that no use of them is scheduled ahead of it.
__device__ __forceinline__ void tmem_ld_wait(float (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
                   "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]),
                   "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]),
                   "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
                 "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

__device__ __forceinline__ void tmem_ld8(uint32_t addr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
                 "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
// 8 columns of this lane times f
__device__ __forceinline__ void scale_o(uint32_t addr, float f) {
    uint32_t r[8];
    tmem_ld8(addr, r);
#pragma unroll
    for (int k = 0; k < 8; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * f);
    tmem_st8(addr, r);
}
// One of the two parts of a call: the prefix (a unit is a kv head) or the own tokens (a kv head of a request)
struct Part {
    vq_kivi_rows st;
    int blocks;       // units x row_blocks x splits
    int splits;       // CTAs along the tokens
    int row_blocks;   // CTAs along the query rows of a unit
    int rows;         // query rows of a unit
    int tiles_packed, tiles;
    int record0;      // first partial record
};
struct TileParams {
    const void *q;
    const int32_t *own_start;
    float scale_log2;
    int H_q, H_kv, S_q, G, causal;
    int wait_test;    // self-test: also wait (briefly, behind all the work) on a barrier that nothing arms
    SharedPartials parts;
    Part prefix, own;
};

// The block is launched with 96 registers a thread; where decoding needs fewer, the two softmax warpgroups
// take over what the two decoding ones can spare (their sum is what the four were launched with: a kernel compiled to
// fewer would wait for registers that nobody gives back, so the launch looks at the count).
constexpr int kLaunchRegisters = 96, kMore = 120, kFewer = 72;
static_assert(kMore + kFewer <= 2 * kLaunchRegisters, "two warpgroups take what the two others give");
template <bool SPARE>
__device__ __forceinline__ void more_registers() {
    if constexpr (SPARE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMore));
}
template <bool SPARE>
__device__ __forceinline__ void fewer_registers() {
    if constexpr (SPARE) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewer));
}

template <int D>
struct Layout {
    static constexpr int HALVES = D / 64;                     // 64-channel (128-byte) halves of a tile
    static constexpr int HALF = kTile * 128;                  // bytes of one half
    static constexpr int TILE = HALVES * HALF;
    static constexpr int Q = 0, K = 2 * TILE, V = 4 * TILE;   // two Q tiles, two stages of K and V
    static constexpr int OUT_ROW = 4 * D + 16;                // a row of O on its way out: padded, conflict-free
    static constexpr int OUT = 2 * kTile * OUT_ROW;           // (over the tiles, when they are done with)
    static constexpr int ML = OUT;                            // (m, l) of every thread's row
    static constexpr int BARS = 6 * TILE;
    static_assert(OUT + 2 * kTile * 8 <= BARS, "rows on their way out fit over the tiles");
    // padded past half an SM's shared memory: one CTA an SM, as it takes all of tensor memory
    static constexpr int BYTES = BARS + 256 > 120 * 1024 ? BARS + 256 : 120 * 1024;
    // 16-byte chunk `c` (0 .. D/8) of row `r`
    __device__ static __forceinline__ uint32_t at(int r, int c) { return (uint32_t)((c >> 3) * HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }
};

enum { kKFull = 0, kKEmpty = 2, kVFull = 4, kVEmpty = 6, kSFull = 8, kPReady = 10, kPVHalf = 14, kODone = 16, kDrain = 18, kIdle = 19, kBars = 20 };

__device__ __forceinline__ uint4 zero4() { return make_uint4(0u, 0u, 0u, 0u); }

// 8 neighbouring codes of a row (SB bytes) as 8 halves; scale and zero - BASE * scale of channel pairs
template <int SB>
__device__ __forceinline__ uint4 decode8(const uint32_t (&w)[SB == 8 ? 2 : 1], const float2 (&sc)[4], const float2 (&ze)[4]) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        constexpr int per = Codes<SB>::kPerWord;
        const float2 c = make_float2(Codes<SB>::get(w[2 * i / per], 2 * i % per), Codes<SB>::get(w[(2 * i + 1) / per], (2 * i + 1) % per));
        const float2 v = fma2(c, sc[i], ze[i]);
        r[i] = pack_f16(v.x, v.y);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

// The same in half precision (half_codes). Word i of the result holds channels i and i + 4: see in_order.
template <int SB>
__device__ __forceinline__ uint4 decode8_half(uint32_t w, const uint32_t (&sc)[4], const uint32_t (&ze)[4]) {
    uint32_t r[4];
    if constexpr (SB == 2) w = __byte_perm(w, 0u, 0x4140);  // codes 0-3 into the low half, 4-7 into the high one
    const uint32_t w8 = w >> 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = hfma2(half_codes<SB>(w, w8, i), sc[i], ze[i]);
    return make_uint4(r[0], r[1], r[2], r[3]);
}
template <int D, int SB, typename T>
__global__ void __launch_bounds__(kThreads, 1) shared_tiles_tc5_kernel(const __grid_constant__ TileParams p) {
    using L = Layout<D>;
    constexpr int CHUNKS = D / 8;      // 8-channel chunks of a row
    constexpr int RB = D * SB / 8;     // bytes of a packed row
    constexpr bool HALF = kHalfDecode<SB, T>;  // decode8_half; channels of a chunk spread
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::BARS);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::BARS + 8 * kBars);
    const uint32_t bar0 = smem_u32(bars);
    auto bar = [&](int i) { return bar0 + 8u * i; };
    let_next_start();

    const bool is_prefix = (int)blockIdx.x < p.prefix.blocks;
    const Part &part = is_prefix ? p.prefix : p.own;
    int blk = is_prefix ? blockIdx.x : blockIdx.x - p.prefix.blocks;
    const int split = blk % part.splits; blk /= part.splits;
    const int rb = blk % part.row_blocks;
    const int unit = blk / part.row_blocks;
    const int b_own = is_prefix ? 0 : unit / p.H_kv;
    const int hk = is_prefix ? unit : unit - b_own * p.H_kv;
    const int n_rows = part.rows, per_req = p.G * p.S_q;
    const bool two = n_rows > kTile;                   // two row tiles, or one that both streams work on
    const int row0 = rb * (two ? 2 * kTile : kTile);
    const vq_kivi_rows &st = part.st;
    const int n_slots = st.n_quant + st.n_res, tiles_packed = part.tiles_packed;
    const int first_slot = is_prefix || !p.own_start ? 0 : min(n_slots, max(0, __ldg(p.own_start + b_own)));
    const int t_first = first_slot < st.n_quant ? first_slot / kTile : min(part.tiles, tiles_packed + (first_slot - st.n_quant) / kTile);
    const int t_lo = t_first + (int)((int64_t)(part.tiles - t_first) * split / part.splits);
    const int t_hi = t_first + (int)((int64_t)(part.tiles - t_first) * (split + 1) / part.splits);
    const int n_tiles = t_hi - t_lo;
    const int n_steps = two ? 2 * n_tiles : n_tiles;

    auto out_row = [&](int r) {  // output row (= row of q) of the unit's query row r
        const int b = is_prefix ? r / per_req : b_own, rem = is_prefix ? r - b * per_req : r;
        return ((int64_t)b * p.H_q + (int64_t)hk * p.G) * p.S_q + rem;
    };
    bool gave_up = false;
    auto wait = [&](int b, uint32_t parity) {  // by whole warps: all lanes go on or none
        if (!gave_up) gave_up = !__all_sync(0xffffffffu, mbar_wait(bar(b), parity));
        return !gave_up;
    };
    uint32_t tmem = 0;
    // Everything before the roles' loops: what the loops need is complete and visible behind it. The
    // decoding warps ask for their first codes before they come here.
    auto ready = [&]() {
        fence_async_smem();
        fence_before();
        __syncthreads();
        fence_after();
        tmem = *tmem_slot;
    };

    if ((smem_u32(smem) & 1023u) != 0) {  // the swizzle assumes it; never seen
        if (tid == 0) atomicExch(&g_shared_timeout, 2);
        return;
    }
    // scores (and the weights over them) of stream s: columns 128 s of tensor memory; its output: 256 + 128 s
    if (warp < 8) {
        // ---- softmax: thread = row -----------------------------------------------------------------
        // First the query tiles: copied as they are (all in flight at once), then made halves in place; rows
        // behind the last are zero. (Small loops: code that runs once is fetched from L2 line by line.)
        constexpr int STEP = 256 / CHUNKS;  // rows that the 256 threads cover at once
        const int qc = tid % CHUNKS, q_rows = (two ? 2 : 1) * kTile;
        auto q_at = [&](int r) { return smem + L::Q + (r / kTile) * L::TILE + L::at(r % kTile, qc); };
        int b = (row0 + tid / CHUNKS) / per_req, rem = row0 + tid / CHUNKS - b * per_req;  // (own: b = 0)
        const int step_b = STEP / per_req, step_rem = STEP - step_b * per_req;
#pragma unroll 1
        for (int r = tid / CHUNKS; r < q_rows; r += STEP) {
            const bool in = row0 + r < n_rows;
            const int64_t row = ((int64_t)(b_own + b) * p.H_q + (int64_t)hk * p.G) * p.S_q + rem;
            const T *src = reinterpret_cast<const T *>(p.q) + (in ? row : 0) * D + 8 * qc;
            b += step_b;
            rem += step_rem;
            if (rem >= per_req) { rem -= per_req; ++b; }
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(q_at(r))), "l"(src), "r"(in ? 16 : 0) : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if constexpr (HALF || std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll 4
            for (int r = tid / CHUNKS; r < q_rows; r += STEP) {
                uint4 *at = reinterpret_cast<uint4 *>(q_at(r));
                const uint4 v = *at;
                *at = in_order<HALF>(make_uint4(as_f16x2<T>(v.x), as_f16x2<T>(v.y), as_f16x2<T>(v.z), as_f16x2<T>(v.w)));
            }
        }
        ready();
        more_registers<HALF>();
        const int s = warp >> 2;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + 128 * s + lane_base, to = ts + 256;
        const int n_mine = two ? n_tiles : (n_tiles - s + 1) / 2;
        const int r = row0 + (two ? s * kTile : 0) + (warp & 3) * 32 + lane;
        // slots [first_slot, lim) are seen by this row
        const int lim = is_prefix || !p.causal ? n_slots : n_slots - p.S_q + r % p.S_q + 1;
        // (tiles within [first_slot, the warp's smallest lim) need no mask)
        const int all_see = __reduce_min_sync(0xffffffffu, lim);
        float m = -INFINITY, l = 0.f;  // reference maximum (times scale, base 2) less kLift, and the weights' sum
        bool far = false;              // (of the whole warp) a maximum lies far from 0
        for (int i = 0; i < n_mine; ++i) {
            const int t = t_lo + (two ? i : 2 * i + s);
            const int slot0 = t < tiles_packed ? t * kTile : st.n_quant + (t - tiles_packed) * kTile;
            // columns [lo, hi) of the tile
            const int lo = first_slot - slot0, hi = min(lim, t < tiles_packed ? st.n_quant : n_slots) - slot0;
            const bool masked = slot0 < first_slot || slot0 + kTile > (t < tiles_packed ? min(all_see, st.n_quant) : all_see);
            if (!wait(kSFull + s, i & 1)) break;
            fence_after();
            float2 sum[2] = {};
            auto largest = [&](int c, float (&v)[32]) {  // of 32 scores, the masked ones dropped
                if (masked) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) v[k] = c + k >= lo && c + k < hi ? v[k] : -INFINITY;
                }
                float mx = max3(v[0], v[1], v[2]), m1 = max3(v[3], v[4], v[5]);
#pragma unroll
                for (int k = 6; k < 30; k += 4) {
                    mx = max3(mx, v[k], v[k + 1]);
                    m1 = max3(m1, v[k + 2], v[k + 3]);
                }
                return fmaxf(max3(mx, m1, v[30]), v[31]);
            };
            float base;
            auto weights = [&](int c, const float (&v)[32]) {
                uint32_t r[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    float2 x = fma2(make_float2(v[2 * k], v[2 * k + 1]), make_float2(p.scale_log2, p.scale_log2), make_float2(base, base));
                    x.x = ex2(x.x);
                    x.y = ex2(x.y);
                    sum[k & 1] = add2(sum[k & 1], x);
                    r[k] = pack_f16(x.x, x.y);
                }
                tmem_st16(ts + c / 2, r);  // (over scores that have been read)
            };
            float v[32], w[32];
            tmem_ld32(ts, v);
            tmem_ld32(ts + 32, w);
#pragma unroll 1
            for (int c = 0; c < kTile; c += 64) {  // half of the tokens: their largest score may first raise m
                tmem_ld_wait(v);
                tmem_ld_wait(w);
                const float m0 = largest(c, v), mx = __fmul_rn(fmaxf(m0, largest(c + 32, w)), p.scale_log2);
                if (__any_sync(0xffffffffu, mx - m > kLazy + kLift)) {  // (a difference: exact however large the two are)
                    const float mn = mx - m > kLazy + kLift ? mx - kLift : m, f = m == -INFINITY ? 0.f : mn == m ? 1.f : ex2(m - mn);
                    m = mn;
                    far = __any_sync(0xffffffffu, m != -INFINITY && fabsf(m) > kFar);
                    l *= f;
#pragma unroll
                    for (int k = 0; k < 2; ++k) { sum[k].x *= f; sum[k].y *= f; }
                    // (the weights of the first half may have been taken by now: O holds them once that P V is done)
                    if (c > 0) wait(kPVHalf + s, i & 1);
                    if (i > 0 || c > 0) {
                        fence_after();
#pragma unroll 1
                        for (int k = 0; k < D; k += 8) scale_o(to + k, f);
                    }
                }
                base = m == -INFINITY ? 0.f : -m;
                if (far) {
                    // There the product that the fused multiply-add does not round exceeds the rounded maximum by half
                    // a step of float32, more than the weights have room for: products are rounded first here.
                    const float back = 1.f / p.scale_log2;
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        v[k] = (__fmul_rn(v[k], p.scale_log2) + base) * back;
                        w[k] = (__fmul_rn(w[k], p.scale_log2) + base) * back;
                    }
                    base = 0.f;
                }
                weights(c, v);
                if (c == 0) tmem_ld32(ts + 64, v);
                weights(c + 32, w);
                if (c == 0) tmem_ld32(ts + 96, w);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(kPReady + 2 * s + (c >> 6)));
            }
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        }
        // O goes out through shared memory: a row a lane there, whole rows at a time to global memory. The
        // tiles it overwrites are done with when both streams are.
        if (n_steps > 0) wait(kODone, 0);
        if (n_steps > 1) wait(kODone + 1, 0);
        fence_after();
        const bool live = r < n_rows;
        const int64_t rec = live ? out_row(r) * p.parts.n_splits + part.record0 + split : 0;
        uint8_t *rows = smem + warp * 32 * L::OUT_ROW, *mine = rows + lane * L::OUT_ROW;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
            float v[32];
            tmem_ld32(to + c, v);
            tmem_ld_wait(v);
            if (n_mine == 0) {
#pragma unroll
                for (int k = 0; k < 32; ++k) v[k] = 0.f;
            }
            // (channels i and i + 4 of a spread chunk are columns 2 i and 2 i + 1)
            float4 *at = reinterpret_cast<float4 *>(mine + 4 * c);
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
                at[k / 4] = HALF ? make_float4(v[k], v[k + 2], v[k + 4], v[k + 6]) : make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                at[k / 4 + 1] = HALF ? make_float4(v[k + 1], v[k + 3], v[k + 5], v[k + 7]) : make_float4(v[k + 4], v[k + 5], v[k + 6], v[k + 7]);
            }
        }
        constexpr int LPR = D / 4;  // lanes that write a row
        if (two) {
            if (live) *reinterpret_cast<float2 *>(p.parts.ml + rec * 2) = make_float2(m, l);
            __syncwarp();
#pragma unroll 4
            for (int i = 0; i < 32; i += 32 / LPR) {
                const int from = i + lane / LPR;
                const float4 v = *reinterpret_cast<const float4 *>(rows + from * L::OUT_ROW + 16 * (lane % LPR));
                const int64_t to_rec = __shfl_sync(0xffffffffu, rec, from);
                if (r - lane + from < n_rows) *reinterpret_cast<float4 *>(p.parts.o + to_rec * D + 4 * (lane % LPR)) = v;
            }
        } else {  // the streams' two records of a row become one; each stream's warps write half of the rows
            float2 *ml = reinterpret_cast<float2 *>(smem + L::ML) + (warp & 3) * 32 + lane;
            ml[s * kTile] = make_float2(m, l);
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const float2 a = ml[0], b = ml[kTile];
            const float mm = fmaxf(a.x, b.x), base = mm == -INFINITY ? 0.f : mm, fa = ex2(a.x - base), fb = ex2(b.x - base);
            if (live && s == 0) *reinterpret_cast<float2 *>(p.parts.ml + rec * 2) = make_float2(mm, a.y * fa + b.y * fb);
            rows = smem + (warp & 3) * 32 * L::OUT_ROW;
#pragma unroll 4
            for (int i = 16 * s; i < 16 * s + 16; i += 32 / LPR) {
                const int from = i + lane / LPR;
                const uint8_t *at = rows + from * L::OUT_ROW + 16 * (lane % LPR);
                const float4 x = *reinterpret_cast<const float4 *>(at), y = *reinterpret_cast<const float4 *>(at + kTile * L::OUT_ROW);
                const float f = __shfl_sync(0xffffffffu, fa, from), g = __shfl_sync(0xffffffffu, fb, from);
                const int64_t to_rec = __shfl_sync(0xffffffffu, rec, from);
                if (r - lane + from < n_rows)
                    *reinterpret_cast<float4 *>(p.parts.o + to_rec * D + 4 * (lane % LPR)) =
                        make_float4(x.x * f + y.x * g, x.y * f + y.y * g, x.z * f + y.z * g, x.w * f + y.w * g);
            }
        }
    } else if (warp < 12) {
        fewer_registers<HALF>();
        // ---- keys: warp w decodes the w-th 32-token group of a tile -----------------------------------
        // lane = (token parity, chunk of 8 channels): the group's scales and zeros of 8 channels stay in registers
        constexpr int TPL = 32 / CHUNKS;          // tokens a warp covers at once: 2 (D = 128) or 4
        constexpr int N = kGroup / TPL;           // tokens a lane decodes
        constexpr int W = SB == 8 ? 2 : 1;
        const int w = warp - 8, chunk = lane % CHUNKS, sub = lane / CHUNKS;
        const uint8_t *codes = st.k_codes + unit * st.k_codes_stride_bh;
        const float *ks = st.k_scale + unit * st.k_param_stride_bh, *kz = st.k_zero + unit * st.k_param_stride_bh;
        const T *exact = reinterpret_cast<const T *>(st.k_res) + unit * st.res_stride_bh;
        uint32_t cur[N][W];   // codes of the tile to decode; each is replaced by the next tile's once it is used
        float4 ns[2], nz[2];  // its scales and zeros
        auto here = [&](int t) { return t < min(t_hi, tiles_packed) && t * kTile + w * kGroup < st.n_quant; };
        auto fetch_codes = [&](int t, int i) {
            const uint8_t *src = codes + ((int64_t)t * kTile + w * kGroup + TPL * i + sub) * RB + chunk * SB;
            if constexpr (SB == 8) {
                const uint2 v = __ldg(reinterpret_cast<const uint2 *>(src));
                cur[i][0] = v.x; cur[i][1] = v.y;
            } else if constexpr (SB == 4) cur[i][0] = __ldg(reinterpret_cast<const uint32_t *>(src));
            else cur[i][0] = __ldg(reinterpret_cast<const uint16_t *>(src));
        };
        auto fetch_params = [&](int t) {
            const int64_t at = ((int64_t)t * (kTile / kGroup) + w) * D + 8 * chunk;
            const float4 *s4 = reinterpret_cast<const float4 *>(ks + at), *z4 = reinterpret_cast<const float4 *>(kz + at);
            ns[0] = __ldg(s4); ns[1] = __ldg(s4 + 1);
            nz[0] = __ldg(z4); nz[1] = __ldg(z4 + 1);
        };
        if (here(t_lo)) {
            fetch_params(t_lo);
#pragma unroll
            for (int i = 0; i < N; ++i) fetch_codes(t_lo, i);
        }
        // (token k of this lane is row 32 w + TPL k + sub: its chunk's place turns with the row modulo 8)
        const uint32_t at0 = L::at(w * kGroup + sub, chunk);
        auto place = [&](int stage, int k) { return smem + L::K + stage * L::TILE + ((at0 ^ ((TPL * k & 7) << 4)) + TPL * k * 128); };
        if (warp == 8 && elect_one()) {
            for (int i = 0; i < kBars; ++i) {
                const bool by_warps = i < kKEmpty || (i >= kVFull && i < kVEmpty) || (i >= kPReady && i < kPVHalf);
                mbar_init(bar(i), by_warps ? 4 : 1);
            }
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        if (n_tiles == 0) ready();
        for (int i = 0; i < n_tiles; ++i) {
            const int t = t_lo + i, stage = i & 1;
            if (t < tiles_packed) {
                const bool some = here(t), more = here(t + 1);
                float2 sc[4], ze[4];
                uint32_t sh[4], zh[4];
                if constexpr (HALF) {
                    const float s8[8] = {ns[0].x, ns[0].y, ns[0].z, ns[0].w, ns[1].x, ns[1].y, ns[1].z, ns[1].w};
                    const float z8[8] = {nz[0].x, nz[0].y, nz[0].z, nz[0].w, nz[1].x, nz[1].y, nz[1].z, nz[1].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) { sh[k] = pack_f16(s8[k], s8[k + 4]); zh[k] = pack_f16(z8[k], z8[k + 4]); }
                } else {
                    sc[0] = {ns[0].x, ns[0].y}; sc[1] = {ns[0].z, ns[0].w}; sc[2] = {ns[1].x, ns[1].y}; sc[3] = {ns[1].z, ns[1].w};
                    const float2 zz[4] = {{nz[0].x, nz[0].y}, {nz[0].z, nz[0].w}, {nz[1].x, nz[1].y}, {nz[1].z, nz[1].w}};
#pragma unroll
                    for (int k = 0; k < 4; ++k) ze[k] = fma2(make_float2(-Codes<SB>::kBase, -Codes<SB>::kBase), sc[k], zz[k]);
                }
                if (more) fetch_params(t + 1);
                if (i >= 2 && !wait(kKEmpty + stage, ((i >> 1) - 1) & 1)) break;
                if (some) {
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        if constexpr (HALF) *reinterpret_cast<uint4 *>(place(stage, k)) = decode8_half<SB>(cur[k][0], sh, zh);
                        else *reinterpret_cast<uint4 *>(place(stage, k)) = decode8<SB>(cur[k], sc, ze);
                        if (more) fetch_codes(t + 1, k);
                    }
                } else {
#pragma unroll 1
                    for (int k = 0; k < N; ++k) *reinterpret_cast<uint4 *>(place(stage, k)) = zero4();
                }
            } else {
                if (i >= 2 && !wait(kKEmpty + stage, ((i >> 1) - 1) & 1)) break;
                const int r0 = (t - tiles_packed) * kTile + w * kGroup;
#pragma unroll 2
                for (int k = 0; k < N; ++k) {
                    const int row = r0 + TPL * k + sub;
                    uint4 v = zero4();
                    if (row < st.n_res) {
                        v = __ldg(reinterpret_cast<const uint4 *>(exact + (int64_t)row * D) + chunk);
                        v = in_order<HALF>(make_uint4(as_f16x2<T>(v.x), as_f16x2<T>(v.y), as_f16x2<T>(v.z), as_f16x2<T>(v.w)));
                    }
                    *reinterpret_cast<uint4 *>(place(stage, k)) = v;
                }
            }
            if (i == 0) ready();  // (the first tile needs nothing of the others)
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(kKFull + stage));
        }
    } else if (warp < 16) {
        fewer_registers<HALF>();
        // ---- values: a thread decodes one 32-channel group (one scale, one zero) of a token ------------
        constexpr int GV = D / kGroup;            // value groups of a token = threads of a token
        constexpr int TPI = 128 / GV;             // tokens the four warps cover at once
        constexpr int N = kTile / TPI;            // tokens a thread decodes
        constexpr int W = SB;                     // words of 32 codes
        // (D = 128: the eight lanes of a quarter-warp store to eight different 16-byte columns)
        const int grp = D == 128 ? (lane & 1) | (lane >> 2 & 2) : lane & 1;
        const int tok = (warp - 12) * (32 / GV) + (D == 128 ? (lane >> 1 & 3) | (lane >> 2 & 4) : lane >> 1);
        const uint8_t *codes = st.v_codes + unit * st.v_codes_stride_bh;
        const float *vs = st.v_scale + unit * st.v_param_stride_bh, *vz = st.v_zero + unit * st.v_param_stride_bh;
        const T *exact = reinterpret_cast<const T *>(st.v_res) + unit * st.res_stride_bh;
        uint32_t cur[N][W];   // as for the keys
        float sc[N], ze[N];
        auto here = [&](int t, int i) { return t < min(t_hi, tiles_packed) && t * kTile + i * TPI + tok < st.n_quant; };
        auto fetch = [&](int t, int i) {
            const int64_t slot = (int64_t)t * kTile + i * TPI + tok;
            const uint8_t *src = codes + slot * RB + grp * (4 * SB);
            if constexpr (W == 2) {
                const uint2 v = __ldg(reinterpret_cast<const uint2 *>(src));
                cur[i][0] = v.x; cur[i][1] = v.y;
            } else {
#pragma unroll
                for (int j = 0; j < W; j += 4) {
                    const uint4 v = __ldg(reinterpret_cast<const uint4 *>(src) + j / 4);
                    cur[i][j] = v.x; cur[i][j + 1] = v.y; cur[i][j + 2] = v.z; cur[i][j + 3] = v.w;
                }
            }
            sc[i] = __ldg(vs + slot * GV + grp);
            ze[i] = __ldg(vz + slot * GV + grp);
        };
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (here(t_lo, i)) fetch(t_lo, i);
        // (row k TPI + tok, chunk 4 grp + j: TPI is a multiple of 8, so only j moves the place)
        const uint32_t at0 = L::at(tok, 4 * grp);
        auto place = [&](int stage, int k, int j) { return smem + L::V + stage * L::TILE + ((at0 ^ (j << 4)) + k * TPI * 128); };
        if (n_tiles == 0) ready();
        for (int i = 0; i < n_tiles; ++i) {
            const int t = t_lo + i, stage = i & 1;
            if (t < tiles_packed) {
                if (i >= 2 && !wait(kVEmpty + stage, ((i >> 1) - 1) & 1)) break;
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    // (values of padding must not reach P V, where their weight is 0, as infinity or NaN)
                    const bool some = here(t, k) && t * kTile + k * TPI + tok >= first_slot;
                    const float sk = sc[k], zk = fmaf(-Codes<SB>::kBase, sc[k], ze[k]);
                    const float2 s8[4] = {{sk, sk}, {sk, sk}, {sk, sk}, {sk, sk}}, z8[4] = {{zk, zk}, {zk, zk}, {zk, zk}, {zk, zk}};
                    const uint32_t s2 = pack_f16(sc[k], sc[k]), z2 = pack_f16(ze[k], ze[k]);
                    const uint32_t sh[4] = {s2, s2, s2, s2}, zh[4] = {z2, z2, z2, z2};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t wd[SB == 8 ? 2 : 1];
                        if constexpr (SB == 8) { wd[0] = cur[k][2 * j]; wd[1] = cur[k][2 * j + 1]; }
                        else if constexpr (SB == 4) wd[0] = cur[k][j];
                        else wd[0] = cur[k][j / 2] >> (16 * (j & 1));
                        uint4 v;
                        if constexpr (HALF) v = decode8_half<SB>(wd[0], sh, zh);
                        else v = decode8<SB>(wd, s8, z8);
                        *reinterpret_cast<uint4 *>(place(stage, k, j)) = some ? v : zero4();
                    }
                    if (here(t + 1, k)) fetch(t + 1, k);
                }
            } else {
                if (i >= 2 && !wait(kVEmpty + stage, ((i >> 1) - 1) & 1)) break;
                const int r0 = (t - tiles_packed) * kTile;
#pragma unroll 1
                for (int k = 0; k < N; ++k) {
                    const int row = k * TPI + tok;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint4 v = zero4();
                        if (r0 + row < st.n_res && st.n_quant + r0 + row >= first_slot) {
                            v = __ldg(reinterpret_cast<const uint4 *>(exact + (int64_t)(r0 + row) * D) + 4 * grp + j);
                            v = in_order<HALF>(make_uint4(as_f16x2<T>(v.x), as_f16x2<T>(v.y), as_f16x2<T>(v.z), as_f16x2<T>(v.w)));
                        }
                        *reinterpret_cast<uint4 *>(place(stage, k, j)) = v;
                    }
                }
            }
            if (i == 0) ready();
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(kVFull + stage));
        }
    } else {
        // ---- the MMAs, all by one thread, in order ------------------------------------------------------
        // (the whole warp walks through the loop, so that descriptors stay in uniform registers)
        const bool elected = elect_one();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        ready();
        // (a descriptor's low word holds the address in 16-byte units: stages and k-steps are added to it)
        const uint64_t dq = make_desc(smem_u32(smem + L::Q), 16, 1024), dk = make_desc(smem_u32(smem + L::K), 16, 1024);
        const uint64_t dv = make_desc(smem_u32(smem + L::V), L::HALF, 1024);
        auto qk = [&](int j) {
            const int s = j & 1, t = two ? j >> 1 : j, stage = t & 1;
            if ((!two || s == 0) && !wait(kKFull + stage, (t >> 1) & 1)) return;
            fence_after();
            const uint64_t a = dq + (two ? s * (L::TILE >> 4) : 0), b = dk + stage * (L::TILE >> 4);
            const uint32_t d = tmem + 128 * s;
            if (elected) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t off = (uint32_t)((k >> 2) * L::HALF + (k & 3) * 32) >> 4;
                    mma_ss(d, a + off, b + off, make_idesc(kTile, false), k > 0);
                }
                mma_commit(bar(kSFull + s));
                if (!two || s == 1) mma_commit(bar(kKEmpty + stage));
            }
            __syncwarp();
        };
        auto pv = [&](int j) {
            const int s = j & 1, t = two ? j >> 1 : j, stage = t & 1;
            if ((!two || s == 0) && !wait(kVFull + stage, (t >> 1) & 1)) return;
            const uint64_t b = dv + stage * (L::TILE >> 4);
            const uint32_t d = tmem + 256 + 128 * s, a = tmem + 128 * s;
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {
                if (!wait(kPReady + 2 * s + half, (j >> 1) & 1)) return;
                fence_after();
                if (elected) {
#pragma unroll
                    for (int k = 0; k < kTile / 32; ++k)
                        mma_ts(d, a + 32 * half + 8 * k, b + half * (kTile / 2 * 128 >> 4) + k * (2048 >> 4), make_idesc(D, true), j >= 2 || half > 0 || k > 0);
                    if (half == 0) mma_commit(bar(kPVHalf + s));
                }
                __syncwarp();
            }
            if (elected) {
                if (!two || s == 1) mma_commit(bar(kVEmpty + stage));
                if (j + 2 >= n_steps) mma_commit(bar(kODone + s));
            }
            __syncwarp();
        };
#pragma unroll 1
        for (int j = -2; j < n_steps && !gave_up; ++j) {
            if (j >= 0) pv(j);
            if (j + 2 < n_steps && !gave_up) qk(j + 2);
        }
        if (gave_up) {  // MMAs in flight still use shared and tensor memory
            if (elected) mma_commit(bar(kDrain));
            __syncwarp();
            mbar_wait(bar(kDrain), 0);
        }
    }
    if (p.wait_test && tid == 0 && !mbar_wait(bar(kIdle), 0, 1u << 10)) gave_up = true;
    if (gave_up) atomicExch(&g_shared_timeout, 1);
    fence_before();
    __syncthreads();
    if (warp == 16) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

int tiles_of(const vq_kivi_rows &st) { return (int)(ceil_div(st.n_quant, kTile) + ceil_div(st.n_res, kTile)); }
int row_blocks_of(int64_t rows) { return (int)ceil_div(rows, rows > kTile ? 2 * kTile : kTile); }

// When `n1` CTAs of `d1` microseconds and then `n2` of `d2`, one an SM, are done
double done_after(int64_t n1, double d1, int64_t n2, double d2, int sms) {
    const int64_t rest = n1 % sms;                 // SMs that are busy d1 longer than the others
    const double t0 = (double)(n1 / sms) * d1, t1 = rest ? t0 + d1 : t0;
    if (n2 == 0) return t1;
    const double late = d1 / d2;
    for (int64_t k = std::max<int64_t>(1, (int64_t)std::min((double)n2 / (double)(sms - rest), ((double)n2 + (double)rest * late) / sms));; ++k)
        if ((sms - rest) * k + rest * std::max<int64_t>(0, (int64_t)((double)k - late)) >= n2) return std::max(t1, t0 + (double)k * d2);
}

template <int D, int SB, typename T>
int32_t launch(const TileParams &p, unsigned blocks, cudaStream_t st) {
    static std::atomic<uint64_t> allowed{0};
    const int32_t rc = allow_shared_memory(&shared_tiles_tc5_kernel<D, SB, T>, Layout<D>::BYTES, allowed);
    if (rc != VQ_OK) return rc;
    if constexpr (kHalfDecode<SB, T>) {
        static const int registers = [] {
            cudaFuncAttributes at;
            return cudaFuncGetAttributes(&at, &shared_tiles_tc5_kernel<D, SB, T>) == cudaSuccess ? at.numRegs : 0;
        }();
        VQ_REQUIRE(registers >= kLaunchRegisters, VQ_ERR_CUDA, "shared_tiles_tc5_kernel: compiled to %d registers, its warps share %d", registers, kLaunchRegisters);
    }
    int dev = 0;
    VQ_CHECK_CUDA(cudaGetDevice(&dev));
    if (!(g_launched.load(std::memory_order_relaxed) & device_bit(dev))) g_launched.fetch_or(device_bit(dev));
    shared_tiles_tc5_kernel<D, SB, T><<<blocks, kThreads, Layout<D>::BYTES, st>>>(p);
    VQ_CHECK_LAUNCH("shared_tiles_tc5_kernel");
    return VQ_OK;
}
template <int D, typename T>
int32_t launch_bits(int sb, const TileParams &p, unsigned blocks, cudaStream_t st) {
    if (sb == 2) return launch<D, 2, T>(p, blocks, st);
    if (sb == 4) return launch<D, 4, T>(p, blocks, st);
    return launch<D, 8, T>(p, blocks, st);
}

}  // namespace

// Splits of the parts along their tokens: the counts with the smallest estimate in microseconds. A CTA (one an
// SM) takes 3.0 a token tile and 13 for the rest with two row tiles, 3.2 and 16 with one. The SMs that the
// prefix leaves idle do `beside`, the own tokens' warp tiles, in SM microseconds, from 3 after its start; what
// is left of that comes behind, on all SMs. A partial record of a row costs 0.2 ns more (written here, read
// by the merge). Fitted to 105 calls of 32 to 8192 query rows behind 1K to 32K tokens that come from HBM, each
// measured at every split count of the prefix: the count chosen is 1.6 % slower than the best one in the mean.
void shared_tiles_tc5_splits(const Tc5Part &prefix, const Tc5Part &own, int D, int wanted, double beside, const DeviceInfo &di, int *prefix_splits, int *own_splits) {
    struct Side {
        int tiles;
        int64_t ctas, rows;
        double rest, step;
        int most;  // two waves, or four splits
        Side(const Tc5Part &p, int D, int sms)
            : tiles(p.st ? tiles_of(*p.st) : 0), ctas(p.st ? p.units * row_blocks_of(p.rows) : 0), rows(p.units * p.rows),
              rest(p.rows > kTile ? 13.0 : 16.0), step((p.rows > kTile ? 3.0 : 3.2) * (D == 128 ? 1.0 : 0.8)),
              most(ctas ? (int)std::min<int64_t>({(int64_t)tiles, 64, std::max<int64_t>(4, 2 * sms / ctas)}) : 0) {}
        double time(int s) const { return s ? rest + step * (double)ceil_div(tiles, s) : 0.0; }
    };
    const Side a(prefix, D, di.sm_count), b(own, D, di.sm_count);
    const int a_lo = !a.tiles ? 0 : wanted > 0 ? std::min({wanted, a.tiles, 64}) : 1, a_hi = wanted > 0 ? a_lo : a.most;
    double least = 1e30;
    for (int t = b.tiles ? 1 : 0; t <= std::min(b.most, 8); ++t) {
        const double bt = b.time(t);
        for (int s = a_lo; s <= a_hi; ++s) {
            const double at = a.time(s);
            double us = done_after(a.ctas * s, at, b.ctas * t, bt, di.sm_count) + 2e-4 * (double)(a.rows * s + b.rows * t) * D / 128;
            if (beside > 0.0) {
                const double idle = (double)(ceil_div(a.ctas * s, di.sm_count) * di.sm_count - a.ctas * s) * (at - 3.0);
                if (beside > idle) us += 1.4 + (beside - idle) / di.sm_count;
            }
            if (us < least) { least = us; *prefix_splits = s; *own_splits = t; }
        }
    }
}

int32_t shared_tiles_tc5_launch(const vq_shared_attend_args &a, const SharedPartials &parts, int prefix_splits, int own_splits, int own_record0,
                                cudaStream_t stream) {
    const int64_t per_req = (int64_t)(a.H_q / a.H_kv) * a.S_q;
    TileParams p = {};
    p.q = a.q;
    p.own_start = a.own_start;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.H_q = a.H_q; p.H_kv = a.H_kv; p.S_q = a.S_q; p.G = a.H_q / a.H_kv;
    p.causal = (a.flags & VQ_ATTEND_CAUSAL) != 0;
    p.parts = parts;
    p.wait_test = knob_take(VQ_KNOB_SHARED_WAIT_TEST);
    int64_t blocks = 0;
    auto part = [&](Part &t, const vq_kivi_rows &st, int64_t units, int64_t rows, int splits, int record0) {
        t.st = st;
        t.splits = std::max(splits, 1);
        t.rows = (int)rows;
        t.row_blocks = row_blocks_of(rows);
        t.tiles_packed = (int)ceil_div(st.n_quant, kTile);
        t.tiles = tiles_of(st);
        t.record0 = record0;
        const int64_t n = splits > 0 ? units * t.row_blocks * splits : 0;
        t.blocks = (int)std::min<int64_t>(n, INT32_MAX);
        blocks += n;
    };
    part(p.prefix, a.prefix, a.H_kv, a.B * per_req, prefix_splits, 0);
    part(p.own, a.own, (int64_t)a.B * a.H_kv, per_req, own_splits, own_record0);
    VQ_REQUIRE(blocks < (1ll << 31), VQ_ERR_SHAPE, "vq_kivi_shared_attend: too many query rows for one launch");
    const unsigned nb = (unsigned)blocks;
    if (a.dtype == VQ_F16) return a.D == 128 ? launch_bits<128, __half>(a.store_bits, p, nb, stream) : launch_bits<64, __half>(a.store_bits, p, nb, stream);
    return a.D == 128 ? launch_bits<128, __nv_bfloat16>(a.store_bits, p, nb, stream) : launch_bits<64, __nv_bfloat16>(a.store_bits, p, nb, stream);
}

int32_t shared_tiles_tc5_take_timeout(int *flag) {
    int dev = 0;
    *flag = 0;
    VQ_CHECK_CUDA(cudaGetDevice(&dev));
    if (!(g_launched.load() & device_bit(dev))) return VQ_OK;  // (a status call costs those who never launch it nothing)
    VQ_CHECK_CUDA(cudaDeviceSynchronize());
    const int zero = 0;
    VQ_CHECK_CUDA(cudaMemcpyFromSymbol(flag, g_shared_timeout, sizeof(int)));
    if (*flag) VQ_CHECK_CUDA(cudaMemcpyToSymbol(g_shared_timeout, &zero, sizeof(int)));
    return VQ_OK;
}

}  // namespace vq
