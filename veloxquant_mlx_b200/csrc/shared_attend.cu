// Attention of a batch that shares a packed prefix: entry point, the warp-tile kernel (every
// request's own tokens, and prefixes with few query rows) and the merge of the partial softmaxes.
//
//   out = softmax(scale q [K_p | K_b]) [V_p | V_b]
//
// Both parts are attended apart, each split along its tokens, into partial records (m, l, o) that
// the merge kernel joins: o = sum_j 2^(m_j - M) o_j / sum_j 2^(m_j - M) l_j.
// The prefix is read once for all B * H_q/H_kv * S_q query rows of a kv head, the own tokens once per
// request. Many query rows go to the tcgen05 kernel of shared_tiles_tc5.cu, few to the warp tiles below.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "kivi_attend.h"
#include "shared_attend.h"

namespace vq {
namespace {

constexpr int kGroup = 32;
constexpr int kExact = 12;  // exact rows of one work item: as many bytes as a packed group of 4-bit codes
constexpr int kWarps = 4;
constexpr int kStages = 2;
// Weights, at most 1, are held times 2^7: float16's smallest step then is 2^-31 of the row's largest weight instead
// of 2^-24, so that many tokens behind one that outweighs them are not lost. The factor is in the exponent: the
// running maximum m is held 7 lower (8 at most where float32 rounds it; 15 could become 16, and 2^16 is no float16).
constexpr float kLift = 7.f;

struct RowsParams {
    const void *q;
    float scale_log2;  // scale * log2(e)
    const int32_t *own_start;
    int B, H_q, H_kv, S_q, G, causal;
    vq_kivi_rows prefix, own;
    SharedPartials parts;
    int np, no;                    // splits of the two parts
    int prefix_tiles, own_tiles;   // row tiles of a prefix unit (one per kv head) and of an own unit
    int prefix_blocks;             // blocks [0, prefix_blocks) work on the prefix, the rest on own tokens
};

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}
// 16 bytes from global to shared memory; zeros when `live` is false
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void lds(uint32_t (&w)[N], const uint8_t *p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 v = *reinterpret_cast<const uint4 *>(p + 4 * i);
            w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
        }
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        w[0] = v.x; w[1] = v.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    }
}

// One stage of a warp's ring: a packed group (key codes | value codes | key scales | key zeros | value
// scales | value zeros) or 12 exact rows (keys | values).
template <int D, int SB>
struct Stage {
    static constexpr int RB = D * SB / 8, GV = D / kGroup;
    static constexpr int KC = 0, VC = KC + kGroup * RB, KS = VC + kGroup * RB, KZ = KS + 4 * D, VS = KZ + 4 * D, VZ = VS + kGroup * GV * 4;
    static constexpr int PACKED = VZ + kGroup * GV * 4;
    static constexpr int ROW = 2 * D, VR = kExact * ROW, EXACT = 2 * kExact * ROW;
    static constexpr int BYTES = PACKED > EXACT ? PACKED : EXACT;
    // Key scales and zeros: the four lanes of a quad read 16-byte chunks that are 128 (64) bytes apart: the
    // chunk's place in its 128-byte line is turned so that they fall on different banks.
    __device__ static __forceinline__ int param_chunk(int j) { return j ^ ((j >> 3) * (D == 128 ? 2 : 1)); }
    // Exact rows: chunk j of row r
    __device__ static __forceinline__ int row_chunk(int r, int j) { return r * ROW + ((j ^ (r & 7)) << 4); }
};

// One CTA: 8 or 16 query rows (NT tiles of 8) of one unit (kv head of the prefix, or kv head of one
// request's own store) over one split of its tokens. Tensor cores by m16n8k16 with tokens (QK^T) and
// channels (PV) on M and query rows on N: the own part has few rows (H_q/H_kv heads, a few drafted
// tokens), of which a tcgen05 tile of 128 would waste nearly all.
// Each warp takes work items in turn (a packed group of 32 tokens, or 12 exact rows), copied by cp.async
// into its own two-stage ring, so that an item is in flight while the one before is decoded; no
// synchronisation between warps until the end. The order of channels and of tokens inside an MMA is
// free: a lane's K fragments are one run of D/4 channels of a token, its V fragments one run of D/8
// channels, and the four tokens of a quad lie in rows whose banks differ.
// In bfloat16 codes are decoded in half precision, two at a time (see half_codes).
// Measured: 64 requests x 8 kv heads with 512 packed and 150 exact tokens (90 MB): 24.5 us = 3.7 TB/s, 57 % of
// the measured copy rate; bound by instruction issue (0.6 a clock and scheduler: about 700 instructions a packed
// group, 450 for twelve exact rows, and a prologue and epilogue per unit as long as four items), HBM at 41 %.
template <int D, int SB, typename T, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT > 1 ? 2 : SB == 8 ? 3 : 4)
shared_attend_rows_kernel(const __grid_constant__ RowsParams p) {
    using S = Stage<D, SB>;
    constexpr int CH = D / 4, CN = D / 8, KS = D / 16;   // channels a lane owns for K, for V; k-steps of QK^T
    constexpr int MT = CN / 2;                           // 16-channel tiles of the output
    constexpr int KW = CH * SB / 32;                     // words of a lane's key codes of one token
    constexpr int VB = CN * SB;                          // bits of a lane's value codes of one token
    constexpr int VW = VB >= 32 ? VB / 32 : 1;
    constexpr int GV = S::GV, RB = S::RB;
    constexpr int ROWS = 8 * NT;
    constexpr float BASE = Codes<SB>::kBase;
    // codes through half precision (half_codes); a lane's channels 8 j + i of K then pair with 8 j + i + 4
    constexpr bool HALF = kHalfDecode<SB, T>;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float sh_m[kWarps][ROWS], sh_l[kWarps][ROWS];
    let_next_start();

    const int lane = threadIdx.x & 31;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int g8 = lane >> 2, c4 = lane & 3;
    const int tau = (g8 >> 1) | ((g8 & 1) << 2);         // token of row g8 of a key tile
    const bool is_prefix = (int)blockIdx.x < p.prefix_blocks;
    int blk = is_prefix ? blockIdx.x : blockIdx.x - p.prefix_blocks;
    const int ns = is_prefix ? p.np : p.no;
    const int n_tiles = is_prefix ? p.prefix_tiles : p.own_tiles;
    const int split = blk % ns; blk /= ns;
    const int tile = blk % n_tiles;
    const int unit = blk / n_tiles;                      // prefix: kv head; own: b * H_kv + kv head
    const int b_own = is_prefix ? 0 : unit / p.H_kv;
    const int hk = is_prefix ? unit : unit - b_own * p.H_kv;
    const vq_kivi_rows &st = is_prefix ? p.prefix : p.own;
    const int per_req = p.G * p.S_q;                     // query rows of one request and kv head
    const int n_rows = is_prefix ? p.B * per_req : per_req;
    auto out_row = [&](int r) {                          // output row (= row of q) of the unit's query row r
        const int b = is_prefix ? r / per_req : b_own, rem = is_prefix ? r - b * per_req : r;
        return ((int64_t)b * p.H_q + (int64_t)hk * p.G) * p.S_q + rem;
    };

    const int n_slots = st.n_quant + st.n_res;
    const int first_slot = is_prefix || !p.own_start ? 0 : min(n_slots, max(0, __ldg(p.own_start + b_own)));
    const int ng = st.n_quant / kGroup;                  // packed items; exact rows start at slot 32 * ng
    const int items = ng + (st.n_res + kExact - 1) / kExact;
    const int i_first = first_slot < st.n_quant ? first_slot / kGroup : ng + (first_slot - st.n_quant) / kExact;
    const int per_split = (items - i_first + ns - 1) / ns;
    const int i_lo = min(items, i_first + split * per_split), i_hi = min(items, i_lo + per_split);

    uint8_t *ring = smem + warp * (kStages * S::BYTES);
    const uint32_t ring_u32 = (uint32_t)__cvta_generic_to_shared(ring);
    const uint8_t *kc = st.k_codes + unit * st.k_codes_stride_bh, *vc = st.v_codes + unit * st.v_codes_stride_bh;
    const float *ks = st.k_scale + unit * st.k_param_stride_bh, *kz = st.k_zero + unit * st.k_param_stride_bh;
    const float *vs = st.v_scale + unit * st.v_param_stride_bh, *vz = st.v_zero + unit * st.v_param_stride_bh;
    const T *kr = reinterpret_cast<const T *>(st.k_res) + unit * st.res_stride_bh;
    const T *vr = reinterpret_cast<const T *>(st.v_res) + unit * st.res_stride_bh;

    // Values of slots before first_slot and of rows behind the last enter the ring as zeros, so that
    // whatever is stored there cannot reach the output (their scores are dropped below).
    auto fetch = [&](int item, int stage) {
        const uint32_t dst = ring_u32 + stage * S::BYTES;
        if (item < ng) {
            const int64_t slot0 = (int64_t)item * kGroup;
            const uint8_t *k0 = kc + slot0 * RB, *v0 = vc + slot0 * RB;
#pragma unroll
            for (int j = lane; j < kGroup * RB / 16; j += 32) {
                copy16(dst + S::KC + 16 * j, k0 + 16 * j, true);
                copy16(dst + S::VC + 16 * j, v0 + 16 * j, true);
            }
            const float *s0 = ks + (int64_t)item * D, *z0 = kz + (int64_t)item * D;
            if (D == 128 || lane < 16) {
                copy16(dst + S::KS + 16 * S::param_chunk(lane), s0 + 4 * lane, true);
                copy16(dst + S::KZ + 16 * S::param_chunk(lane), z0 + 4 * lane, true);
                // (a 16-byte chunk holds the scales of one token (D = 128) or two; a padding token that
                // shares a chunk with a live one is dealt with where values are decoded)
                const bool live = slot0 + (4 * lane + 3) / GV >= first_slot;
                copy16(dst + S::VS + 16 * lane, vs + slot0 * GV + 4 * lane, live);
                copy16(dst + S::VZ + 16 * lane, vz + slot0 * GV + 4 * lane, live);
            }
        } else {
            const int r0 = (item - ng) * kExact;
#pragma unroll
            for (int j = lane; j < kExact * (D / 8); j += 32) {
                const int r = j / (D / 8), ch = j % (D / 8);
                const bool in = r0 + r < st.n_res, seen = in && st.n_quant + r0 + r >= first_slot;
                const int64_t at = in ? (int64_t)(r0 + r) * D + 8 * ch : 0;
                copy16(dst + S::row_chunk(r, ch), kr + at, in);
                copy16(dst + S::VR + S::row_chunk(r, ch), vr + at, seen);
            }
        }
    };

    // Q: row g8 of each tile, channels c4*CH ..
    uint32_t qb[NT][CH / 2];
    int lim[NT][2];  // first slot that rows 2*c4 and 2*c4 + 1 of a tile do not see
    if (i_lo + warp < i_hi) fetch(i_lo + warp, 0);
    asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = tile * ROWS + 8 * nt + g8;
#pragma unroll
        for (int i = 0; i < CH / 2; ++i) qb[nt][i] = 0u;
        if (r < n_rows) {
            const uint4 *src = reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(p.q) + out_row(r) * D + c4 * CH);
#pragma unroll
            for (int i = 0; i < CH / 8; ++i) {
                const uint4 v = __ldg(src + i);
                const uint4 w = in_order<HALF>(make_uint4(as_f16x2<T>(v.x), as_f16x2<T>(v.y), as_f16x2<T>(v.z), as_f16x2<T>(v.w)));
                qb[nt][4 * i] = w.x; qb[nt][4 * i + 1] = w.y; qb[nt][4 * i + 2] = w.z; qb[nt][4 * i + 3] = w.w;
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int rr = tile * ROWS + 8 * nt + 2 * c4 + i;
            lim[nt][i] = rr >= n_rows ? 0 : is_prefix || !p.causal ? n_slots : n_slots - p.S_q + rr % p.S_q + 1;
        }
    }

    int all_see = INT_MAX;  // slots that every live row sees need no mask
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (tile * ROWS + 8 * nt + 2 * c4 + i < n_rows) all_see = min(all_see, lim[nt][i]);
    all_see = __reduce_min_sync(0xffffffffu, all_see);

    float o[NT][MT][4] = {};
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) { m[nt][0] = m[nt][1] = -INFINITY; l[nt][0] = l[nt][1] = 0.f; }

    // Scores s[tile][2 * (16-token tile)...] of one item to weights: masks, running maxima, rescale of o.
    // Returns the weights as B fragments of the item's 16-token steps.
    auto softmax = [&](auto steps_c, float (&s)[NT][2][4], int slot0, uint32_t (&pb)[NT][2][2]) {
        constexpr int STEPS = decltype(steps_c)::value;
        const int end = STEPS == 1 ? slot0 + kExact : INT_MAX;  // (the last rows of an exact tile are not there)
        const bool all_seen = STEPS == 2 && slot0 >= first_slot && slot0 + kGroup <= all_see;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float mx[2] = {-INFINITY, -INFINITY};
            if (all_seen) {
#pragma unroll
                for (int k = 0; k < STEPS; ++k)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        s[nt][k][c] = __fmul_rn(s[nt][k][c], p.scale_log2);  // (rounded here: the maximum and the weights see the same)
                        mx[c & 1] = fmaxf(mx[c & 1], s[nt][k][c]);
                    }
            } else {
#pragma unroll
                for (int k = 0; k < STEPS; ++k)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int slot = slot0 + 16 * k + 8 * (c >> 1) + tau;
                        s[nt][k][c] = slot >= first_slot && slot < min(lim[nt][c & 1], end) ? __fmul_rn(s[nt][k][c], p.scale_log2) : -INFINITY;
                        mx[c & 1] = fmaxf(mx[c & 1], s[nt][k][c]);
                    }
            }
            float base[2], f[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], d));
                const float mn = fmaxf(m[nt][i], mx[i] - kLift);
                base[i] = mn == -INFINITY ? 0.f : mn;
                f[i] = ex2(m[nt][i] - base[i]);
                m[nt][i] = mn;
                l[nt][i] *= f[i];
            }
            if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
                for (int j = 0; j < MT; ++j) { o[nt][j][0] *= f[0]; o[nt][j][1] *= f[1]; o[nt][j][2] *= f[0]; o[nt][j][3] *= f[1]; }
            }
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                float e[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    e[c] = ex2(s[nt][k][c] - base[c & 1]);
                    l[nt][c & 1] += e[c];
                }
                pb[nt][k][0] = transpose8x8(pack_f16(e[0], e[1]));
                pb[nt][k][1] = transpose8x8(pack_f16(e[2], e[3]));
            }
        }
    };

    int stage = 0;
    for (int item = i_lo + warp; item < i_hi; item += kWarps, stage ^= 1) {
        if (item + kWarps < i_hi) fetch(item + kWarps, stage ^ 1);
        asm volatile("cp.async.commit_group;" ::: "memory");
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        const uint8_t *buf = ring + stage * S::BYTES;
        float s[NT][2][4] = {};
        uint32_t pb[NT][2][2];
        if (item < ng) {
            // ---- S^T = K Q^T: rows of a key tile are tokens tau(g8), 8 + tau(g8) ----------------------
            uint32_t w[4][KW];
#pragma unroll
            for (int j = 0; j < 4; ++j) lds(w[j], buf + S::KC + (8 * j + tau) * RB + c4 * (CH * SB / 8));
            auto qk = [&](int k, const uint32_t (&a)[4][2]) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma16816(s[nt][0], a[0][0], a[1][0], a[0][1], a[1][1], qb[nt][2 * k], qb[nt][2 * k + 1]);
                    mma16816(s[nt][1], a[2][0], a[3][0], a[2][1], a[3][1], qb[nt][2 * k], qb[nt][2 * k + 1]);
                }
            };
            if constexpr (HALF) {
#pragma unroll
                for (int k = 0; k < KS; k += 2) {  // eight channels: pairs (0, 4) (1, 5) to one MMA, (2, 6) (3, 7) to the next
                    float4 sc[2], ze[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int at = 16 * S::param_chunk(c4 * (CH / 4) + k + i);
                        sc[i] = *reinterpret_cast<const float4 *>(buf + S::KS + at);
                        ze[i] = *reinterpret_cast<const float4 *>(buf + S::KZ + at);
                    }
                    const uint32_t sh[4] = {pack_f16(sc[0].x, sc[1].x), pack_f16(sc[0].y, sc[1].y), pack_f16(sc[0].z, sc[1].z), pack_f16(sc[0].w, sc[1].w)};
                    const uint32_t zh[4] = {pack_f16(ze[0].x, ze[1].x), pack_f16(ze[0].y, ze[1].y), pack_f16(ze[0].z, ze[1].z), pack_f16(ze[0].w, ze[1].w)};
                    uint32_t a[2][4][2];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t word = SB == 4 ? w[j][k / 2] : __byte_perm(w[j][k / 4], 0u, k / 2 % 2 ? 0x4342 : 0x4140);
                        const uint32_t w8 = word >> 8;
#pragma unroll
                        for (int i = 0; i < 4; ++i) a[i >> 1][j][i & 1] = hfma2(half_codes<SB>(word, w8, i), sh[i], zh[i]);
                    }
                    qk(k, a[0]);
                    qk(k + 1, a[1]);
                }
            } else {
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    const int at = 16 * S::param_chunk(c4 * (CH / 4) + k);
                    const float4 sc = *reinterpret_cast<const float4 *>(buf + S::KS + at), zz = *reinterpret_cast<const float4 *>(buf + S::KZ + at);
                    const float2 s0 = make_float2(sc.x, sc.y), s1 = make_float2(sc.z, sc.w), nb = make_float2(-BASE, -BASE);
                    const float2 z0 = fma2(nb, s0, make_float2(zz.x, zz.y)), z1 = fma2(nb, s1, make_float2(zz.z, zz.w));
                    uint32_t a[4][2];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t word = w[j][4 * k / Codes<SB>::kPerWord];
                        const int i0 = 4 * k % Codes<SB>::kPerWord;
                        const float2 x = fma2(make_float2(Codes<SB>::get(word, i0), Codes<SB>::get(word, i0 + 1)), s0, z0);
                        const float2 y = fma2(make_float2(Codes<SB>::get(word, i0 + 2), Codes<SB>::get(word, i0 + 3)), s1, z1);
                        a[j][0] = pack_f16(x.x, x.y);
                        a[j][1] = pack_f16(y.x, y.y);
                    }
                    qk(k, a);
                }
            }
            const int slot0 = item * kGroup;
            softmax(std::integral_constant<int, 2>{}, s, slot0, pb);
            // ---- O^T += V^T P^T: a quad's tokens of a step are c4, c4 + 4, c4 + 8, c4 + 12 -------------
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t x[4][VW];
                float2 sc[4], ze[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int tok = 16 * k + 4 * t + c4;
                    const uint8_t *src = buf + S::VC + tok * RB + g8 * (VB / 8);
                    if constexpr (VB == 16) x[t][0] = *reinterpret_cast<const uint16_t *>(src);
                    else lds(x[t], src);
                    const int at = 4 * (tok * GV + g8 * CN / kGroup);
                    float a = *reinterpret_cast<const float *>(buf + S::VS + at), z = *reinterpret_cast<const float *>(buf + S::VZ + at);
                    if (D == 64 && slot0 + tok < first_slot) a = z = 0.f;
                    if constexpr (!HALF) z = fmaf(-BASE, a, z);
                    sc[t] = make_float2(a, a);
                    ze[t] = make_float2(z, z);
                }
                auto pv = [&](int j, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {  // channels 2j, 2j + 1 of the four tokens
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][j], a0, a1, a2, a3, pb[nt][k][0], pb[nt][k][1]);
                };
                if constexpr (HALF) {
                    // a half of two tokens' words side by side: their codes of a channel are a pair
                    const uint32_t s01 = pack_f16(sc[0].x, sc[1].x), s23 = pack_f16(sc[2].x, sc[3].x), z01 = pack_f16(ze[0].x, ze[1].x), z23 = pack_f16(ze[2].x, ze[3].x);
                    constexpr int PER = 16 / SB;  // codes of a half word
#pragma unroll
                    for (int j = 0; j < CN; j += PER) {
                        const uint32_t sel = j / PER % 2 ? 0x7632 : 0x5410;
                        const uint32_t y01 = __byte_perm(x[0][j / (2 * PER)], x[1][j / (2 * PER)], sel), y23 = __byte_perm(x[2][j / (2 * PER)], x[3][j / (2 * PER)], sel);
                        uint32_t v01[PER], v23[PER];
#pragma unroll
                        for (int i = 0; i < PER; ++i) {
                            // (2 bits: codes 4-7 of a half lie in its upper byte)
                            const uint32_t a = SB == 2 && i >= 4 ? y01 >> 8 : y01, b = SB == 2 && i >= 4 ? y23 >> 8 : y23;
                            v01[i] = hfma2(half_codes<SB>(a, a >> 8, i & 3), s01, z01);
                            v23[i] = hfma2(half_codes<SB>(b, b >> 8, i & 3), s23, z23);
                        }
#pragma unroll
                        for (int i = 0; i < PER; i += 2) pv((j + i) / 2, v01[i], v01[i + 1], v23[i], v23[i + 1]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < MT; ++j) {
                        float2 v[4];
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            const uint32_t word = x[t][2 * j / Codes<SB>::kPerWord];
                            const int i0 = 2 * j % Codes<SB>::kPerWord;
                            v[t] = fma2(make_float2(Codes<SB>::get(word, i0), Codes<SB>::get(word, i0 + 1)), sc[t], ze[t]);
                        }
                        pv(j, pack_f16(v[0].x, v[1].x), pack_f16(v[0].y, v[1].y), pack_f16(v[2].x, v[3].x), pack_f16(v[2].y, v[3].y));
                    }
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < CH / 8; ++i) {
                uint32_t a[2][4];
                lds(a[0], buf + S::row_chunk(tau, c4 * (CH / 8) + i));
                lds(a[1], buf + S::row_chunk(min(8 + tau, kExact - 1), c4 * (CH / 8) + i));
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint4 x = in_order<HALF>(make_uint4(as_f16x2<T>(a[j][0]), as_f16x2<T>(a[j][1]), as_f16x2<T>(a[j][2]), as_f16x2<T>(a[j][3])));
                    a[j][0] = x.x; a[j][1] = x.y; a[j][2] = x.z; a[j][3] = x.w;
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma16816(s[nt][0], a[0][0], a[1][0], a[0][1], a[1][1], qb[nt][4 * i], qb[nt][4 * i + 1]);
                    mma16816(s[nt][0], a[0][2], a[1][2], a[0][3], a[1][3], qb[nt][4 * i + 2], qb[nt][4 * i + 3]);
                }
            }
            softmax(std::integral_constant<int, 1>{}, s, st.n_quant + (item - ng) * kExact, pb);
#pragma unroll
            for (int i = 0; i < CN / 8; ++i) {
                uint32_t x[kExact / 4][4];
#pragma unroll
                for (int t = 0; t < kExact / 4; ++t) {
                    lds(x[t], buf + S::VR + S::row_chunk(4 * t + c4, g8 * (CN / 8) + i));
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[t][k] = as_f16x2<T>(x[t][k]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t a0 = __byte_perm(x[0][j], x[1][j], 0x5410), a1 = __byte_perm(x[0][j], x[1][j], 0x7632);
                    const uint32_t a2 = x[2][j] & 0xffffu, a3 = x[2][j] >> 16;  // (rows 12 to 15 are zero)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][4 * i + j], a0, a1, a2, a3, pb[nt][0][0], pb[nt][0][1]);
                }
            }
        }
        __syncwarp();  // the stage is read before it is refilled
    }

    // ---- the four warps' partials into one record per row (the rings are done with) ----------------
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    constexpr int LD = D + 4;
    float *sh_o = reinterpret_cast<float *>(smem);  // [warp][row][channel]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], d);
            const int r = 8 * nt + 2 * c4 + i;
            if (g8 == 0) { sh_m[warp][r] = m[nt][i]; sh_l[warp][r] = l[nt][i]; }
            float *dst = sh_o + (warp * ROWS + r) * LD + g8 * CN;
#pragma unroll
            for (int j = 0; j < MT; ++j) *reinterpret_cast<float2 *>(dst + 2 * j) = make_float2(o[nt][j][i], o[nt][j][2 + i]);
        }
    __syncthreads();
    const int slot_of = (is_prefix ? 0 : p.np) + split;
    for (int i = threadIdx.x; i < ROWS * D / 4; i += kWarps * 32) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        if (tile * ROWS + r >= n_rows) break;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sh_m[w][r]);
        const float bs = mm == -INFINITY ? 0.f : mm;
        float ll = 0.f, acc[4] = {};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = ex2(sh_m[w][r] - bs);
            ll = fmaf(sh_l[w][r], f, ll);
            const float4 v = *reinterpret_cast<const float4 *>(sh_o + (w * ROWS + r) * LD + d);
            acc[0] = fmaf(v.x, f, acc[0]); acc[1] = fmaf(v.y, f, acc[1]); acc[2] = fmaf(v.z, f, acc[2]); acc[3] = fmaf(v.w, f, acc[3]);
        }
        const int64_t rec = out_row(tile * ROWS + r) * p.parts.n_splits + slot_of;
        *reinterpret_cast<float4 *>(p.parts.o + rec * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (d == 0) *reinterpret_cast<float2 *>(p.parts.ml + rec * 2) = make_float2(mm, ll);
    }
    // The merge waits for this kernel alone: it must not end before the tcgen05 kernel does. (One block waits: the
    // others make room.)
    if (blockIdx.x == gridDim.x - 1) wait_for_previous();
}

template <int D, int SB, typename T, int NT>
int32_t launch_rows(const RowsParams &p, unsigned blocks, bool dependent, cudaStream_t st) {
    constexpr int ring = kWarps * kStages * Stage<D, SB>::BYTES, merge = kWarps * 8 * NT * (D + 4) * 4;
    constexpr int smem = ring > merge ? ring : merge;
    static std::atomic<uint64_t> allowed{0};
    const int32_t rc = allow_shared_memory(&shared_attend_rows_kernel<D, SB, T, NT>, smem, allowed);
    if (rc != VQ_OK) return rc;
    return launch_dependent(&shared_attend_rows_kernel<D, SB, T, NT>, "shared_attend_rows_kernel", blocks, kWarps * 32, smem, st, dependent, p);
}

// Joins the records of an output row: `ways` warps (1 or 4) take its records in turn, each lane D/32
// channels; every warp has all of the row's (m, l) in its lanes. Bound by latency (a few KB a row, from
// L2), so eight records are asked for at a time, the first eight together with the (m, l).
constexpr int kMaxRecords = 128;  // 64 splits of either part

template <int D, typename T>
__global__ void __launch_bounds__(128) shared_attend_merge_kernel(const SharedPartials parts, int64_t rows, int ways, T *__restrict__ out, float *__restrict__ lse) {
    constexpr int C = D / 32, AHEAD = 8;
    using V = typename std::conditional<C == 4, float4, float2>::type;
    __shared__ float sh[4][D];
    __shared__ float sh_w[4][kMaxRecords];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part = warp % ways;
    const int64_t row = (int64_t)blockIdx.x * (4 / ways) + warp / ways;
    const int n = parts.n_splits;
    float ll = 0.f, mm = -INFINITY, acc[C] = {};
    wait_for_previous();
    if (row < rows) {
        const float2 *ml = reinterpret_cast<const float2 *>(parts.ml) + row * n;
        const V *po = reinterpret_cast<const V *>(parts.o + row * n * D) + lane;
        V v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (part + i * ways < n) v[i] = po[(int64_t)(part + i * ways) * 32];
        float2 r[kMaxRecords / 32];
#pragma unroll
        for (int i = 0; i < kMaxRecords / 32; ++i) {
            r[i] = 32 * i + lane < n ? ml[32 * i + lane] : make_float2(-INFINITY, 0.f);
            mm = fmaxf(mm, r[i].x);
        }
        mm = warp_max(mm);
        const float bs = mm == -INFINITY ? 0.f : mm;
#pragma unroll
        for (int i = 0; i < kMaxRecords / 32; ++i) {
            const float f = ex2(r[i].x - bs);  // the record's weight
            ll = fmaf(r[i].y, f, ll);
            sh_w[warp][32 * i + lane] = f;
        }
        ll = warp_sum(ll);
        __syncwarp();
        for (int j0 = part;; ) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                if (j0 + i * ways >= n) break;
                const float f = sh_w[warp][j0 + i * ways];
                const float *e = reinterpret_cast<const float *>(&v[i]);
#pragma unroll
                for (int c = 0; c < C; ++c) acc[c] = fmaf(e[c], f, acc[c]);
            }
            j0 += AHEAD * ways;
            if (j0 >= n) break;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                if (j0 + i * ways < n) v[i] = po[(int64_t)(j0 + i * ways) * 32];
        }
    }
    if (ways > 1) {
#pragma unroll
        for (int c = 0; c < C; ++c) sh[warp][lane * C + c] = acc[c];
        __syncthreads();
        if (warp != 0) return;
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] = (sh[0][lane * C + c] + sh[1][lane * C + c]) + (sh[2][lane * C + c] + sh[3][lane * C + c]);
    }
    if (row >= rows) return;
    const float inv = ll > 0.f ? 1.f / ll : ll == 0.f ? 0.f : ll;  // nothing seen: zeros; NaN stays
    alignas(8) T res[C];
#pragma unroll
    for (int c = 0; c < C; ++c) res[c] = from_f32<T>(acc[c] * inv);
    using O = typename std::conditional<C == 4, uint2, uint32_t>::type;
    reinterpret_cast<O *>(out + row * D)[lane] = *reinterpret_cast<const O *>(res);
    if (lse && lane == 0) lse[row] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * 0.6931471805599453f;
}

struct Plan {
    int prefix_tc5, own_tc5;  // splits of the parts that the tcgen05 kernel takes (0: it does not)
    int np, no;               // partial records of the two parts
    int row_tile;             // query rows of a warp tile: 8 or 16
    int prefix_tiles, own_tiles;
    int64_t rows;
};

int32_t plan_of(const vq_shared_attend_args &a, const DeviceInfo &di, Plan *out) {
    Plan pl = {};
    const int64_t per_req = (int64_t)(a.H_q / a.H_kv) * a.S_q, all = a.B * per_req;
    pl.rows = (int64_t)a.B * a.H_q * a.S_q;
    const vq_kivi_rows &pre = a.prefix, &own = a.own;
    const int ip = pre.n_quant / kGroup + (int)ceil_div(pre.n_res, kExact), io = own.n_quant / kGroup + (int)ceil_div(own.n_res, kExact);
    // The tcgen05 kernel decodes a token once for 128 or 256 query rows, the warp tiles for 8 or 16, but it
    // takes 5 us longer to start and end. Measured with 8 kv heads, warp tiles / tcgen05 in us: 64 rows
    // behind 1K tokens 10.3 / 12.2, 2K 13.9 / 12.8, 8K 28.7 / 16.7; 256 behind 512: 18.6 / 15.6; 32 behind 2K
    // 9.6 / 12.4, 4K 11.8 / 13.4, 8K 19.6 / 16.1; 16 behind 32K 27.1 / 30.3; own tokens, 1 request of 256 rows
    // over 662: 22.5 / 16.7; 8 of 36 over 662: 26.5 / 19.9. It masks scores before it multiplies them, so it takes
    // positive scales alone (-inf * 0 is NaN; the warp tiles mask the product).
    auto pays = [&](int64_t units, int64_t rows, const vq_kivi_rows &st) {
        return rows >= 32 && (double)units * (double)rows * ((double)st.n_quant + st.n_res) >= (rows < 64 && units < 32 ? 2 << 20 : 1 << 20);
    };
    const bool can = a.scale * 1.4426950408889634f > 0.f;
    VQ_REQUIRE(a.variant != 2 || (can && ip), VQ_ERR_SHAPE, "vq_kivi_shared_attend: the tcgen05 kernel needs a prefix and a positive scale");
    const int64_t units = (int64_t)a.B * a.H_kv;
    const bool prefix_tc5 = can && ip && (a.variant == 2 || (a.variant == 0 && pays(a.H_kv, all, pre)));
    const bool own_tc5 = can && io && (a.variant == 2 ? per_req > 32 : a.variant == 0 && pays(units, per_req, own));
    pl.row_tile = (prefix_tc5 ? per_req : all) > 8 ? 16 : 8;
    pl.prefix_tiles = (int)ceil_div(all, pl.row_tile);
    pl.own_tiles = (int)ceil_div(per_req, pl.row_tile);
    auto splits = [&](int64_t tiles, int items) {
        // As many CTAs as fit the GPU at once, but at least two work items a warp (512 units of 26 items: 1 split
        // 25 us, 2 28 us, 4 33 us), or one while every CTA has an SM to itself (8 units of 14 items: 2 splits 8.3 us, 4
        // 6.9, 8 6.9, 16 7.5; of 32: 4 splits 6.6, 8 5.6, 16 5.8).
        const int64_t few = ceil_div(items, 2 * kWarps), more = std::min(ceil_div(items, kWarps), (int64_t)di.sm_count / tiles);
        return (int)std::max<int64_t>(1, std::min<int64_t>({(int64_t)di.sm_count * 4 / tiles, std::max<int64_t>(few, more), 64}));
    };
    if (io && !own_tc5) pl.no = splits(units * pl.own_tiles, io);
    if (ip && !prefix_tc5) pl.np = a.n_splits > 0 ? std::min({a.n_splits, ip, 64}) : splits((int64_t)a.H_kv * pl.prefix_tiles, ip);
    if (prefix_tc5 || own_tc5) {
        // An SM full of warp tiles does an item a warp in 0.5 us for each block; to start and end takes three items.
        double beside = 0.0;
        if (io && !own_tc5)
            beside = 0.5 * (pl.row_tile == 16 ? 1.2 : 1.0) * (a.D == 128 ? 1.0 : 0.85) * (double)(units * pl.own_tiles * pl.no) * ((double)ceil_div(io, pl.no * kWarps) + 3.0);
        shared_tiles_tc5_splits({prefix_tc5 ? &pre : nullptr, a.H_kv, all}, {own_tc5 ? &own : nullptr, units, per_req}, a.D, a.n_splits, beside, di, &pl.prefix_tc5, &pl.own_tc5);
        if (prefix_tc5) pl.np = pl.prefix_tc5;
        if (own_tc5) pl.no = pl.own_tc5;
    }
    *out = pl;
    return VQ_OK;
}

int32_t validate(const vq_shared_attend_args &a) {
    const char *fn = "vq_kivi_shared_attend";
    VQ_REQUIRE(a.B >= 1 && a.H_q >= 1 && a.H_kv >= 1 && a.S_q >= 1 && a.H_q % a.H_kv == 0, VQ_ERR_SHAPE,
               "%s: B, H_q, H_kv, S_q must be >= 1 and H_q=%d a multiple of H_kv=%d", fn, a.H_q, a.H_kv);
    VQ_REQUIRE(a.dtype == VQ_F16 || a.dtype == VQ_BF16, VQ_ERR_DTYPE, "%s: float16 or bfloat16 expected", fn);
    VQ_REQUIRE(a.D == 64 || a.D == 128, VQ_ERR_SHAPE, "%s: D=%d must be 64 or 128", fn, a.D);
    VQ_REQUIRE(a.group == kGroup, VQ_ERR_SHAPE, "%s: group=%d must be 32", fn, a.group);
    VQ_REQUIRE(a.store_bits == 2 || a.store_bits == 4 || a.store_bits == 8, VQ_ERR_SHAPE, "%s: store_bits=%d must be 2, 4 or 8", fn, a.store_bits);
    VQ_REQUIRE((a.flags & ~VQ_ATTEND_CAUSAL) == 0 && a.variant >= 0 && a.variant <= 2 && a.n_splits >= 0, VQ_ERR_SHAPE,
               "%s: unknown flags (%d), variant (%d) or n_splits (%d)", fn, a.flags, a.variant, a.n_splits);
    VQ_REQUIRE((int64_t)a.B * a.H_q < (1ll << 31) && (int64_t)a.B * a.H_q * a.S_q < (1ll << 31), VQ_ERR_SHAPE, "%s: too many query rows", fn);
    VQ_REQUIRE(a.q && a.out, VQ_ERR_SHAPE, "%s: q/out is NULL", fn);
    VQ_REQUIRE(is_aligned(a.q, 16) && is_aligned(a.out, 16), VQ_ERR_ALIGN, "%s: q and out must be 16-byte aligned", fn);
    for (const vq_kivi_rows *s : {&a.prefix, &a.own}) {
        const char *which = s == &a.prefix ? "prefix" : "own";
        VQ_REQUIRE(s->n_quant >= 0 && s->n_res >= 0 && s->n_quant % kGroup == 0, VQ_ERR_SHAPE, "%s: %s: n_quant=%d must be a multiple of 32 and n_res=%d not negative",
                   fn, which, s->n_quant, s->n_res);
        VQ_REQUIRE((int64_t)s->n_quant + s->n_res < (1ll << 31) - 256, VQ_ERR_SHAPE, "%s: %s: too many tokens", fn, which);
        if (s->n_quant) {
            VQ_REQUIRE(s->k_codes && s->v_codes && s->k_scale && s->k_zero && s->v_scale && s->v_zero, VQ_ERR_SHAPE, "%s: %s: a packed tensor is NULL", fn, which);
            VQ_REQUIRE(is_aligned(s->k_codes, 16) && is_aligned(s->v_codes, 16) && is_aligned(s->k_scale, 16) && is_aligned(s->k_zero, 16) &&
                           is_aligned(s->v_scale, 16) && is_aligned(s->v_zero, 16) && s->k_codes_stride_bh % 16 == 0 && s->v_codes_stride_bh % 16 == 0 &&
                           s->k_param_stride_bh % 4 == 0 && s->v_param_stride_bh % 4 == 0,
                       VQ_ERR_ALIGN, "%s: %s: packed tensors and their slabs must be 16-byte aligned", fn, which);
        }
        if (s->n_res) {
            VQ_REQUIRE(s->k_res && s->v_res, VQ_ERR_SHAPE, "%s: %s: exact rows are NULL", fn, which);
            VQ_REQUIRE(is_aligned(s->k_res, 16) && is_aligned(s->v_res, 16) && s->res_stride_bh % 8 == 0, VQ_ERR_ALIGN, "%s: %s: exact rows must be 16-byte aligned", fn, which);
        }
    }
    return VQ_OK;
}

int64_t workspace_of(const Plan &pl, int D) { return pl.rows * (pl.np + pl.no) * ((int64_t)D + 2) * (int64_t)sizeof(float); }

template <int D, typename T>
int32_t launch_all(const vq_shared_attend_args &a, const Plan &pl, const DeviceInfo &di, cudaStream_t st) {
    RowsParams p = {};
    p.q = a.q;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.own_start = a.own_start;
    p.B = a.B; p.H_q = a.H_q; p.H_kv = a.H_kv; p.S_q = a.S_q; p.G = a.H_q / a.H_kv;
    p.causal = (a.flags & VQ_ATTEND_CAUSAL) != 0;
    p.prefix = a.prefix;
    p.own = a.own;
    p.np = pl.np; p.no = pl.no;
    p.parts.n_splits = pl.np + pl.no;
    p.parts.o = (float *)a.workspace;
    p.parts.ml = p.parts.o + pl.rows * p.parts.n_splits * D;
    p.prefix_tiles = pl.prefix_tiles;
    p.own_tiles = pl.own_tiles;
    const bool tc5 = pl.prefix_tc5 || pl.own_tc5;
    const int64_t pb = pl.prefix_tc5 ? 0 : (int64_t)pl.np * pl.prefix_tiles * a.H_kv;
    const int64_t blocks = pb + (pl.own_tc5 ? 0 : (int64_t)pl.no * pl.own_tiles * a.B * a.H_kv);
    VQ_REQUIRE(blocks < (1ll << 31), VQ_ERR_SHAPE, "vq_kivi_shared_attend: too many query rows for one launch");
    p.prefix_blocks = (int)pb;
    if (tc5) {
        const int32_t rc = shared_tiles_tc5_launch(a, p.parts, pl.prefix_tc5, pl.own_tc5, pl.np, st);
        if (rc != VQ_OK) return rc;
    }
    if (blocks) {
        // (behind the tcgen05 kernel: its blocks take the SMs that kernel leaves, then those where it is done)
        const bool wide = pl.row_tile == 16;
        const unsigned nb = (unsigned)blocks;
        int32_t rc;
        if (a.store_bits == 2) rc = wide ? launch_rows<D, 2, T, 2>(p, nb, tc5, st) : launch_rows<D, 2, T, 1>(p, nb, tc5, st);
        else if (a.store_bits == 4) rc = wide ? launch_rows<D, 4, T, 2>(p, nb, tc5, st) : launch_rows<D, 4, T, 1>(p, nb, tc5, st);
        else rc = wide ? launch_rows<D, 8, T, 2>(p, nb, tc5, st) : launch_rows<D, 8, T, 1>(p, nb, tc5, st);
        if (rc != VQ_OK) return rc;
    }
    const int ways = p.parts.n_splits > 8 ? 4 : 1;
    return launch_dependent(&shared_attend_merge_kernel<D, T>, "shared_attend_merge_kernel", (unsigned)ceil_div(pl.rows * ways, 4), 128, 0, st,
                            tc5 || blocks > 0, p.parts, pl.rows, ways, (T *)a.out, a.lse);
}

}  // namespace
}  // namespace vq

extern "C" int64_t vq_kivi_shared_attend_workspace_bytes(const vq_shared_attend_args *args) {
    using namespace vq;
    if (!args || validate(*args) != VQ_OK) return 0;
    DeviceInfo di;
    if (device_info(&di) != VQ_OK) { di.sm_count = 148; di.smem_optin = 227 * 1024; }
    Plan pl;
    if (plan_of(*args, di, &pl) != VQ_OK) return 0;
    return workspace_of(pl, args->D) + 16;
}

extern "C" int32_t vq_kivi_shared_attend(const vq_shared_attend_args *args, void *stream) {
    using namespace vq;
    VQ_REQUIRE(args != nullptr, VQ_ERR_SHAPE, "vq_kivi_shared_attend: args is NULL");
    const vq_shared_attend_args &a = *args;
    int32_t rc = validate(a);
    if (rc != VQ_OK) return rc;
    DeviceInfo di;
    rc = device_info(&di);
    if (rc != VQ_OK) return rc;
    Plan pl;
    rc = plan_of(a, di, &pl);
    if (rc != VQ_OK) return rc;
    const int64_t need = workspace_of(pl, a.D);
    VQ_REQUIRE(need == 0 || (a.workspace != nullptr && a.workspace_bytes >= need), VQ_ERR_CAPACITY,
               "vq_kivi_shared_attend: workspace of %lld bytes needed, %lld given", (long long)need, (long long)a.workspace_bytes);
    VQ_REQUIRE(is_aligned(a.workspace, 16), VQ_ERR_ALIGN, "vq_kivi_shared_attend: workspace must be 16-byte aligned");
    cudaStream_t st = (cudaStream_t)stream;
    if (a.dtype == VQ_F16) return a.D == 128 ? launch_all<128, __half>(a, pl, di, st) : launch_all<64, __half>(a, pl, di, st);
    return a.D == 128 ? launch_all<128, __nv_bfloat16>(a, pl, di, st) : launch_all<64, __nv_bfloat16>(a, pl, di, st);
}
