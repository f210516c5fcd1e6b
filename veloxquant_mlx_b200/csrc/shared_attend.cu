// Attention of a batch that shares a packed prefix: entry point, the warp-tile kernel (every
// request's own tokens, and prefixes with few query rows) and the merge of the partial softmaxes.
//
//   out = softmax(scale q [K_p | K_b]) [V_p | V_b]
//
// Both parts are attended apart, each split along its tokens, into partial records (m, l, o) that
// the merge kernel joins: o = sum_j 2^(m_j - M) o_j / sum_j 2^(m_j - M) l_j.
// The prefix is read once for all B * H_q/H_kv * S_q query rows of a kv head (from 33 rows on by the
// tcgen05 kernel of shared_prefix_tc5.cu), the own tokens once per request.
#include <algorithm>
#include <type_traits>

#include "kivi_attend.h"
#include "shared_attend.h"

namespace vq {
namespace {

constexpr int kGroup = 32;
constexpr int kRowTile = 16;
constexpr int kWarps = 4;

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

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const void *p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p) + i / 4);
            w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
        }
    } else if constexpr (N == 2) {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
        w[0] = v.x; w[1] = v.y;
    } else {
        w[0] = __ldg(reinterpret_cast<const uint32_t *>(p));
    }
}

// One CTA: 16 query rows of one unit (kv head of the prefix, or kv head of one request's own store)
// over one split of its 32-token groups, four warps taking groups in turn. Tensor cores by
// m16n8k16 with query rows on M: 16 rows are what the own part has (H_q/H_kv heads, a few drafted
// tokens), a tile a tcgen05 MMA would leave seven eighths empty. Codes go straight from global
// memory to registers: the order of channels inside an MMA is free, so a thread's B fragment of
// QK^T is one contiguous run of D/4 channels of a token, and of PV a run of D/8 channels.
// Bound by HBM for few rows in principle; by instruction issue in practice (about 3 instructions a code).
template <int D, int SB, typename T>
__global__ void __launch_bounds__(kWarps * 32)
shared_attend_rows_kernel(const __grid_constant__ RowsParams p) {
    constexpr int CH = D / 4, CN = D / 8, KS = D / 16;   // channels a thread owns for K, for V; k-steps of QK^T
    constexpr int KW = CH * SB / 32;                     // words of a thread's key codes of one token
    constexpr int VB = CN * SB;                          // bits of a thread's value codes of one token
    constexpr int VW = VB >= 32 ? VB / 32 : 1;
    constexpr int GV = D / kGroup;
    __shared__ float sh_o[kWarps][kRowTile][D + 4];
    __shared__ float sh_m[kWarps][kRowTile], sh_l[kWarps][kRowTile];

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g8 = lane >> 2, l4 = lane & 3;
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

    const int64_t n_slots = (int64_t)st.n_quant + st.n_res;
    const int ng = st.n_quant / kGroup;                  // packed groups; exact rows start at slot 32 * ng
    const int groups = ng + (st.n_res + kGroup - 1) / kGroup;
    const int first_slot = is_prefix || !p.own_start ? 0 : max(0, __ldg(p.own_start + b_own));
    const int g_first = min(groups, first_slot / kGroup);
    const int per_split = (groups - g_first + ns - 1) / ns;
    const int g_lo = min(groups, g_first + split * per_split), g_hi = min(groups, g_lo + per_split);

    // this thread's two query rows: output row (= row of q), and the first slot that they do not see
    int64_t out_row[2];
    int lim[2];
    bool live[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = tile * kRowTile + g8 + 8 * i;
        live[i] = r < n_rows;
        const int rr = live[i] ? r : 0;
        const int b = is_prefix ? rr / per_req : b_own, rem = is_prefix ? rr - b * per_req : rr;
        out_row[i] = ((int64_t)b * p.H_q + (int64_t)hk * p.G) * p.S_q + rem;
        lim[i] = !live[i] ? 0 : is_prefix || !p.causal ? (int)n_slots : (int)n_slots - p.S_q + rem % p.S_q + 1;
    }

    // Q: row g8 (+8), channels l4*CH ..
    uint32_t qa[KS][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t w[CH / 2] = {};
        if (live[i]) load_words(w, reinterpret_cast<const T *>(p.q) + out_row[i] * D + l4 * CH);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            qa[k][i] = as_f16x2<T>(w[2 * k]);
            qa[k][2 + i] = as_f16x2<T>(w[2 * k + 1]);
        }
    }

    float o[CN][4] = {};
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const uint8_t *kc = st.k_codes + unit * st.k_codes_stride_bh, *vc = st.v_codes + unit * st.v_codes_stride_bh;
    const float *ks = st.k_scale + unit * st.k_param_stride_bh, *kz = st.k_zero + unit * st.k_param_stride_bh;
    const float *vs = st.v_scale + unit * st.v_param_stride_bh, *vz = st.v_zero + unit * st.v_param_stride_bh;
    const T *kr = reinterpret_cast<const T *>(st.k_res) + unit * st.res_stride_bh;
    const T *vr = reinterpret_cast<const T *>(st.v_res) + unit * st.res_stride_bh;

    for (int grp = g_lo + warp; grp < g_hi; grp += kWarps) {
        const bool packed = grp < ng;
        const int slot0 = grp * kGroup;
        float s[4][4] = {};
        // ---- S = Q K^T -----------------------------------------------------------------------
        if (packed) {
            uint32_t w[4][KW];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                load_words(w[j], kc + (int64_t)(slot0 + 8 * j + g8) * (D * SB / 8) + l4 * (CH * SB / 8));
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const float4 sc = __ldg(reinterpret_cast<const float4 *>(ks + (int64_t)grp * D + l4 * CH + 4 * k));
                const float4 ze = __ldg(reinterpret_cast<const float4 *>(kz + (int64_t)grp * D + l4 * CH + 4 * k));
                const float z0 = fmaf(-Codes<SB>::kBase, sc.x, ze.x), z1 = fmaf(-Codes<SB>::kBase, sc.y, ze.y);
                const float z2 = fmaf(-Codes<SB>::kBase, sc.z, ze.z), z3 = fmaf(-Codes<SB>::kBase, sc.w, ze.w);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t word = w[j][4 * k / Codes<SB>::kPerWord];
                    const int i0 = 4 * k % Codes<SB>::kPerWord;
                    const uint32_t b0 = pack_f16(fmaf(Codes<SB>::get(word, i0), sc.x, z0), fmaf(Codes<SB>::get(word, i0 + 1), sc.y, z1));
                    const uint32_t b1 = pack_f16(fmaf(Codes<SB>::get(word, i0 + 2), sc.z, z2), fmaf(Codes<SB>::get(word, i0 + 3), sc.w, z3));
                    mma16816(s[j], qa[k], b0, b1);
                }
            }
        } else {
            const int row0 = slot0 - ng * kGroup;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t w[CH / 2] = {};
                const int row = row0 + 8 * j + g8;
                if (row < st.n_res) load_words(w, kr + (int64_t)row * D + l4 * CH);
#pragma unroll
                for (int k = 0; k < KS; ++k) mma16816(s[j], qa[k], as_f16x2<T>(w[2 * k]), as_f16x2<T>(w[2 * k + 1]));
            }
        }
        // ---- softmax: scores outside [first_slot, lim) are dropped whatever they are ------------
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int slot = slot0 + 8 * j + 2 * l4 + (c & 1);
                s[j][c] = slot >= first_slot && slot < lim[c >> 1] ? s[j][c] * p.scale_log2 : -INFINITY;
                mx[c >> 1] = fmaxf(mx[c >> 1], s[j][c]);
            }
        float base[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
            const float mn = fmaxf(m[i], mx[i]);
            base[i] = mn == -INFINITY ? 0.f : mn;
            const float alpha = ex2(m[i] - base[i]);
            m[i] = mn;
            l[i] *= alpha;
#pragma unroll
            for (int j = 0; j < CN; ++j) { o[j][2 * i] *= alpha; o[j][2 * i + 1] *= alpha; }
        }
        uint32_t pa[2][4];  // P as A fragments of the two 16-token steps
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float e[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                e[c] = ex2(s[j][c] - base[c >> 1]);
                l[c >> 1] += e[c];
            }
            pa[j >> 1][(j & 1) * 2] = pack_f16(e[0], e[1]);
            pa[j >> 1][(j & 1) * 2 + 1] = pack_f16(e[2], e[3]);
        }
        // ---- O += P V: slots before first_slot may hold anything; their values enter as 0 --------
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            if (packed) {
                uint32_t w[4][VW];
                float sc[4], ze[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int64_t slot = slot0 + 16 * kk + 2 * l4 + (t & 1) + 8 * (t >> 1);
                    const uint8_t *src = vc + slot * (D * SB / 8) + g8 * (VB / 8);
                    if constexpr (VB == 16) w[t][0] = __ldg(reinterpret_cast<const uint16_t *>(src));
                    else load_words(w[t], src);
                    const int64_t pi = slot * GV + g8 * CN / kGroup;
                    const bool dead = slot < first_slot;
                    sc[t] = dead ? 0.f : __ldg(vs + pi);
                    ze[t] = dead ? 0.f : fmaf(-Codes<SB>::kBase, sc[t], __ldg(vz + pi));
                }
#pragma unroll
                for (int j = 0; j < CN; ++j) {
                    float v[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        v[t] = fmaf(Codes<SB>::get(w[t][j / Codes<SB>::kPerWord], j % Codes<SB>::kPerWord), sc[t], ze[t]);
                    mma16816(o[j], pa[kk], pack_f16(v[0], v[1]), pack_f16(v[2], v[3]));
                }
            } else {
                uint32_t w[4][CN / 2];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int slot = slot0 + 16 * kk + 2 * l4 + (t & 1) + 8 * (t >> 1);
                    const int row = slot - ng * kGroup;
#pragma unroll
                    for (int i = 0; i < CN / 2; ++i) w[t][i] = 0u;
                    if (row < st.n_res && slot >= first_slot) load_words(w[t], vr + (int64_t)row * D + g8 * CN);
#pragma unroll
                    for (int i = 0; i < CN / 2; ++i) w[t][i] = as_f16x2<T>(w[t][i]);
                }
#pragma unroll
                for (int j = 0; j < CN; ++j) {
                    const uint32_t sel = j & 1 ? 0x7632u : 0x5410u;
                    mma16816(o[j], pa[kk], __byte_perm(w[0][j / 2], w[1][j / 2], sel), __byte_perm(w[2][j / 2], w[3][j / 2], sel));
                }
            }
        }
    }

    // ---- the four warps' partials into one record per row ----------------------------------------
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        const int r = g8 + 8 * i;
        if (l4 == 0) { sh_m[warp][r] = m[i]; sh_l[warp][r] = l[i]; }
#pragma unroll
        for (int j = 0; j < CN; ++j) {
            sh_o[warp][r][2 * l4 * CN + j] = o[j][2 * i];
            sh_o[warp][r][(2 * l4 + 1) * CN + j] = o[j][2 * i + 1];
        }
    }
    __syncthreads();
    const int slot_of = (is_prefix ? 0 : p.np) + split;
    for (int i = threadIdx.x; i < kRowTile * D / 4; i += kWarps * 32) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        const int rr = tile * kRowTile + r;
        if (rr >= n_rows) break;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sh_m[w][r]);
        const float bs = mm == -INFINITY ? 0.f : mm;
        float ll = 0.f, acc[4] = {};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = ex2(sh_m[w][r] - bs);
            ll = fmaf(sh_l[w][r], f, ll);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = fmaf(sh_o[w][r][d + c], f, acc[c]);
        }
        const int b = is_prefix ? rr / per_req : b_own, rem = is_prefix ? rr - b * per_req : rr;
        const int64_t rec = (((int64_t)b * p.H_q + (int64_t)hk * p.G) * p.S_q + rem) * p.parts.n_splits + slot_of;
        *reinterpret_cast<float4 *>(p.parts.o + rec * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (d == 0) *reinterpret_cast<float2 *>(p.parts.ml + rec * 2) = make_float2(mm, ll);
    }
}

// Joins the records of an output row: `ways` warps (1 or 4) take its records in turn, each lane D/32
// channels; every warp has all of the row's (m, l) in its lanes. Bound by latency (a few KB a row, from
// L2), so eight records are requested at a time.
constexpr int kMaxRecords = 128;  // 64 splits of either part

template <int D, typename T>
__global__ void __launch_bounds__(128) shared_attend_merge_kernel(const SharedPartials parts, int64_t rows, int ways, T *__restrict__ out, float *__restrict__ lse) {
    constexpr int C = D / 32;
    using V = typename std::conditional<C == 4, float4, float2>::type;
    __shared__ float sh[4][D];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part = warp % ways;
    const int64_t row = (int64_t)blockIdx.x * (4 / ways) + warp / ways;
    const int n = parts.n_splits;
    float ll = 0.f, mm = -INFINITY, acc[C] = {};
    if (row < rows) {
        const float2 *ml = reinterpret_cast<const float2 *>(parts.ml) + row * n;
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
            r[i].x = ex2(r[i].x - bs);  // the record's weight
            ll = fmaf(r[i].y, r[i].x, ll);
        }
        ll = warp_sum(ll);
        const V *po = reinterpret_cast<const V *>(parts.o + row * n * D) + lane;
#pragma unroll
        for (int i = 0; i < kMaxRecords / 32; ++i) {
            const int last = min(32, n - 32 * i);
#pragma unroll 8
            for (int j = part; j < last; j += ways) {
                const V v = po[(int64_t)(32 * i + j) * 32];
                const float f = __shfl_sync(0xffffffffu, r[i].x, j);
                const float *e = reinterpret_cast<const float *>(&v);
#pragma unroll
                for (int c = 0; c < C; ++c) acc[c] = fmaf(e[c], f, acc[c]);
            }
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
    bool tc5;
    int np, no;
    int prefix_tiles, own_tiles;
    int64_t rows;
};

int groups_of(const vq_kivi_rows &st) { return st.n_quant / kGroup + (st.n_res + kGroup - 1) / kGroup; }

int32_t plan_of(const vq_shared_attend_args &a, const DeviceInfo &di, Plan *out) {
    Plan pl = {};
    const int64_t per_req = (int64_t)(a.H_q / a.H_kv) * a.S_q;
    pl.rows = (int64_t)a.B * a.H_q * a.S_q;
    const int gp = groups_of(a.prefix), go = groups_of(a.own);
    const int64_t ctas = (int64_t)di.sm_count * 3;
    auto splits = [&](int64_t units, int groups) {
        // enough CTAs to fill the GPU, but at least two groups a warp
        return (int)std::max<int64_t>(1, std::min<int64_t>({ceil_div(ctas, units), ceil_div(groups, 2 * kWarps), 64}));
    };
    const char *why = shared_prefix_tc5_supported(a);
    VQ_REQUIRE(a.variant != 2 || why == nullptr, VQ_ERR_SHAPE, "vq_kivi_shared_attend: tcgen05 kernel unavailable: %s", why);
    pl.tc5 = gp > 0 && why == nullptr && a.variant != 1;
    pl.prefix_tiles = (int)ceil_div(a.B * per_req, kRowTile);
    pl.own_tiles = (int)ceil_div(per_req, kRowTile);
    pl.no = go ? splits((int64_t)a.B * a.H_kv * pl.own_tiles, go) : 0;
    pl.np = !gp ? 0 : pl.tc5 ? shared_prefix_tc5_splits(a, di) : a.n_splits > 0 ? std::min({a.n_splits, gp, 64}) : splits((int64_t)a.H_kv * pl.prefix_tiles, gp);
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
    VQ_REQUIRE((int64_t)a.B * a.H_q * a.S_q < (1ll << 31), VQ_ERR_SHAPE, "%s: too many query rows", fn);
    VQ_REQUIRE(a.q && a.out, VQ_ERR_SHAPE, "%s: q/out is NULL", fn);
    VQ_REQUIRE(is_aligned(a.q, 16) && is_aligned(a.out, 16), VQ_ERR_ALIGN, "%s: q and out must be 16-byte aligned", fn);
    for (const vq_kivi_rows *s : {&a.prefix, &a.own}) {
        const char *which = s == &a.prefix ? "prefix" : "own";
        VQ_REQUIRE(s->n_quant >= 0 && s->n_res >= 0 && s->n_quant % kGroup == 0, VQ_ERR_SHAPE, "%s: %s: n_quant=%d must be a multiple of 32 and n_res=%d not negative",
                   fn, which, s->n_quant, s->n_res);
        VQ_REQUIRE((int64_t)s->n_quant + s->n_res < (1ll << 31) - 64, VQ_ERR_SHAPE, "%s: %s: too many tokens", fn, which);
        if (s->n_quant) {
            VQ_REQUIRE(s->k_codes && s->v_codes && s->k_scale && s->k_zero && s->v_scale && s->v_zero, VQ_ERR_SHAPE, "%s: %s: a packed tensor is NULL", fn, which);
            VQ_REQUIRE(is_aligned(s->k_codes, 16) && is_aligned(s->v_codes, 16) && is_aligned(s->k_scale, 16) && is_aligned(s->k_zero, 16) &&
                           is_aligned(s->v_scale, 16) && is_aligned(s->v_zero, 16) && s->k_codes_stride_bh % 16 == 0 && s->v_codes_stride_bh % 16 == 0 &&
                           s->k_param_stride_bh % 4 == 0,
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
    const int64_t pb = pl.tc5 ? 0 : (int64_t)pl.np * pl.prefix_tiles * a.H_kv;
    const int64_t blocks = pb + (int64_t)pl.no * pl.own_tiles * a.B * a.H_kv;
    VQ_REQUIRE(blocks < (1ll << 31), VQ_ERR_SHAPE, "vq_kivi_shared_attend: too many query rows for one launch");
    p.prefix_blocks = (int)pb;
    if (pl.tc5) {
        const int32_t rc = shared_prefix_tc5_launch(a, p.parts, pl.np, di, st);
        if (rc != VQ_OK) return rc;
    }
    if (blocks) {
        if (a.store_bits == 2) shared_attend_rows_kernel<D, 2, T><<<(unsigned)blocks, kWarps * 32, 0, st>>>(p);
        else if (a.store_bits == 4) shared_attend_rows_kernel<D, 4, T><<<(unsigned)blocks, kWarps * 32, 0, st>>>(p);
        else shared_attend_rows_kernel<D, 8, T><<<(unsigned)blocks, kWarps * 32, 0, st>>>(p);
        VQ_CHECK_LAUNCH("shared_attend_rows_kernel");
    }
    const int ways = p.parts.n_splits > 8 ? 4 : 1;
    shared_attend_merge_kernel<D, T><<<(unsigned)ceil_div(pl.rows * ways, 4), 128, 0, st>>>(p.parts, pl.rows, ways, (T *)a.out, a.lse);
    VQ_CHECK_LAUNCH("shared_attend_merge_kernel");
    return VQ_OK;
}

}  // namespace
}  // namespace vq

extern "C" int64_t vq_kivi_shared_attend_workspace_bytes(const vq_shared_attend_args *args) {
    using namespace vq;
    if (!args || args->H_kv < 1 || args->H_q % args->H_kv || args->B < 1 || args->S_q < 1) return 0;
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
