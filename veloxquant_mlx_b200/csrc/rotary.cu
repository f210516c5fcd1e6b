// Rotary positions: pairs of channels turned by position * frequency, forward and inverse, with an
// optional plain copy of a third tensor in the same launch (the append of a decode step).
//
//   t = p * turns[c]            (turns = frequency / 2 pi, 64 bits)
//   y_a = f (a cos 2 pi t - b sin 2 pi t),  y_b = f (b cos 2 pi t + a sin 2 pi t)
//
// Bound by HBM (every element is read and written once; 3 flops an element) or, for a decode step,
// by the launch. The angle must not be formed in 32 bits: at position 2^20 a float32 angle is off by
// up to 2^-5 of a radian. Here the turn count is a 64-bit product reduced to [-1/2, 1/2] in 64 bits
// (two instructions a pair), so that sincospif gets a small argument and needs no table.
// Measured: 4 x 8191 tokens, 40 heads of 128 in bfloat16, heads in [B, S, H, D] order: 110 us for 671 MB =
// 6.1 TB/s, 94 % of the measured copy rate; one token of 40 heads: 2.4 us; 64 tokens and the append: 3.1 us.
#include <algorithm>

#include "common.cuh"

namespace vq {
namespace {

constexpr int kThreads = 128;

struct RotaryParams {
    const char *x[3];
    char *y[3];
    int64_t xs[3][3], ys[3][3];  // bytes
    int h_end[3];                // heads of tensors 0..i together
    int heads_total;
    int S;
    int64_t n_tok;               // B * S
    int half, D;                 // pairs of a head; channels
    int units;                   // work units of a head (rotating, then copying)
    int rot_units;
    int head_lanes;              // threads that share the heads of one (token, unit)
    float sign, factor;
    const void *positions;
    int pos_bytes;
    int64_t pos_stride_b, pos_stride_s, pos_offset;
    const double *turns;
};

template <int BYTES>
struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = uint16_t; };

// One unit: V pairs of one head. Half layout: V channels from c and V from half + c; interleaved:
// 2V channels from 2c. A copying unit takes 2V channels behind the rotated part (V at the very end).
// A thread keeps its (token, unit) and walks over heads, so that the V sines and cosines are
// computed once for heads_total / head_lanes heads; neighbouring threads take neighbouring units,
// so that a warp reads whole rows.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
    using R = typename Raw<V * (int)sizeof(T)>::type;
    const int64_t item = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int per_tok = p.units * p.head_lanes;
    const int64_t tok = item / per_tok;
    if (tok >= p.n_tok) return;
    const int rest = (int)(item - tok * per_tok);
    const int hl = rest / p.units, u = rest - hl * p.units;
    const int64_t b = tok / p.S, s = tok - b * p.S;
    const bool rot = u < p.rot_units;
    // element offsets of the unit's two vectors inside a head
    int c0, c1;
    if (rot) {
        c0 = INTERLEAVED ? 2 * V * u : V * u;
        c1 = INTERLEAVED ? c0 + V : c0 + p.half;
    } else {
        c0 = 2 * p.half + 2 * V * (u - p.rot_units);
        c1 = c0 + V;
    }
    const bool two = c1 < p.D;
    float co[V], si[V];
    if (rot) {
        int64_t pos = p.pos_offset;
        if (p.positions) {
            const int64_t i = b * p.pos_stride_b + s * p.pos_stride_s;
            pos += p.pos_bytes == 8 ? __ldg((const long long *)p.positions + i) : (long long)__ldg((const int *)p.positions + i);
        } else {
            pos += s;
        }
        const double dp = (double)pos;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            double t = dp * __ldg(p.turns + V * u + i);
            t -= rint(t);
            sincospif(2.f * (float)t, &si[i], &co[i]);
            co[i] *= p.factor;
            si[i] *= p.sign;  // (factor, negated for the inverse)
        }
    }
    constexpr int U = V * sizeof(T) == 16 ? 4 : 2;  // heads in flight
    for (int h0 = hl; h0 < p.heads_total; h0 += U * p.head_lanes) {
        R ra[U], rb[U];
        char *out[U];
        bool turn[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int h = h0 + i * p.head_lanes;
            out[i] = nullptr;
            turn[i] = false;
            if (h < p.heads_total) {
                const int w = h < p.h_end[0] ? 0 : h < p.h_end[1] ? 1 : 2;
                const int64_t hh = w == 0 ? h : h - p.h_end[w - 1];
                const char *src = p.x[w] + b * p.xs[w][0] + hh * p.xs[w][1] + s * p.xs[w][2];
                out[i] = p.y[w] + b * p.ys[w][0] + hh * p.ys[w][1] + s * p.ys[w][2];
                turn[i] = rot && w < 2;
                ra[i] = *reinterpret_cast<const R *>(src + c0 * (int)sizeof(T));
                if (two) rb[i] = *reinterpret_cast<const R *>(src + c1 * (int)sizeof(T));
            }
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (out[i] == nullptr) continue;
            if (turn[i]) {
                alignas(16) T a[2 * V];
                *reinterpret_cast<R *>(a) = ra[i];
                *reinterpret_cast<R *>(a + V) = rb[i];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    T &ea = INTERLEAVED ? a[2 * j] : a[j];
                    T &eb = INTERLEAVED ? a[2 * j + 1] : a[V + j];
                    const float fa = to_f32<T>(ea), fb = to_f32<T>(eb);
                    ea = from_f32<T>(fa * co[j] - fb * si[j]);
                    eb = from_f32<T>(fb * co[j] + fa * si[j]);
                }
                ra[i] = *reinterpret_cast<R *>(a);
                rb[i] = *reinterpret_cast<R *>(a + V);
            }
            *reinterpret_cast<R *>(out[i] + c0 * (int)sizeof(T)) = ra[i];
            if (two) *reinterpret_cast<R *>(out[i] + c1 * (int)sizeof(T)) = rb[i];
        }
    }
}

template <typename T, int V>
void launch(const RotaryParams &p, bool interleaved, unsigned blocks, cudaStream_t st) {
    if (interleaved) rotary_kernel<T, V, true><<<blocks, kThreads, 0, st>>>(p);
    else rotary_kernel<T, V, false><<<blocks, kThreads, 0, st>>>(p);
}

}  // namespace
}  // namespace vq

extern "C" int32_t vq_rotary(const vq_rotary_args *args, void *stream) {
    using namespace vq;
    VQ_REQUIRE(args != nullptr, VQ_ERR_SHAPE, "vq_rotary: args is NULL");
    const vq_rotary_args &a = *args;
    VQ_REQUIRE(a.dtype >= 0 && a.dtype <= 2, VQ_ERR_DTYPE, "vq_rotary: unknown dtype %d", a.dtype);
    VQ_REQUIRE(a.B >= 0 && a.B < (1ll << 31) && a.S >= 0 && a.S < (1ll << 31) && a.D >= 2 && a.D <= 65536, VQ_ERR_SHAPE, "vq_rotary: bad sizes (B=%lld, S=%lld, D=%d)",
               (long long)a.B, (long long)a.S, a.D);
    VQ_REQUIRE(a.rotary_dim >= 2 && a.rotary_dim <= a.D && a.rotary_dim % 2 == 0, VQ_ERR_SHAPE,
               "vq_rotary: rotary_dim=%d must be even and in 2..D=%d", a.rotary_dim, a.D);
    VQ_REQUIRE(a.layout == 0 || a.layout == 1, VQ_ERR_SHAPE, "vq_rotary: layout must be 0 (half) or 1 (interleaved), got %d", a.layout);
    VQ_REQUIRE(a.positions == nullptr || a.pos_bytes == 4 || a.pos_bytes == 8, VQ_ERR_DTYPE, "vq_rotary: positions must be 4 or 8 bytes wide");
    VQ_REQUIRE(a.turns != nullptr, VQ_ERR_SHAPE, "vq_rotary: turns is NULL");
    RotaryParams p = {};
    const int64_t es = (int64_t)dtype_size(a.dtype);
    int64_t align = 16;  // the widest vector every address allows: 16 bytes or less
    auto fits = [&](int64_t bytes) {
        while (align > es && bytes % align) align >>= 1;
    };
    int64_t total = 0;
    for (int i = 0; i < 3; ++i) {
        const bool on = a.x[i] != nullptr;
        VQ_REQUIRE(!on || (a.y[i] != nullptr && a.heads[i] >= 0), VQ_ERR_SHAPE, "vq_rotary: tensor %d has no output or a negative head count", i);
        total += on ? a.heads[i] : 0;
        p.h_end[i] = (int)total;
        if (!on) continue;
        p.x[i] = (const char *)a.x[i];
        p.y[i] = (char *)a.y[i];
        VQ_REQUIRE((intptr_t)a.x[i] % es == 0 && (intptr_t)a.y[i] % es == 0, VQ_ERR_ALIGN, "vq_rotary: tensor %d is not aligned to its type", i);
        fits((int64_t)(intptr_t)a.x[i]);
        fits((int64_t)(intptr_t)a.y[i]);
        const int64_t size[3] = {a.B, a.heads[i], a.S};
        for (int j = 0; j < 3; ++j) {
            p.xs[i][j] = a.x_stride[i][j] * es;
            p.ys[i][j] = a.y_stride[i][j] * es;
            if (size[j] > 1) {
                fits(p.xs[i][j]);
                fits(p.ys[i][j]);
            }
        }
    }
    VQ_REQUIRE(total < (1 << 24), VQ_ERR_SHAPE, "vq_rotary: too many heads (%lld)", (long long)total);
    const int64_t n_tok = a.B * a.S;
    if (n_tok == 0 || total == 0) return VQ_OK;
    VQ_REQUIRE(n_tok < (1ll << 38), VQ_ERR_SHAPE, "vq_rotary: too many tokens (%lld)", (long long)n_tok);  // (more than a launch's threads)
    DeviceInfo di;
    int32_t rc = device_info(&di);
    if (rc != VQ_OK) return rc;
    // vector width: V elements, so that the halves (or the interleaved pairs) and the copied rest split evenly
    const int half = a.rotary_dim / 2;
    fits((a.layout ? (int64_t)a.rotary_dim / 2 : (int64_t)half) * es);
    fits((int64_t)(a.D - a.rotary_dim) * es);
    const int V = (int)(align / es);
    p.half = half;
    p.D = a.D;
    p.rot_units = half / V;
    p.units = p.rot_units + (int)ceil_div(a.D - a.rotary_dim, 2 * V);
    p.heads_total = (int)total;
    p.S = (int)a.S;
    p.n_tok = n_tok;
    p.factor = a.factor;
    p.sign = a.inverse ? -a.factor : a.factor;
    p.positions = a.positions;
    p.pos_bytes = a.pos_bytes;
    p.pos_stride_b = a.pos_stride_b;
    p.pos_stride_s = a.pos_stride_s;
    p.pos_offset = a.pos_offset;
    p.turns = a.turns;
    // Heads per thread: many where there are tokens enough to fill the GPU (the sines are shared), one
    // where there are not (a decode step is bound by its latency).
    const int64_t fill = (int64_t)di.sm_count * 1024;
    const int64_t lanes = std::min<int64_t>(total, std::max<int64_t>(ceil_div(total, 12), ceil_div(fill, n_tok * p.units)));
    p.head_lanes = (int)lanes;
    VQ_REQUIRE((double)n_tok * p.units * (double)lanes < (double)(1ll << 31) * (kThreads - 1), VQ_ERR_SHAPE, "vq_rotary: too many tokens (%lld)", (long long)n_tok);
    const int64_t blocks = ceil_div(n_tok * p.units * lanes, kThreads);
    cudaStream_t st = (cudaStream_t)stream;
    const bool il = a.layout == 1;
    const unsigned nb = (unsigned)blocks;
    if (a.dtype == VQ_F32) {
        if (V == 4) launch<float, 4>(p, il, nb, st);
        else if (V == 2) launch<float, 2>(p, il, nb, st);
        else launch<float, 1>(p, il, nb, st);
    } else if (a.dtype == VQ_F16) {
        if (V == 8) launch<__half, 8>(p, il, nb, st);
        else if (V == 4) launch<__half, 4>(p, il, nb, st);
        else if (V == 2) launch<__half, 2>(p, il, nb, st);
        else launch<__half, 1>(p, il, nb, st);
    } else {
        if (V == 8) launch<__nv_bfloat16, 8>(p, il, nb, st);
        else if (V == 4) launch<__nv_bfloat16, 4>(p, il, nb, st);
        else if (V == 2) launch<__nv_bfloat16, 2>(p, il, nb, st);
        else launch<__nv_bfloat16, 1>(p, il, nb, st);
    }
    VQ_CHECK_LAUNCH("rotary_kernel");
    return VQ_OK;
}
