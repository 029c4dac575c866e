// What ellm_attn_set_scores and ellm_attn_set_shared_prefix add to the attention kernels.
//
// Scores.  With t = q.k of a (row, key) pair the plain kernels use  scale * t.  Here
//     s = cap * tanh(scale * t / cap)            when a cap is set, else scale * t
//     s = s - slope[head] * |position - key|     when slopes are set
// and a row sees the keys of ONE interval [lo, hi):  lo = row_begin[sequence][position] (0 without
// that array),  hi = max(position + 1, prefix_lens[sequence]), never past the keys written so far.
// All of it is computed in log2 units (log2(e) folded into the constants), as the softmax is.
//
// Shared prefix.  The row's keys are `plen` rows of a second pair of K/V buffers, seen whole by every
// row of every sequence, followed by the sequence's own cache rows 0 ..= position.
//
// The tanh.  cap * tanh shifts an exponent, so what counts is the error of the product: relative to the
// score where the cap hardly bends it, absolute where it saturates.  Two forms, both odd polynomials
// (least-squares fits of P(u) / tanh(u) reweighted to equal ripple) near zero:
//   * any u: 4 terms for |u| < 1/4 (2.5e-9 off before fp32's own roundings), 1 - 2 / (1 + e^(2u)) beyond (1e-7 absolute);
//     two special-function operations per score;
//   * 6 terms for |u| <= 1 (relative error 6.1e-7: 6e-5 of an exponent at cap 128; five terms have 6.9e-6), on packed
//     pairs and without the special-function unit, which is what the chunk kernel is short of.  That kernel takes it
//     whenever 64 scores of each row of a warp are in range.
#pragma once
#include "common.cuh"

namespace ellm {

struct ScoreMods {
    float scale_log2 = 0.0f;               // scale * log2(e): without a cap
    float cap_in = 0.0f;                   // scale / cap
    float cap_log2 = 0.0f;                 // cap * log2(e); 0 = no cap
    const float* slopes = nullptr;         // [q_heads] or nullptr
    const int32_t* row_begin = nullptr;    // [max_batch][rb_stride] or nullptr
    long long rb_stride = 0;
    const int32_t* prefix_lens = nullptr;  // [max_batch] or nullptr
    long long max_seq = 0;
    const __nv_bfloat16* pk = nullptr;     // shared prefix: element (kv head, row, c) at h * ps1 + row * ps2 + c
    const __nv_bfloat16* pv = nullptr;
    long long ps1 = 0, ps2 = 0;
    long long plen = 0;
};

// The interval [lo, hi) of the row at position `pos` of sequence b, whose keys end at `end`.
__device__ __forceinline__ void row_interval(const ScoreMods& m, int b, long long pos, long long end, long long& lo, long long& hi) {
    hi = pos + 1;
    if (m.prefix_lens && pos >= 0) hi = max(hi, static_cast<long long>(m.prefix_lens[b]));
    hi = min(hi, end);
    lo = 0;
    if (m.row_begin && pos >= 0 && pos < m.max_seq) lo = max(0, m.row_begin[b * m.rb_stride + pos]);
}

__device__ __forceinline__ float fast_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// coefficients of u, u^3, ..., u^11 of the polynomial for |u| <= kTanhPolyMax
constexpr float kTanhPolyMax = 1.0f;
constexpr float kTanhC0 = 0.9999994040f, kTanhC1 = -0.3332904279f, kTanhC2 = 0.1328143328f, kTanhC3 = -0.0516056642f,
                kTanhC4 = 0.0167431068f, kTanhC5 = -0.0030670569f;
// tanh of any argument (saturates through e^(2u) = 0 and infinity; NaN stays NaN)
__device__ __forceinline__ float tanh_any(float u) {
    const float v = u * u;
    const float near_zero = u * (1.0f + v * (-0.3333320618f + v * (0.1332313269f + v * -0.0513277203f)));
    const float beyond = 1.0f - 2.0f * fast_rcp(1.0f + fast_exp2(u * (2.0f * kLog2e)));
    return v < 0.0625f ? near_zero : beyond;
}

// Score of one (row, key) pair in log2 units; `dist` = |position - key|, slope_log2 = slope * log2(e).
__device__ __forceinline__ float mod_score(const ScoreMods& m, float t, float slope_log2, float dist) {
    const float s = m.cap_log2 != 0.0f ? m.cap_log2 * tanh_any(t * m.cap_in) : t * m.scale_log2;
    return m.slopes ? s - slope_log2 * dist : s;
}

// One row by one warp, key by key, touching only the keys the row sees.  The tiled kernels multiply
// masked keys' V rows by a zero probability, and 0 * NaN (or infinity) is NaN: a row whose tiled result
// is not finite is recomputed here, so that what a masked key holds never shows.  If the row itself sees
// a NaN the result stays NaN (and the walk stops once every column is).  All 32 lanes call with the same
// arguments; lane = 4 consecutive channels.
__device__ __noinline__ void exact_row(const ScoreMods m, const __nv_bfloat16* q, const __nv_bfloat16* k, const __nv_bfloat16* v,
                                       long long s2, const __nv_bfloat16* pk, const __nv_bfloat16* pv, long long pos, long long lo,
                                       long long hi, float slope_log2, __nv_bfloat16* out, float* lse, int lane) {
    float qf[4];
    {
        const uint2 u = *reinterpret_cast<const uint2*>(q + lane * 4);
        const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
        const float2 c = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
        qf[0] = a.x; qf[1] = a.y; qf[2] = c.x; qf[3] = c.y;
    }
    float mx = -INFINITY, l = 0.0f, o[4] = {0.f, 0.f, 0.f, 0.f};
    const long long own = hi > lo ? hi - lo : 0;
    const long long total = m.plen + own;
    constexpr int kN = 4;   // keys requested together: the walk's time is that of its loads
    for (long long i = 0; i < total; i += kN) {
        uint2 uk[kN], uv[kN];
        float x[kN], p[kN];
#pragma unroll
        for (int n = 0; n < kN; ++n) {
            const long long at = min(i + n, total - 1);
            const bool pre = at < m.plen;
            const long long key = pre ? at : lo + (at - m.plen);
            uk[n] = *reinterpret_cast<const uint2*>((pre ? pk + key * m.ps2 : k + key * s2) + lane * 4);
            uv[n] = *reinterpret_cast<const uint2*>((pre ? pv + key * m.ps2 : v + key * s2) + lane * 4);
            if (i + n >= total) uv[n] = make_uint2(0u, 0u);
            x[n] = static_cast<float>(pos > key ? pos - key : key - pos);
        }
        float m_new = mx;
#pragma unroll
        for (int n = 0; n < kN; ++n) {
            const float2 ka = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&uk[n].x));
            const float2 kb = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&uk[n].y));
            float t = qf[0] * ka.x + qf[1] * ka.y + qf[2] * kb.x + qf[3] * kb.y;
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) t += __shfl_xor_sync(0xffffffffu, t, s);
            x[n] = i + n < total ? mod_score(m, t, slope_log2, x[n]) : -INFINITY;
            m_new = fmaxf(m_new, x[n]);
        }
        const float msub = m_new == -INFINITY ? 0.0f : m_new;
        const float corr = fast_exp2(mx - msub);
        mx = m_new;
        l *= corr;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] *= corr;
#pragma unroll
        for (int n = 0; n < kN; ++n) {
            const float2 va = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&uv[n].x));
            const float2 vb = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&uv[n].y));
            p[n] = fast_exp2(x[n] - msub);
            l += p[n];
            o[0] += p[n] * va.x;
            o[1] += p[n] * va.y;
            o[2] += p[n] * vb.x;
            o[3] += p[n] * vb.y;
        }
        if ((i & 63) == 60 && __all_sync(0xffffffffu, isnan(l) && isnan(o[0]) && isnan(o[1]) && isnan(o[2]) && isnan(o[3]))) break;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint2 r;
    r.x = pack_bf16(o[0] * inv, o[1] * inv);
    r.y = pack_bf16(o[2] * inv, o[3] * inv);
    *reinterpret_cast<uint2*>(out + lane * 4) = r;
    if (lse && lane == 0) *lse = l == 0.0f ? -INFINITY : (mx + log2f(l)) * kLn2;
}

}  // namespace ellm
