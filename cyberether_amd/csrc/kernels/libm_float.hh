// libm_float.hh -- select-form (branch-free) restatement of the host libm's single-precision
// tanhf, for use inside gfx950 kernels.  No HIP dependency: the same text compiles for the host
// (tests/test_libm_float.py builds it with g++ and sweeps it against libm.so.6 bit for bit).
//
// Why: the Range module calls libm tanhf (src/domains/core/range/module_impl_native_cpu.cc:67-82).
// On the reference's CPU target (x86-64 glibc; this image ships 2.35) that is the FDLIBM float
// pair tanhf -> expm1f (Sun Microsystems' s_tanhf.c / s_expm1f.c as carried in glibc
// sysdeps/ieee754/flt-32), which is accurate to ~1 ulp but NOT correctly rounded, so only a
// restatement of the same operation sequence reproduces its bits.  The published algorithm is a
// ladder of data-dependent branches; on a 64-lane wavefront every lane would walk every taken
// branch, so all alternatives are computed and selected (v_cndmask), with identical arithmetic in
// the selected lane: one rounding per written operation, no FMA (-ffp-contract=off).
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define JST_FN __host__ __device__ __forceinline__
#else
#define JST_FN static inline
#endif

namespace jst::dev {

JST_FN uint32_t f2u(float f) { return __builtin_bit_cast(uint32_t, f); }
JST_FN float u2f(uint32_t u) { return __builtin_bit_cast(float, u); }

// expm1f(x) for the arguments tanhf feeds it: x = 2|a| with 1 <= |a| < 22, or x = -2|a| with
// 2^-55 <= |a| < 1.  (Other x produce an unspecified value that the caller discards.)
JST_FN float libm_expm1f_for_tanh(float x) {
    constexpr float ln2_hi = 6.9313812256e-01f, ln2_lo = 9.0580006145e-06f,
                    invln2 = 1.4426950216e+00f, Q1 = -3.3333335072e-02f, Q2 = 1.5873016091e-03f,
                    Q3 = -7.9365076090e-05f, Q4 = 4.0082177293e-06f, Q5 = -2.0109921195e-07f;
    const uint32_t bits = f2u(x);
    const uint32_t hx = bits & 0x7fffffffu;
    const bool neg = (bits >> 31) != 0;
    const bool red = hx > 0x3eb17218u;  // |x| > 0.5 ln2: argument reduction
    const bool mid = hx < 0x3F851592u;  // ... and |x| < 1.5 ln2: k = +-1

    const int32_t kg = (int32_t)(invln2 * x + (neg ? -0.5f : 0.5f));
    const float tg = (float)kg;
    const float hi_g = x - tg * ln2_hi, lo_g = tg * ln2_lo;
    const float hi_m = neg ? x + ln2_hi : x - ln2_hi;
    const float lo_m = neg ? -ln2_lo : ln2_lo;
    const float hi = mid ? hi_m : hi_g, lo = mid ? lo_m : lo_g;
    const int32_t k = red ? (mid ? (neg ? -1 : 1) : kg) : 0;
    const float xr_red = hi - lo;
    const float c_red = (hi - xr_red) - lo;
    const float xr = red ? xr_red : x;
    const float c = red ? c_red : 0.0f;

    const float hfx = 0.5f * xr;
    const float hxs = xr * hfx;
    const float r1 = 1.0f + hxs * (Q1 + hxs * (Q2 + hxs * (Q3 + hxs * (Q4 + hxs * Q5))));
    const float t = 3.0f - r1 * hfx;
    const float e = hxs * ((r1 - t) / (6.0f - xr * t));

    const float res_0 = xr - (xr * e - hxs);  // k == 0 (c is 0)
    float e2 = (xr * (e - c) - c);
    e2 -= hxs;
    const float res_m1 = 0.5f * (xr - e2) - 0.5f;
    const float res_p1 = (xr < -0.25f) ? -2.0f * (e2 - (xr + 0.5f)) : 1.0f + 2.0f * (xr - e2);
    const uint32_t kshift = (uint32_t)k << 23;  // "add k to y's exponent"
    const float d = e2 - xr;
    const float y_far = u2f(f2u(1.0f - d) + kshift) - 1.0f;  // k <= -2 or k > 56
    const float t_lo = u2f(0x3f800000u - (0x1000000u >> ((uint32_t)k & 31u)));  // 1 - 2^-k
    const float y_lo = u2f(f2u(t_lo - d) + kshift);                              // 2 <= k < 23
    const float t_hi = u2f((uint32_t)(0x7f - k) << 23);                          // 2^-k
    float y_hi = xr - (e2 + t_hi);                                               // 23 <= k <= 56
    y_hi += 1.0f;
    y_hi = u2f(f2u(y_hi) + kshift);

    float r = (k < 23) ? y_lo : y_hi;
    r = (k <= -2 || k > 56) ? y_far : r;
    r = (k == 1) ? res_p1 : r;
    r = (k == -1) ? res_m1 : r;
    r = (k == 0) ? res_0 : r;
    r = (hx < 0x33000000u) ? x : r;  // |x| < 2^-25 (only reached unreduced)
    return r;
}

JST_FN float libm_tanhf(float x) {
    const uint32_t jx = f2u(x);
    const uint32_t ix = jx & 0x7fffffffu;
    const float ax = u2f(ix);
    const bool ge1 = ix >= 0x3f800000u;
    const float two_ax = 2.0f * ax;
    const float t = libm_expm1f_for_tanh(ge1 ? two_ax : -two_ax);
    const float q = (ge1 ? 2.0f : t) / (t + 2.0f);
    float z = ge1 ? 1.0f - q : -q;             // one - two/(t+two)   |   -t/(t+two)
    z = (ix >= 0x41b00000u) ? 1.0f : z;        // |x| >= 22 (and +-inf): one - tiny == 1.0f
    float r = ((jx >> 31) != 0) ? -z : z;
    r = (ix < 0x24000000u) ? x * (1.0f + x) : r;  // |x| < 2^-55, including +-0
    r = (ix > 0x7f800000u) ? x + x : r;           // NaN
    return r;
}

// Correctly rounded a / b for the operand ranges tanhf produces (|b| in [1, 2^64], quotient and
// residuals far from the subnormal range).  On the device this is the compiler's own FDIV32
// expansion (rcp, two Newton steps on the reciprocal, two on the quotient, final fma) WITHOUT the
// v_div_scale / v_div_fixup range handling and its VCC hazards; on the host it is the IEEE divide.
// Both are correctly rounded, hence equal.
#if defined(__HIP_DEVICE_COMPILE__)
JST_FN float div_rn_midrange(float a, float b) {
    float r = __builtin_amdgcn_rcpf(b);
    const float e0 = __builtin_fmaf(-b, r, 1.0f);
    r = __builtin_fmaf(e0, r, r);
    float q = a * r;
    const float e1 = __builtin_fmaf(-b, q, a);
    q = __builtin_fmaf(e1, r, q);
    const float e2 = __builtin_fmaf(-b, q, a);
    return __builtin_fmaf(e2, r, q);
}
#else
JST_FN float div_rn_midrange(float a, float b) { return a / b; }
#endif
#if defined(__HIP_DEVICE_COMPILE__)
// Candidate shorter divides (see the hooks below): v1 drops the last residual correction, v2 the Newton
// step on the reciprocal, v3 both.
JST_FN float div_v1(float a, float b) {
    float r = __builtin_amdgcn_rcpf(b);
    const float e0 = __builtin_fmaf(-b, r, 1.0f);
    r = __builtin_fmaf(e0, r, r);
    float q = a * r;
    const float e1 = __builtin_fmaf(-b, q, a);
    return __builtin_fmaf(e1, r, q);
}
JST_FN float div_v2(float a, float b) {
    const float r = __builtin_amdgcn_rcpf(b);
    float q = a * r;
    const float e1 = __builtin_fmaf(-b, q, a);
    q = __builtin_fmaf(e1, r, q);
    const float e2 = __builtin_fmaf(-b, q, a);
    return __builtin_fmaf(e2, r, q);
}
JST_FN float div_v3(float a, float b) {
    const float r = __builtin_amdgcn_rcpf(b);
    const float q = a * r;
    const float e1 = __builtin_fmaf(-b, q, a);
    return __builtin_fmaf(e1, r, q);
}
JST_FN float div_v4(float a, float b) { return a * __builtin_amdgcn_rcpf(b); }  // NOT correctly rounded: sweep sensitivity check
#else
JST_FN float div_v4(float a, float b) { return a / b; }
JST_FN float div_v1(float a, float b) { return a / b; }
JST_FN float div_v2(float a, float b) { return a / b; }
JST_FN float div_v3(float a, float b) { return a / b; }
#endif
// copysign(|magnitude|, sign_of): one v_bfi_b32 instead of a compare + select pair
JST_FN float with_sign_of(float magnitude, float sign_of) {
    return u2f((f2u(magnitude) & 0x7fffffffu) | (f2u(sign_of) & 0x80000000u));
}

// Branch-structured variant of the same two functions, following the published control flow
// (s_tanhf.c / s_expm1f.c) instead of computing every alternative: on the GPU a divergent `if`
// costs an exec-mask update and is skipped outright when no lane of the wavefront takes it, which
// is cheaper than the select form as soon as a reconstruction class is absent from a wavefront,
// and it drops the cmp+cndmask pair per alternative.  Arithmetic identical, operation by operation.
JST_FN float libm_expm1f_for_tanh_branchy(float x) {
    constexpr float ln2_hi = 6.9313812256e-01f, ln2_lo = 9.0580006145e-06f,
                    invln2 = 1.4426950216e+00f, Q1 = -3.3333335072e-02f, Q2 = 1.5873016091e-03f,
                    Q3 = -7.9365076090e-05f, Q4 = 4.0082177293e-06f, Q5 = -2.0109921195e-07f;
    const uint32_t bits = f2u(x);
    const uint32_t hx = bits & 0x7fffffffu;
    int32_t k = 0;
    float c = 0.0f;
    if (hx > 0x3eb17218u) {          // |x| > 0.5 ln2
        float hi, lo;
        if (hx < 0x3F851592u) {      // and |x| < 1.5 ln2: k = +-1 by the sign of x
            hi = x - with_sign_of(ln2_hi, x);   // x + ln2_hi == x - (-ln2_hi), bit for bit
            lo = with_sign_of(ln2_lo, x);
            k = 1 | ((int32_t)bits >> 31);      // neg ? -1 : 1
        } else {
            k = (int32_t)(invln2 * x + with_sign_of(0.5f, x));
            const float t = (float)k;
            hi = x - t * ln2_hi;
            lo = t * ln2_lo;
        }
        x = hi - lo;
        c = (hi - x) - lo;
    } else if (hx < 0x33000000u) {   // |x| < 2^-25
        return x;
    }
    const float hfx = 0.5f * x;
    const float hxs = x * hfx;
    const float r1 = 1.0f + hxs * (Q1 + hxs * (Q2 + hxs * (Q3 + hxs * (Q4 + hxs * Q5))));
    float t = 3.0f - r1 * hfx;
    float e = hxs * div_rn_midrange(r1 - t, 6.0f - x * t);
    if (k == 0) return x - (x * e - hxs);
    e = (x * (e - c) - c);
    e -= hxs;
    if (k == -1) return 0.5f * (x - e) - 0.5f;
    if (k == 1) return (x < -0.25f) ? -2.0f * (e - (x + 0.5f)) : 1.0f + 2.0f * (x - e);
    const uint32_t kshift = (uint32_t)k << 23;
    if (k <= -2 || k > 56) return u2f(f2u(1.0f - (e - x)) + kshift) - 1.0f;
    if (k < 23) {
        t = u2f(0x3f800000u - (0x1000000u >> ((uint32_t)k & 31u)));  // 1 - 2^-k
        return u2f(f2u(t - (e - x)) + kshift);
    }
    t = u2f((uint32_t)(0x7f - k) << 23);  // 2^-k
    float y = x - (e + t);
    y += 1.0f;
    return u2f(f2u(y) + kshift);
}

JST_FN float libm_tanhf_branchy(float x) {
    const uint32_t jx = f2u(x);
    const uint32_t ix = jx & 0x7fffffffu;
    const float ax = u2f(ix);
    const bool ge1 = ix >= 0x3f800000u;
    const float two_ax = 2.0f * ax;
    // one expm1f evaluation serves both |x| >= 1 (argument 2|x|) and |x| < 1 (argument -2|x|)
    const float t = libm_expm1f_for_tanh_branchy(ge1 ? two_ax : -two_ax);
    const float q = div_rn_midrange(ge1 ? 2.0f : t, t + 2.0f);
    float z = ge1 ? 1.0f - q : -q;             // one - two/(t+two)   |   -t/(t+two)
    if (ix >= 0x41b00000u) z = 1.0f;           // |x| >= 22 (and +-inf): one - tiny == 1.0f
    float r = u2f(f2u(z) ^ (jx & 0x80000000u));  // (jx < 0) ? -z : z
    if (ix < 0x24000000u) r = x * (1.0f + x);  // |x| < 2^-55, including +-0
    if (ix > 0x7f800000u) r = x + x;           // NaN
    return r;
}

// Division hooks of the main-path form.  tanhf is a function of ONE float, so is every operand pair its
// two divisions ever see: a cheaper sequence than the fully general correctly rounded divide is admissible
// as soon as an exhaustive device sweep (tools/ubench/exact_sweep.hip, tests/test_gpu_exact_sweep.py) shows
// it returns the correctly rounded quotient on all of them.
// Result of that sweep on MI355X (all 2^32 arguments, 0 mismatches, round 2): the shortest candidate, div_v3
// = v_rcp_f32, one product, one exact residual, one fused correction, is correctly rounded on both operand
// families; the uncorrected product div_v4 is not (93 720 wrong tanhf values), which is how the sweep shows
// that it can tell.
#ifndef JST_DIV_EXPM1
#define JST_DIV_EXPM1(a, b) div_v3(a, b)
#endif
#ifndef JST_DIV_TANH
#define JST_DIV_TANH(a, b) div_v3(a, b)
#endif

// ---- main-path form ---------------------------------------------------------------------------
// One straight-line evaluation, free of compare/select pairs, for 2^-26 <= |x| < 7.5 -- every
// argument the Range module produces for a value inside (or within 1.4 spans of) its display range.
// On gfx950 a v_cmp -> v_cndmask pair costs two half-rate instructions plus the SGPR-hazard nops
// between them, and the published ladder of classes turns into a dozen exec-mask regions per
// element, so the classes are merged arithmetically instead:
//   * the expm1f argument a = +-2|x| gets its sign by a bit operation;
//   * ONE argument reduction serves all of them: glibc's |a| <= 0.5 ln2 (k = 0, no reduction) and
//     0.5 ln2 < |a| < 1.5 ln2 (k = +-1 by the sign) shortcuts compute exactly what the general
//     formula k = (int)(invln2*a +- 0.5), hi = a - k*ln2_hi, lo = k*ln2_lo computes whenever the
//     general k agrees (k*ln2_hi, k*ln2_lo are exact for |k| <= 1; k = 0 gives hi = a, lo = c = 0);
//     it does agree on every float of both intervals (tests/test_libm_float.py sweeps all of them);
//   * the reconstructions for k <= -2 and 2 <= k < 23 are one formula: 0x1000000 >> (k & 31) is 0
//     for k in {-7..-1}, i.e. t = 1 - 2^-k degenerates to the `one` of the k <= -2 branch, and the
//     trailing `- one` of that branch becomes `- (|x| >= 1 ? 0 : 1)` (y - 0 == y bit for bit);
//   * k == 0 and k == -1 (|x| < 0.52, the middle quarter of the display range) keep their own
//     three-operation reconstructions, in one exec-masked block that wavefronts without such a
//     lane skip;
//   * z = (|x| >= 1 ? 1 : 0) - (|x| >= 1 ? 2 : t) / (t + 2): `0 - q` is `-q` bit for bit (q != 0).
// Everything else (|x| < 2^-26 incl. 0, |x| >= 7.5 incl. inf, NaN) is reported through `rare` and
// left to libm_tanhf_branchy.  Same operations in the same order as s_tanhf.c / s_expm1f.c on the
// taken path, so the bits are glibc's.
JST_FN float libm_tanhf_main(float x, bool& rare) {
    constexpr float ln2_hi = 6.9313812256e-01f, ln2_lo = 9.0580006145e-06f,
                    invln2 = 1.4426950216e+00f, Q1 = -3.3333335072e-02f, Q2 = 1.5873016091e-03f,
                    Q3 = -7.9365076090e-05f, Q4 = 4.0082177293e-06f, Q5 = -2.0109921195e-07f;
    const uint32_t jx = f2u(x);
    const uint32_t ix = jx & 0x7fffffffu;
    rare = (ix - 0x32800000u) >= (0x40f00000u - 0x32800000u);
    const uint32_t mA = (uint32_t)((int32_t)(0x3f7fffffu - ix) >> 31);  // ~0 when |x| >= 1
    const float a = u2f((ix + 0x00800000u) | (~mA & 0x80000000u));       // +-2|x|
    const int32_t k = (int32_t)(invln2 * a + with_sign_of(0.5f, a));
    const float t = (float)k;
    const float hi = a - t * ln2_hi, lo = t * ln2_lo;
    const float xr = hi - lo;
    const float c = (hi - xr) - lo;
    const float hfx = 0.5f * xr;
    const float hxs = xr * hfx;
    const float r1 = 1.0f + hxs * (Q1 + hxs * (Q2 + hxs * (Q3 + hxs * (Q4 + hxs * Q5))));
    const float t3 = 3.0f - r1 * hfx;
    const float e = hxs * JST_DIV_EXPM1(r1 - t3, 6.0f - xr * t3);
    float e2 = (xr * (e - c) - c);
    e2 -= hxs;
    const float tl = u2f(0x3f800000u - (0x1000000u >> ((uint32_t)k & 31u)));  // 1 - 2^-k (1 for k < 0)
    const float y = u2f(f2u(tl - (e2 - xr)) + ((uint32_t)k << 23));
    float em1 = y - u2f(~mA & 0x3f800000u);
    if ((uint32_t)(k + 1) < 2u) {  // k == 0 or k == -1
#if defined(__HIP_DEVICE_COMPILE__) && !defined(JST_TANH_KBLOCK_SELECT)
        __asm__ volatile("");  // keep it a branch (a wavefront without such a lane skips it); if-converted it is
                               // six operations and two selects for everyone
#endif
        const float r0 = xr - (xr * e - hxs);
        const float rm = 0.5f * (xr - e2) - 0.5f;
        em1 = (k == 0) ? r0 : rm;
    }
    const float num = u2f((mA & 0x40000000u) | (~mA & f2u(em1)));
    const float q = JST_DIV_TANH(num, em1 + 2.0f);
    const float z = u2f(mA & 0x3f800000u) - q;
    return u2f(f2u(z) ^ (jx & 0x80000000u));
}


// =================================================================================================
// sinf / cosf / atanf / atan2f with the values of the host libm that the reference's FM module calls
// (src/domains/dsp/fm/module_impl_native_cpu.cc:93,123-139): glibc 2.35 on x86-64 with FMA.  None of the four is
// correctly rounded there, so equal bits need the same approximations, and these come from published methods and
// from the functions' RETURNED VALUES alone (tools/fit_fm_trig.py derives every constant below and prints it):
//   * sinf / cosf: the method of Arm's optimized routines (Dijkstra, 2018): in F64, reduction by the nearest multiple of
//     pi/2, one odd / even polynomial of degree 7 / 8, ONE rounding to F32.  The coefficients are the centre of the
//     region to which the values returned for all 2^31 positive floats confine them (none is outside its rounding
//     interval; the tightest is 6.7e-10 ulp inside).  Horner's rule, every a * b + c fused.  The reduction is fused as
//     well, because the values say so (n * pi/2 rounded before the subtraction: 6 sines and 11 cosines differ), and
//     they place its end, too: 117.8 (0x1.d7384cp+6) still takes pi/2 rounded to F64, 120.95 (0x1.e3ce26p+6) already
//     the exact reduction.
//   * atanf / atan2f: FDLIBM's method (Sun Microsystems, 1993) in F32 arithmetic, one rounding per written operation
//     (-ffp-contract=off), IEEE divisions.  The polynomial is the minimax one, its high coefficients moved by a few
//     ulps until all returned values agree (14 of 3.3e8 differ without).
// tests/test_libm_float.py compares all four with the host's (sinf / cosf / atanf: every float).
// =================================================================================================
JST_FN double fma_d(double a, double b, double c) { return __builtin_fma(a, b, c); }

namespace trig {
constexpr double kTwoOverPi = 0x1.45f306dc9c883p-1, kHalfPi = 0x1.921fb54442d18p+0;
constexpr double S0 = -0x1.555545995a5e2p-3, S1 = 0x1.110760522fc28p-7, S2 = -0x1.994eb376f69d8p-13;
constexpr double C0 = -0x1.ffffffd0c6278p-2, C1 = 0x1.55553e106acb7p-5, C2 = -0x1.6c087e8a43afbp-10,
                 C3 = 0x1.993430476b822p-16;
}  // namespace trig

// x = m 2^e (m: 24 bits, value >= 64) reduced exactly: x * 2/pi = 4 (whole turns) + n + fraction, n the nearest of 0..3.
// Bits of 2/pi that only add whole turns are skipped and 96 bits kept, of whose product with m the low 32 are dropped:
// 2 bits of n and 62 of the fraction, exact to 2^-61 (Payne and Hanek's method).  Returns fraction * pi/2.
JST_FN double trig_reduce_exact(uint32_t bits, int32_t& n) {
    // 2/pi: word k holds the bits of weight 2^(31 - 32 k) downwards
    const uint32_t two_over_pi[8] = {0x00000000u, 0xa2f9836eu, 0x4e441529u, 0xfc2757d1u,
                                     0xf534ddc0u, 0xdb629599u, 0x3c439041u, 0xfe5163abu};
    const uint32_t m = (bits & 0x7fffffu) | 0x800000u;
    const uint32_t at = ((bits >> 23) & 0xffu) - 120u;  // weight 2^(1 - e), e = exponent - 150: at most 134, word 4 + 3
    const uint32_t w = at >> 5, s = at & 31u;
    const uint32_t t0 = two_over_pi[w], t1 = two_over_pi[w + 1], t2 = two_over_pi[w + 2], t3 = two_over_pi[w + 3];
    const uint32_t h = (uint32_t)((((uint64_t)t0 << 32 | t1) << s) >> 32), c = (uint32_t)((((uint64_t)t1 << 32 | t2) << s) >> 32),
                   l = (uint32_t)((((uint64_t)t2 << 32 | t3) << s) >> 32);
    uint64_t q = ((uint64_t)(m * h) << 32) + (uint64_t)m * c + (((uint64_t)m * l) >> 32);
    const uint64_t k = (q + (1ull << 61)) >> 62;
    n = (int32_t)(k & 3u);
    q -= k << 62;
    return (double)(int64_t)q * (trig::kHalfPi * 0x1p-62);
}

// sin(|y| + quarter * pi/2): quarter 0 gives sinf up to its sign, 1 gives cosf
JST_FN float trig_from_quarter(float y, int32_t quarter) {
    using namespace trig;
    const uint32_t bits = f2u(y) & 0x7fffffffu;
    const double a = (double)u2f(bits);
    double r;
    int32_t n;
    if (bits < 0x42f00000u) {  // |y| < 120
        n = (int32_t)fma_d(a, kTwoOverPi, 0.5);
        r = fma_d(-(double)n, kHalfPi, a);
    } else if (bits < 0x7f800000u) {
        r = trig_reduce_exact(bits, n);
    } else {
        return y - y;  // infinity, NaN -> NaN
    }
    n += quarter;
    const double z = r * r;
    const double p = (n & 1) ? fma_d(z, fma_d(z, fma_d(z, fma_d(z, C3, C2), C1), C0), 1.0)
                             : fma_d(r * z, fma_d(z, fma_d(z, S2, S1), S0), r);
    return (float)((n & 2) ? -p : p);
}
JST_FN float libm_sinf(float y) {
    if ((f2u(y) & 0x7fffffffu) < 0x39800000u) return y;  // |y| < 2^-12: y^2 / 6 is less than half an ulp
    const float r = trig_from_quarter(y, 0);
    return u2f(f2u(r) ^ (f2u(y) & 0x80000000u));
}
JST_FN float libm_cosf(float y) { return trig_from_quarter(y, 1); }

JST_FN float libm_atanf(float x) {
    // atan of 1/2, 1, 3/2, infinity: the value chopped to F32, and the rest of it chopped to F32
    const float atan_hi[4] = {u2f(0x3eed6338u), u2f(0x3f490fdau), u2f(0x3f7b985eu), u2f(0x3fc90fdau)};
    const float atan_lo[4] = {u2f(0x31ac3769u), u2f(0x33222168u), u2f(0x33140fb4u), u2f(0x33a22168u)};
    const float a0 = u2f(0x3eaaaaabu), a1 = u2f(0xbe4ccccdu), a2 = u2f(0x3e124925u), a3 = u2f(0xbde38e38u),
                a4 = u2f(0x3dba2e6eu), a5 = u2f(0xbd9d8795u), a6 = u2f(0x3d886b32u), a7 = u2f(0xbd6ef183u),
                a8 = u2f(0x3d4bdac7u), a9 = u2f(0xbd159eedu), a10 = u2f(0x3c8567a2u);
    const uint32_t sign = f2u(x) & 0x80000000u, ix = f2u(x) & 0x7fffffffu;
    const float ax = u2f(ix);
    if (ix > 0x7f800000u) return x + x;                              // NaN
    if (ix < 0x31000000u) return x;                                  // |x| < 2^-29
    if (ix >= 0x4c000000u) return u2f(f2u(atan_hi[3] + atan_lo[3]) | sign);  // |x| >= 2^25: pi/2
    float t = ax;
    int id = -1;  // atan(x) = atan(c) + atan(t) with c = 1/2, 1, 3/2, infinity
    if (ax >= 2.4375f) {
        id = 3;
        t = -1.0f / ax;
    } else if (ax >= 1.1875f) {
        id = 2;
        t = (ax - 1.5f) / (1.0f + 1.5f * ax);
    } else if (ax >= 0.6875f) {
        id = 1;
        t = (ax - 1.0f) / (ax + 1.0f);
    } else if (ax >= 0.4375f) {
        id = 0;
        t = (2.0f * ax - 1.0f) / (2.0f + ax);
    }
    const float z = t * t, w = z * z;
    const float even = z * (a0 + w * (a2 + w * (a4 + w * (a6 + w * (a8 + w * a10)))));
    const float odd = w * (a1 + w * (a3 + w * (a5 + w * (a7 + w * a9))));
    const float tail = t * (even + odd);
    const float r = id < 0 ? t - tail : atan_hi[id] - ((tail - atan_lo[id]) - t);
    return u2f(f2u(r) | sign);
}

// The angle of |y / x| in the first quadrant, mirrored for x < 0 (pi as an F32 pair), with the sign of y.
JST_FN float libm_atan2f(float y, float x) {
    const float pi = u2f(0x40490fdbu), pi_lo = u2f(0xb3bbbd2eu);  // F32(pi), F32(pi - F32(pi))
    const float half_pi = u2f(0x3fc90fdbu), quarter_pi = u2f(0x3f490fdbu), three_quarter_pi = u2f(0x4016cbe4u);
    const uint32_t ix = f2u(x) & 0x7fffffffu, iy = f2u(y) & 0x7fffffffu;
    const bool left = (f2u(x) >> 31) != 0;
    if (ix > 0x7f800000u || iy > 0x7f800000u) return x + y;  // NaN
    const bool x_inf = ix == 0x7f800000u, y_inf = iy == 0x7f800000u;
    float r;
    if (x_inf && y_inf) {
        r = left ? three_quarter_pi : quarter_pi;
    } else if (iy == 0 || x_inf) {
        r = left ? pi : 0.0f;
    } else if (ix == 0 || y_inf) {
        r = half_pi;
    } else {
        const float z = libm_atanf(u2f(f2u(y / x) & 0x7fffffffu));
        r = left ? pi - (z - pi_lo) : z;
    }
    return with_sign_of(r, y);
}

}  // namespace jst::dev
