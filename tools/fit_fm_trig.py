#!/usr/bin/env python3
"""Derives the constants of libm_sinf / libm_cosf / libm_atanf / libm_atan2f (cyberether_amd/csrc/kernels/libm_float.hh) from
mathematics and from what the C library's sinf, cosf and atanf RETURN -- calls of the public functions, nothing else.

sinf, cosf.  The argument is widened to F64, reduced to r in [-pi/4, pi/4] by a multiple of pi/2 and one of
    sin r ~ r + r z (S0 + z (S1 + z S2))            z = r^2
    cos r ~ 1 + z (C0 + z (C1 + z (C2 + z C3)))
is rounded to F32 once.  A function value that the library returned confines the polynomial at that argument to one rounding
interval of F32, which is LINEAR in the coefficients.  2^31 arguments confine three (four) coefficients to a sliver; this
program finds its centre with cutting planes: solve a small linear program for the point furthest from every interval's end
(in units of the result's ulp), rescan with finer strides for the arguments that are tightest there, repeat.  An end of an
interval is widened or narrowed by half an F64 ulp, by the parity of the F32 neighbour: the F64 result itself is rounded,
and a tie goes to even.

atanf.  FDLIBM's published method (Sun Microsystems 1993): |x| below 7/16 directly, otherwise through atan(c) + atan(t) with
c = 1/2, 1, 3/2, infinity on [7/16, 11/16), [11/16, 19/16), [19/16, 39/16) and above, atan(c) as a chopped F32 pair, and
    atan t ~ t - t (z (a0 + w (a2 + ...)) + w (a1 + w (a3 + ...)))     z = t^2, w = z^2, every operation one F32 rounding.
The coefficients are the minimax polynomial's (Remez on [0, (7/16)^2], weight z), rounded to F32; the high ones are then
moved by a few ulps, one or two at a time, until every returned value agrees.

    python tools/fit_fm_trig.py         (about three minutes on eight cores, x86-64 glibc 2.35 on a CPU with FMA)
prints the constants in the form the header holds them in."""
import ctypes as C
import itertools
import math
import os
import subprocess
import tempfile
from decimal import Decimal as D, getcontext

import numpy as np
from scipy.optimize import linprog

getcontext().prec = 60
THREADS = os.cpu_count() or 1

SOURCE = r"""
#include <math.h>
#include <stdint.h>
#include <string.h>
#include <atomic>
#include <mutex>
#include <thread>
#include <vector>
static float u2f(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }
static uint32_t f2u(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }
template <class F> static void parallel(uint64_t n, int threads, F f) {
    std::vector<std::thread> th;
    for (int t = 0; t < threads; ++t) th.emplace_back([=] { f(n * t / threads, n * (t + 1) / threads); });
    for (auto& t : th) t.join();
}
static double reduce(float f, double hpi, const uint32_t* T, int* n) {
    if (f < 120.0f) {
        *n = (int)__builtin_fma((double)f, 1.0 / hpi, 0.5);
        return __builtin_fma(-(double)*n, hpi, (double)f);
    }
    const uint32_t b = f2u(f), m = (b & 0x7fffff) | 0x800000;
    const int p = (int)(b >> 23) - 120, w = p >> 5, s = p & 31;
    auto win = [&](int k) { return (uint32_t)((((uint64_t)T[w + k] << 32 | T[w + k + 1]) << s) >> 32); };
    uint64_t q = ((uint64_t)(m * win(0)) << 32) + (uint64_t)m * win(1) + (((uint64_t)m * win(2)) >> 32);
    const uint64_t k = (q + (1ull << 61)) >> 62;
    *n = (int)(k & 3);
    q -= k << 62;
    return (double)(int64_t)q * (hpi * 0x1p-62);
}
// the arguments at which polynomial `cosine` comes closer than `near` ulps to an end of the returned value's interval:
// {reduced argument, distance to the lower end, to the upper end, ulp}
extern "C" long tightest(int cosf_called, int cosine, uint32_t start, uint32_t stride, uint64_t count, const double* hi, const double* lo,
                         int nc, double hpi, const uint32_t* T, double near, double* out, long cap, int threads) {
    std::mutex mu;
    long got = 0;
    parallel(count, threads, [&](uint64_t from, uint64_t to) {
        std::vector<double> rows;
        for (uint64_t i = from; i < to; ++i) {
            const float f = u2f(start + (uint32_t)(i * stride));
            int n;
            const double r = reduce(f, hpi, T, &n);
            if ((((n & 1) != 0) != (cosf_called == 1)) != (cosine == 1)) continue;
            const float fr = fabsf(cosf_called ? cosf(f) : sinf(f));
            const long double z = (long double)r * r;
            long double p = 0;
            for (int k = nc - 1; k >= 0; --k) p = p * z + ((long double)hi[k] + lo[k]);
            p = fabsl(cosine ? 1.0L + z * p : r + r * z * p);
            const uint32_t b = f2u(fr);
            const double up = ((double)fr + u2f(b + 1)) * 0.5, dn = ((double)fr + u2f(b - 1)) * 0.5, ulp = up - dn;
            const double tie = (b & 1) ? -0x1p-30 : 0x1p-30;  // half an F64 ulp in F32 ulps
            const double a = (double)((p - dn) / ulp) + tie, c = (double)((up - p) / ulp) + tie;
            if (a < near || c < near) rows.insert(rows.end(), {cosine ? r : fabs(r), a, c, ulp});
        }
        std::lock_guard<std::mutex> g(mu);
        for (size_t i = 0; i < rows.size(); i += 4, ++got)
            if (got < cap) memcpy(out + 4 * got, &rows[i], 32);
    });
    return got < cap ? got : cap;
}
static float atan_form(float ax, const float* a, const float* hi, const float* lo) {
    int id = -1;
    float x = ax;
    if (ax < 0.4375f) {}
    else if (ax < 0.6875f) { id = 0; x = (2.0f * ax - 1.0f) / (2.0f + ax); }
    else if (ax < 1.1875f) { id = 1; x = (ax - 1.0f) / (ax + 1.0f); }
    else if (ax < 2.4375f) { id = 2; x = (ax - 1.5f) / (1.0f + 1.5f * ax); }
    else { id = 3; x = -1.0f / ax; }
    const float z = x * x, w = z * z;
    const float s1 = z * (a[0] + w * (a[2] + w * (a[4] + w * (a[6] + w * (a[8] + w * a[10])))));
    const float s2 = w * (a[1] + w * (a[3] + w * (a[5] + w * (a[7] + w * a[9]))));
    if (id < 0) return x - x * (s1 + s2);
    return hi[id] - ((x * (s1 + s2) - lo[id]) - x);
}
extern "C" long atan_differs(const float* a, const float* hi, const float* lo, uint32_t start, uint64_t count, uint32_t* out, long cap, int threads) {
    std::atomic<long> n{0};
    parallel(count, threads, [&](uint64_t from, uint64_t to) {
        for (uint64_t i = from; i < to; ++i) {
            const float x = u2f(start + (uint32_t)i);
            if (f2u(atan_form(x, a, hi, lo)) != f2u(atanf(x))) {
                const long k = n++;
                if (k < cap) out[k] = start + (uint32_t)i;
            }
        }
    });
    return n;
}
extern "C" long atan_differs_at(const float* a, const float* hi, const float* lo, const uint32_t* u, long n) {
    long bad = 0;
    for (long i = 0; i < n; ++i) bad += f2u(atan_form(u2f(u[i]), a, hi, lo)) != f2u(atanf(u2f(u[i])));
    return bad;
}
"""


def compile_scanner():
    tmp = tempfile.mkdtemp()
    src, out = os.path.join(tmp, "scan.cc"), os.path.join(tmp, "scan.so")
    with open(src, "w") as f:
        f.write(SOURCE)
    subprocess.check_call(["g++", "-O2", "-std=c++20", "-ffp-contract=off", "-fno-builtin", "-mfma", "-fPIC", "-shared", src, "-o", out, "-lm", "-lpthread"])
    lib = C.CDLL(out)
    p = C.c_void_p
    lib.tightest.restype = lib.atan_differs.restype = lib.atan_differs_at.restype = C.c_long
    lib.tightest.argtypes = [C.c_int, C.c_int, C.c_uint32, C.c_uint32, C.c_uint64, p, p, C.c_int, C.c_double, p, C.c_double, p, C.c_long, C.c_int]
    lib.atan_differs.argtypes = [p, p, p, C.c_uint32, C.c_uint64, p, C.c_long, C.c_int]
    lib.atan_differs_at.argtypes = [p, p, p, p, C.c_long]
    return lib


def bits(x):
    return int(np.float32(x).view(np.uint32))


def ptr(a):
    return a.ctypes.data


# ---- pi, 2/pi, atan from their series ---------------------------------------------------------------------------------------
def atan_tail(z):
    """(x - atan x) / x^3 at x^2 = z: 1/3 - z/5 + z^2/7 - ..."""
    s, t, k = D(0), D(1), 0
    while abs(t) > D(10) ** -57:
        s += t / (2 * k + 3)
        t *= -z
        k += 1
    return s


def atan(x):
    return x - x ** 3 * atan_tail(x * x)


def machin_pi():
    def arctan_inverse(n):
        s, t, k = D(0), D(1) / n, 0
        while abs(t) > D(10) ** -(getcontext().prec - 2):
            s += t / (2 * k + 1)
            t /= -(n * n)
            k += 1
        return s
    return 4 * (4 * arctan_inverse(5) - arctan_inverse(239))


PI = machin_pi()


def two_over_pi_words(words):
    """Word 0 holds the bits of weight 2^31 .. 2^0 of 2/pi (all zero), word k those of weight 2^(31-32k) downwards."""
    getcontext().prec = 120
    v = int(D(2) / machin_pi() * D(2) ** (32 * (words - 1)))
    getcontext().prec = 60
    return np.array([(v >> (32 * (words - 1 - k))) & 0xffffffff for k in range(words)], np.uint32)


# ---- sinf / cosf ------------------------------------------------------------------------------------------------------------
def fit_polynomial(lib, cosine, hpi, table):
    first = 2 if cosine else 3
    c = [np.longdouble((-1) ** (k + 1)) / math.factorial(first + 2 * k) for k in range(4 if cosine else 3)]  # Taylor
    largest = float(np.uint32(0x7f7fffff).view(np.float32))
    own, every = (2.0 ** -12, math.pi / 4), (2.0 ** -12, largest)
    for stride, near, (lo, hi) in ((20011, 9, own), (2003, 2e-2, own), (211, 2e-3, own), (17, 2e-4, own), (1, 1e-5, own),
                                   (1, 1e-6, every), (1, 2e-7, every), (1, 2e-7, every)):
        rows = []
        for called in ((cosine,) if hi < 1 else (0, 1)):
            buf = np.zeros((400000, 4))
            h = np.array([float(v) for v in c])
            l = np.array([float(v - np.longdouble(float(v))) for v in c])
            n = lib.tightest(called, cosine, bits(lo), stride, (bits(hi) - bits(lo)) // stride, ptr(h), ptr(l), len(c), hpi, ptr(table),
                             near, ptr(buf), len(buf), THREADS)
            rows.append(buf[:n])
        x, below, above, ulp = np.vstack(rows).T
        basis = np.stack([x ** (first + 2 * k) for k in range(len(c))], 1) / ulp[:, None]
        slack = np.concatenate([below, above])
        scale = max(1e-12, float(np.percentile(np.abs(np.minimum(below, above)), 50)))
        col = np.abs(basis).max(0)
        rhs = slack / scale
        keep = rhs < np.abs(rhs).min() * 1e4 + 1e4
        a = np.vstack([np.hstack([-basis / col, np.ones((len(x), 1))]), np.hstack([basis / col, np.ones((len(x), 1))])])[keep]
        r = linprog([0.0] * len(c) + [-1.0], A_ub=a, b_ub=rhs[keep], bounds=[(-1e9, 1e9)] * len(c) + [(None, 1e9)], method="highs")
        assert r.status == 0, r.message
        c = [v + np.longdouble(d) for v, d in zip(c, r.x[:-1] * scale / col)]
        print(f"  {'cos' if cosine else 'sin'}: {len(x)} arguments, outside their interval before this step {int((np.minimum(below, above) < 0).sum())}, "
              f"furthest possible distance {r.x[-1] * scale:.3g} ulp", flush=True)
    return [float(v) for v in c]


# ---- atanf ------------------------------------------------------------------------------------------------------------------
def solve(a, b):
    n = len(a)
    m = [row[:] + [v] for row, v in zip(a, b)]
    for i in range(n):
        p = max(range(i, n), key=lambda r: abs(m[r][i]))
        m[i], m[p] = m[p], m[i]
        for r in range(n):
            if r != i and m[r][i] != 0:
                f = m[r][i] / m[i][i]
                m[r] = [u - f * v for u, v in zip(m[r], m[i])]
    return [m[i][n] / m[i][i] for i in range(n)]


def minimax_atan(degree, end, samples=4000):
    """Remez: the polynomial p(z) of that degree that minimises max z |tail(z) - p(z)| on (0, end]."""
    n = degree + 2
    grid = [end * (1 - D(math.cos(math.pi * (i + 0.5) / samples))) / 2 for i in range(samples)] + [end]
    f = [atan_tail(z) for z in grid]
    at = [round((i + 1) * samples / n) for i in range(n)]
    while True:
        sol = solve([[grid[i] ** k if k else D(1) for k in range(degree + 1)] + [(-1) ** j / grid[i]] for j, i in enumerate(at)], [f[i] for i in at])
        c = sol[:-1]
        err = [z * (v - sum(ck * (z ** k if k else 1) for k, ck in enumerate(c))) for z, v in zip(grid, f)]
        ext = []
        for i, e in enumerate(err):
            if (i == 0 or abs(e) >= abs(err[i - 1])) and (i == samples or abs(e) >= abs(err[i + 1])):
                if ext and (e > 0) == (err[ext[-1]] > 0):
                    if abs(e) > abs(err[ext[-1]]):
                        ext[-1] = i
                else:
                    ext.append(i)
        while len(ext) > n:
            ext.pop(0 if abs(err[ext[0]]) < abs(err[ext[-1]]) else -1)
        assert len(ext) == n
        if ext == at:
            return c
        at = ext


def chop(d):
    f = np.float32(float(d))
    return f if D(float(f)) <= d else np.nextafter(f, np.float32(0))


def fit_atan(lib):
    values = [atan(D(1) / 2), PI / 4, PI / 4 + atan(D(1) / 5), PI / 2]  # atan of 1/2, 1, 3/2, infinity
    hi = np.array([chop(v) for v in values], np.float32)
    lo = np.array([chop(v - D(float(h))) for v, h in zip(values, hi)], np.float32)
    a = np.array([float(v) for v in minimax_atan(10, (D(7) / 16) ** 2)], np.float32)
    start, count = bits(2.0 ** -14), bits(2.0 ** 25) - bits(2.0 ** -14)  # below x itself, from 2^25 on pi/2
    buf = np.zeros(100000, np.uint32)

    def moved(v, k, d):
        w = v.copy()
        w.view(np.int32)[k] += d
        return w

    def differs(v):
        return lib.atan_differs(ptr(v), ptr(hi), ptr(lo), start, count, ptr(buf), len(buf), THREADS)
    print(f"  atan: {differs(a)} of {count} values differ with the minimax coefficients as they are", flush=True)
    moves = [(k, s * d) for k, ds in ((4, (1,)), (5, (1, 2, 3)), (6, (1, 2, 4, 6, 8)), (7, (4, 8, 16, 32, 64, 128)), (8, (32, 64, 128, 256, 512)),
                                      (9, (128, 512, 2048)), (10, (512, 4096))) for d in ds for s in (1, -1)]
    watch = set()  # every argument whose value some move changes to a wrong one
    for k, d in moves:
        watch |= set(buf[:min(differs(moved(a, k, d)), len(buf))].tolist())
    u = np.array(sorted(watch), np.uint32)

    def wrong(v):
        return lib.atan_differs_at(ptr(v), ptr(hi), ptr(lo), ptr(u), len(u))
    best = wrong(a)
    while best:
        steps = [(m,) for m in moves] + [p for p in itertools.combinations(moves, 2) if p[0][0] != p[1][0]]
        trial = []
        for step in steps:
            v = a
            for k, d in step:
                v = moved(v, k, d)
            trial.append((wrong(v), len(step), step))
        score, _, step = min(trial)
        assert score < best, "no step of one or two moves helps"
        best = score
        for k, d in step:
            a = moved(a, k, d)
    print(f"  atan: {differs(a)} differ after the moves", flush=True)
    return a, hi, lo


def main():
    lib = compile_scanner()
    hpi = float(PI / 2)
    table = two_over_pi_words(8)
    s = fit_polynomial(lib, 0, hpi, table)
    c = fit_polynomial(lib, 1, hpi, table)
    a, hi, lo = fit_atan(lib)
    print("2/pi       ", ", ".join(f"0x{int(v):08x}u" for v in table))
    print("pi/2       ", hpi.hex(), "  2/pi", float(2 / PI).hex())
    print("sin S0..S2 ", ", ".join(v.hex() for v in s))
    print("cos C0..C3 ", ", ".join(v.hex() for v in c))
    print("atan a0..a10", ", ".join(f"0x{int(v):08x}u" for v in a.view(np.uint32)))
    print("atan hi    ", ", ".join(f"0x{int(v):08x}u" for v in hi.view(np.uint32)))
    print("atan lo    ", ", ".join(f"0x{int(v):08x}u" for v in lo.view(np.uint32)))
    pi32 = np.float32(float(PI))
    for name, v in (("pi", pi32), ("pi - F32(pi)", np.float32(float(PI - D(float(pi32))))), ("pi/2", np.float32(float(PI / 2))),
                    ("pi/4", np.float32(float(PI / 4))), ("3 pi/4", np.float32(float(3 * PI / 4)))):
        print(f"{name:12s} 0x{int(v.view(np.uint32)):08x}u")


if __name__ == "__main__":
    main()
