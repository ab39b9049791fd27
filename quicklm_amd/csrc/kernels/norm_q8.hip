// RMSNorm with the residual's addition and an output in 8 bits, one scale a
// row: the activations of the 8-bit matrix product (gemm_a8.hip).
//   r = x + delta                        (one fp32 rounding; stored as `sum`)
//   y = r / sqrt(mean(r^2) + eps) * (1 + w)
//   s = max|y| / 127 (1 for a row of zeros),  q = rne(y / s)
// The root mean square is a factor of both y and s, so the bytes depend only
// on t = r (1 + w): q = rne(127 t / max|t|), and s = max|t| / 127 / rms. The
// sum of squares and max|t| therefore come out of ONE pass over the row held
// in registers, with one block reduction.
//
// t, the sums and the quotient are in 64 bits: in 32 bits the quotient's own
// rounding error (2^-24 of up to 127 steps) moves about one byte in 10^5 to
// the other side of a rounding border; in 64 bits the byte is that of the exact
// quotient, unless that lies within 127 2^-50 of a border, and squares of large
// values do not overflow. gfx950 runs fp64 vector operations at the rate of
// unpacked fp32 ones and the kernel is bound by memory, so this costs nothing
// that shows: 8192 x 4096 with the sum stored moves 436 MB in 82 to 87 us, 5.0
// to 5.3 TB/s, where a 4 GiB copy reaches 4.75.

#include "common.hpp"

namespace {

// rows of any stride: vectors of four aligned to one element only
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32u __attribute__((aligned(1)));

// Reductions of doubles over the wave as common.hpp's of floats: each half
// moved by DPP, and by lane swaps across rows of 16.
template <int CTRL>
__device__ __forceinline__ double dpp_mov_f64(double v) {
    const long long b = __double_as_longlong(v);
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)b, CTRL, 0xf, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xf, 0xf, false);
    return __longlong_as_double((long long)hi << 32 | lo);
}
template <bool SUM>
__device__ __forceinline__ double wave_reduce_f64(double v) {
    auto op = [](double a, double b) { return SUM ? a + b : fmax(a, b); };
    v = op(v, dpp_mov_f64<kDppXor1>(v));
    v = op(v, dpp_mov_f64<kDppXor2>(v));
    v = op(v, dpp_mov_f64<kDppHalfMirror>(v));
    v = op(v, dpp_mov_f64<kDppMirror>(v));
    auto swapped = [&](auto lo, auto hi) {
        return op(__longlong_as_double((long long)hi[0] << 32 | lo[0]),
                  __longlong_as_double((long long)hi[1] << 32 | lo[1]));
    };
    long long b = __double_as_longlong(v);
    v = swapped(__builtin_amdgcn_permlane16_swap((unsigned)b, (unsigned)b, false, false),
                __builtin_amdgcn_permlane16_swap((unsigned)(b >> 32), (unsigned)(b >> 32), false,
                                                 false));
    b = __double_as_longlong(v);
    return swapped(__builtin_amdgcn_permlane32_swap((unsigned)b, (unsigned)b, false, false),
                   __builtin_amdgcn_permlane32_swap((unsigned)(b >> 32), (unsigned)(b >> 32),
                                                    false, false));
}

constexpr int kMaxRows = 1 << 21;  // a launch's threads fit 32 bits

struct NormArgs {
    const float* x;
    const float* delta;  // NULL: nothing is added
    const float* w;
    float* sum;  // NULL: the sum is not stored; may be x or delta itself
    int8_t* q;
    float* scales;
    long long ldx, ldd, lds, ldq;
    int rows, n;
    float eps;
};

// Both inputs are read once: past the caches (2048 x 2560 23.5 -> 20.4 us).
__device__ __forceinline__ f32x4u stream4(const float* p) {
    return __builtin_nontemporal_load(reinterpret_cast<const f32x4u*>(p));
}

// One value's byte. Next to a rounding border the product with the rounded
// reciprocal may fall on the other side: there the quotient is divided out.
__device__ __forceinline__ int quant_t(double t, double inv, double top) {
    const double v = t * inv;
    double r = rint(v);
    if (fabs(fabs(v - r) - 0.5) < 1e-9) r = rint(t * 127.0 / top);
    return (int)r;
}

// What a thread has seen of a row.
struct RowStat {
    double ss = 0.0;   // sum of r^2
    double top = 0.0;  // max |t|
    double bad = 0.0;  // NaN once a t is not finite (fmax drops NaN)
    __device__ __forceinline__ void add(float r, float w) {
        const double rd = (double)r, t = rd * (1.0 + (double)w);
        ss = fma(rd, rd, ss);
        top = fmax(top, fabs(t));
        bad = fma(t, 0.0, bad);
    }
};

// WPR waves share a row. HOLD: the row stays in registers as V vectors of four
// a thread; otherwise (rows longer than 4 * 64 * WPR * V) it is read twice.
template <int WPR, int V, bool HOLD>
__global__ __launch_bounds__(WPR >= 4 ? WPR * QLM_WAVE : 256) void k_norm_q8(NormArgs a) {
    constexpr int WAVES = WPR >= 4 ? WPR : 4;  // waves of a workgroup
    constexpr int RPB = WAVES / WPR;           // rows of a workgroup
    constexpr int TPR = WPR * QLM_WAVE;        // threads of a row
    __shared__ double red[3][WAVES];
    const int wave = threadIdx.x / QLM_WAVE;
    const int t = threadIdx.x % TPR;
    const long long row = (long long)blockIdx.x * RPB + wave / WPR;
    const bool live = row < a.rows;  // waves past the last row only meet the barrier
    const float* xr = a.x + row * a.ldx;
    const float* dr = a.delta ? a.delta + row * a.ldd : nullptr;
    float* sr = a.sum ? a.sum + row * a.lds : nullptr;
    const int n4 = a.n >> 2, tail = a.n & 3;
    RowStat st;
    f32x4u keep[HOLD ? V : 1];
    float keep_tail = 0.0f;
    if (live) {
        auto four = [&](int i, f32x4u v) {
            const f32x4u w = *reinterpret_cast<const f32x4u*>(a.w + 4 * (size_t)i);
            if (sr) *reinterpret_cast<f32x4u*>(sr + 4 * (size_t)i) = v;
            st.add(v.x, w.x);
            st.add(v.y, w.y);
            st.add(v.z, w.z);
            st.add(v.w, w.w);
        };
        if constexpr (HOLD) {
            // every request of the row goes out before the first use
            f32x4u d[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int i = t + j * TPR;
                keep[j] = f32x4u{0.0f, 0.0f, 0.0f, 0.0f};
                if (i < n4) keep[j] = stream4(xr + 4 * (size_t)i);
            }
            if (dr) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int i = t + j * TPR;
                    d[j] = f32x4u{0.0f, 0.0f, 0.0f, 0.0f};
                    if (i < n4) d[j] = stream4(dr + 4 * (size_t)i);
                }
#pragma unroll
                for (int j = 0; j < V; ++j) keep[j] += d[j];
            }
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (t + j * TPR < n4) four(t + j * TPR, keep[j]);
        } else {
            for (int i = t; i < n4; i += TPR) {
                f32x4u v = *reinterpret_cast<const f32x4u*>(xr + 4 * (size_t)i);
                if (dr) v += *reinterpret_cast<const f32x4u*>(dr + 4 * (size_t)i);
                four(i, v);
            }
        }
        if (t < tail) {
            const int i = 4 * n4 + t;
            keep_tail = xr[i];
            if (dr) keep_tail += dr[i];
            if (sr) sr[i] = keep_tail;
            st.add(keep_tail, a.w[i]);
        }
    }
    st.ss = wave_reduce_f64<true>(st.ss + st.bad);
    st.top = wave_reduce_f64<false>(st.top);
    if constexpr (WPR > 1) {
        if (threadIdx.x % QLM_WAVE == 0) {
            red[0][wave] = st.ss;
            red[1][wave] = st.top;
        }
        __syncthreads();
        const int w0 = wave / WPR * WPR;
        st.ss = red[0][w0];
        st.top = red[1][w0];
#pragma unroll
        for (int i = 1; i < WPR; ++i) {
            st.ss += red[0][w0 + i];
            st.top = fmax(st.top, red[1][w0 + i]);
        }
    }
    if (!live) return;
    // A row with a value that is not finite has no scale: NaN, bytes 0, so
    // that its products come out NaN as those of the unquantised row do.
    float s = (float)(st.top / 127.0 / sqrt(st.ss / (double)a.n + (double)a.eps));
    const bool fine = s < INFINITY;  // false for NaN too
    double top = st.top;
    if (!(top > 0.0) || !fine) {
        s = fine ? 1.0f : NAN;
        top = INFINITY;  // every byte 0
    }
    const double inv = 127.0 / top;
    if (t == 0) a.scales[row] = s;
    int8_t* qr = a.q + row * a.ldq;
    auto one = [&](float r, float w) -> unsigned {
        const double v = (double)r * (1.0 + (double)w);
        return top < INFINITY ? (unsigned)quant_t(v, inv, top) & 0xffu : 0u;
    };
    auto pack = [&](int i, f32x4u v) {
        const f32x4u w = *reinterpret_cast<const f32x4u*>(a.w + 4 * (size_t)i);
        *reinterpret_cast<u32u*>(qr + 4 * (size_t)i) = one(v.x, w.x) | one(v.y, w.y) << 8 |
                                                       one(v.z, w.z) << 16 | one(v.w, w.w) << 24;
    };
    if constexpr (HOLD) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (t + j * TPR < n4) pack(t + j * TPR, keep[j]);
    } else {
        // the row again: what this thread stored, or its two terms
        for (int i = t; i < n4; i += TPR) {
            f32x4u v;
            if (sr) {
                v = *reinterpret_cast<const f32x4u*>(sr + 4 * (size_t)i);
            } else {
                v = *reinterpret_cast<const f32x4u*>(xr + 4 * (size_t)i);
                if (dr) v += *reinterpret_cast<const f32x4u*>(dr + 4 * (size_t)i);
            }
            pack(i, v);
        }
    }
    if (t < tail) qr[4 * n4 + t] = (int8_t)one(keep_tail, a.w[4 * n4 + t]);
}

template <int WPR, int V, bool HOLD = true>
void launch(const NormArgs& a, hipStream_t st) {
    constexpr int WAVES = WPR >= 4 ? WPR : 4, RPB = WAVES / WPR;
    hipLaunchKernelGGL((k_norm_q8<WPR, V, HOLD>), dim3((unsigned)((a.rows + RPB - 1) / RPB)),
                       dim3(WAVES * QLM_WAVE), 0, st, a);
}

}  // namespace

extern "C" int qlm_add_rms_norm_q8(const float* x, int ldx, const float* delta, int ldd,
                                   const float* w, float eps, float* sum, int lds, int8_t* q,
                                   int ldq, float* scales, int rows, int n, void* stream) {
    if (!x || !w || !q || !scales || rows <= 0 || n <= 0) return QLM_ERR_ARG;
    if (ldx < n || ldq < n || (delta && ldd < n) || (sum && lds < n)) return QLM_ERR_ARG;
    if (sum && !delta) return QLM_ERR_ARG;
    if (!(eps >= 0.0f)) return QLM_ERR_ARG;
    // the sum in place of one of its terms needs that term's rows
    if (sum && ((sum == x && lds != ldx) || (sum == delta && lds != ldd))) return QLM_ERR_ARG;
    const NormArgs a{x, delta, w, sum, q, scales, ldx, ldd, lds, ldq, rows, n, eps};
    if (rows > kMaxRows) return QLM_ERR_SHAPE;
    hipStream_t st = as_stream(stream);
    const int n4 = n / 4 + (n % 4 != 0);  // n + 3 may pass 2^31
    // Few rows are bound by latency: more waves share one (1 x 2560 4.5 us with
    // 4 waves, 3.7 with 8). Many are bound by the loads in flight, of which a
    // thread then has more while its registers leave room for other rows (8192 x
    // 2560 54 us with 4 waves of 3 vectors, 59 of 4, 61 with 8 of 2; 8192 x 4096
    // 85 with 4 of 4, 82 with 8 of 2). Up to 1024 values a wave takes a row alone
    // once rows are many (n 1024, four waves a row and one: 2048 rows 9.9 and 11.4
    // us, 4096 rows 16.5 and 15.8, 16384 rows 49.2 and 47.6). From 4097 values on 16
    // waves hold the row up to 16384 of them, which beats reading it twice also
    // where most of their places are empty (2048 x 5120 35.8 us and 40.3, 8192 x
    // 8192 167 and 183, 2048 x 16384 87 and 99).
    if (n4 <= 64)
        launch<1, 1>(a, st);
    else if (n4 <= 256)
        rows <= 2048 ? launch<4, 1>(a, st) : launch<1, 4>(a, st);
    else if (n4 <= 768)
        rows < 1024 ? launch<8, 2>(a, st) : launch<4, 3>(a, st);
    else if (n4 <= 1024)
        launch<8, 2>(a, st);
    else if (n4 <= 4096)
        launch<16, 4>(a, st);
    else
        launch<16, 1, false>(a, st);
    return qlm_launch_status();
}

// Loads this file's code object on the current device now; the runtime
// otherwise loads it at the first launch of one of its kernels.
hipError_t qlm_load_norm_q8() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(k_norm_q8<4, 3, true>));
}
