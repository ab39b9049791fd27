// Matrix product of 8-bit rows and 8-bit weights on the gfx950 int8 matrix
// cores, one scale a row and one a channel:
//   y[m, n] = sx[m] * sw[n] * sum_k x[m, k] * q[n, k]
// The sums are exact in int32 (|x|, |q| <= 128 and K < 2^17), so they may be
// split and joined in any order without changing a bit; each is rounded to
// fp32 once and scaled.
//
// Both operands meet v_mfma_i32_16x16x64_i8 as 16 x 64 fragments of 1 KB,
// lane l = 16 c + r holding columns 16 c .. + 15 of row r. The tile-major
// weights (qlm_mx_swizzle) are stored that way, and a wave's load of 16 rows
// of x puts them that way. The weights are the first operand: a lane of the
// result then holds four neighbouring outputs of one row of x.
//
// Few rows (M <= 64), k_a8_stream: bound by the stream of the weights; the
// waves of a workgroup split K over one 16-row weight tile.
// More rows, k_a8_tile: both operands staged through LDS.

#include "common.hpp"

namespace {

enum { EPI_STORE = 0, EPI_RESID = 1, EPI_SWIGLU = 2 };
typedef int v4i __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

struct A8Args {
    const int8_t* x;
    const float* sx;
    const int8_t* q;
    const float* sw;
    float* y;
    long long ldx, ldy;
    int M, N, K;
    int tiles;  // 16-row weight tiles (of a half, for SwiGLU)
};

// Four neighbouring outputs n .. n + 3 of row m.
template <int EPI>
__device__ __forceinline__ void put4(const A8Args& a, int m, int n, v4i s0, v4i s1) {
    if (m >= a.M || n >= a.N) return;
    const float sx = a.sx[m];
    float* dst = a.y + (size_t)m * a.ldy + n;
    const bool whole = n + 4 <= a.N;
    f32x4u w0{0, 0, 0, 0}, w1{0, 0, 0, 0}, old{0, 0, 0, 0}, v;
    if (whole) {
        w0 = *reinterpret_cast<const f32x4u*>(a.sw + n);
        if constexpr (EPI == EPI_SWIGLU) w1 = *reinterpret_cast<const f32x4u*>(a.sw + a.N + n);
        if constexpr (EPI == EPI_RESID) old = *reinterpret_cast<const f32x4u*>(dst);
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (n + i < a.N) {
                w0[i] = a.sw[n + i];
                if constexpr (EPI == EPI_SWIGLU) w1[i] = a.sw[a.N + n + i];
                if constexpr (EPI == EPI_RESID) old[i] = dst[i];
            }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float p = (float)s0[i] * sx * w0[i];
        if constexpr (EPI == EPI_SWIGLU)
            v[i] = silu_f(p) * ((float)s1[i] * sx * w1[i]);
        else if constexpr (EPI == EPI_RESID)
            v[i] = old[i] + p;
        else
            v[i] = p;
    }
    if (whole) {
        *reinterpret_cast<f32x4u*>(dst) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (n + i < a.N) dst[i] = v[i];
    }
}

// MT 16-row tiles of x against one weight tile (SwiGLU: the gate tile and its
// up tile) a workgroup; NW waves take the 64-column blocks in turn and add
// their sums in LDS (integers: in any order).
template <int EPI, int MT, int NW>
__global__ __launch_bounds__(NW * QLM_WAVE) void k_a8_stream(A8Args a) {
    constexpr int H = EPI == EPI_SWIGLU ? 2 : 1;
    constexpr int U = 4;
    __shared__ int sums[H * MT * 256];
    const int lane = threadIdx.x & (QLM_WAVE - 1), wave = threadIdx.x / QLM_WAVE;
    for (int i = threadIdx.x; i < H * MT * 256; i += NW * QLM_WAVE) sums[i] = 0;
    __syncthreads();
    const int nblk = a.K >> 6, tile = blockIdx.x;
    const int8_t* xr[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
        xr[t] = a.x + (size_t)min(16 * t + (lane & 15), a.M - 1) * a.ldx + (lane >> 4) * 16;
    const v4i* wq[H];
#pragma unroll
    for (int h = 0; h < H; ++h)
        wq[h] = reinterpret_cast<const v4i*>(a.q) +
                ((size_t)h * a.tiles + tile) * nblk * QLM_WAVE + lane;
    v4i acc[H][MT];
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[h][t] = v4i{0, 0, 0, 0};
    for (int b = wave; b < nblk; b += NW * U) {
        v4i w[U][H], x[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int bu = b + u * NW, bc = min(bu, nblk - 1);
#pragma unroll
            for (int h = 0; h < H; ++h) w[u][h] = wq[h][(size_t)bc * QLM_WAVE];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                x[u][t] = *reinterpret_cast<const v4i*>(xr[t] + (size_t)bc * 64);
                if (bu >= nblk) x[u][t] = v4i{0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int t = 0; t < MT; ++t)
                    acc[h][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u][h], x[u][t],
                                                                     acc[h][t], 0, 0, 0);
    }
    // lane l holds outputs n = 4 (l >> 4) + i of row m = l & 15
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                atomicAdd(&sums[((h * MT + t) * 4 + i) * QLM_WAVE + lane], acc[h][t][i]);
    __syncthreads();
    if (wave < MT) {
        v4i s[2];
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                s[h][i] = sums[((h * MT + wave) * 4 + i) * QLM_WAVE + lane];
        if constexpr (H == 1) s[1] = s[0];
        put4<EPI>(a, 16 * wave + (lane & 15), 16 * tile + 4 * (lane >> 4), s[0], s[1]);
    }
}

// BM = 16 WM FM rows of x and BN = 16 WN FN weight rows a workgroup, WM x WN
// waves of FM x FN fragments each.
template <int EPI, int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(WM * WN * QLM_WAVE) void k_a8_tile(A8Args a) {
    constexpr int NW = WM * WN, BF = WN * FN, AF = WM * FM;  // fragments a stage
    constexpr bool SW = EPI == EPI_SWIGLU;
    constexpr int OF = SW ? FN / 2 : FN;  // output fragments of a wave
    __shared__ __attribute__((aligned(16))) v4i smem[(AF + BF) * QLM_WAVE];
    const int lane = threadIdx.x & (QLM_WAVE - 1), wave = threadIdx.x / QLM_WAVE;
    const int wm = wave / WN, wn = wave % WN;
    const int nblk = a.K >> 6;
    const int m0 = blockIdx.y * AF * 16, t0 = blockIdx.x * WN * OF;
    // staged fragment f: rows of x, then weight tiles in the waves' order
    auto src = [&](int f) -> const int8_t* {
        if (f < AF)
            return a.x + (size_t)min(m0 + 16 * f + (lane & 15), a.M - 1) * a.ldx +
                   (lane >> 4) * 16;
        const int g = f - AF, w = g / FN, j = g % FN;
        const int h = SW ? j / OF : 0;
        const int t = min(t0 + w * OF + (SW ? j % OF : j), a.tiles - 1);
        return a.q + ((size_t)(h * a.tiles + t) * nblk * QLM_WAVE + lane) * 16;
    };
    constexpr int L = (AF + BF + NW - 1) / NW;
    const int8_t* from[L];
#pragma unroll
    for (int l = 0; l < L; ++l) from[l] = src(min(wave + l * NW, AF + BF - 1));
    v4i acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = v4i{0, 0, 0, 0};
    for (int b = 0; b < nblk; ++b) {
        v4i in[L];
#pragma unroll
        for (int l = 0; l < L; ++l)
            in[l] = *reinterpret_cast<const v4i*>(
                from[l] + (size_t)b * (wave + l * NW < AF ? 64 : 1024));
        __syncthreads();
#pragma unroll
        for (int l = 0; l < L; ++l)
            if (wave + l * NW < AF + BF) smem[(wave + l * NW) * QLM_WAVE + lane] = in[l];
        __syncthreads();
        v4i x[FM], w[FN];
#pragma unroll
        for (int i = 0; i < FM; ++i) x[i] = smem[(wm * FM + i) * QLM_WAVE + lane];
#pragma unroll
        for (int j = 0; j < FN; ++j) w[j] = smem[(AF + wn * FN + j) * QLM_WAVE + lane];
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] =
                    __builtin_amdgcn_mfma_i32_16x16x64_i8(w[j], x[i], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < OF; ++j)
            put4<EPI>(a, m0 + (wm * FM + i) * 16 + (lane & 15),
                      (t0 + wn * OF + j) * 16 + 4 * (lane >> 4), acc[i][j],
                      acc[i][SW ? j + OF : j]);
}

template <int EPI>
void launch(const A8Args& a, hipStream_t st) {
    constexpr int NW = 8;
    if (a.M <= 16) {
        hipLaunchKernelGGL((k_a8_stream<EPI, 1, NW>), dim3(a.tiles), dim3(NW * QLM_WAVE), 0, st, a);
    } else if (a.M <= 32) {
        hipLaunchKernelGGL((k_a8_stream<EPI, 2, NW>), dim3(a.tiles), dim3(NW * QLM_WAVE), 0, st, a);
    } else if (a.M <= 64) {
        hipLaunchKernelGGL((k_a8_stream<EPI, 4, NW>), dim3(a.tiles), dim3(NW * QLM_WAVE), 0, st, a);
    } else {
        constexpr int ot = EPI == EPI_SWIGLU ? 4 : 8;
        hipLaunchKernelGGL((k_a8_tile<EPI, 2, 2, 4, 4>),
                           dim3((a.tiles + ot - 1) / ot, (a.M + 127) / 128), dim3(256), 0, st, a);
    }
}

}  // namespace

extern "C" size_t qlm_matmul_a8_workspace_bytes(int M, int N, int K, int epilogue) {
    (void)M, (void)N, (void)K, (void)epilogue;
    return 0;
}

extern "C" int qlm_matmul_a8(const int8_t* x, int ldx, const float* x_scales,
                             const int8_t* q_tiles, const float* s_rows, float* y, int ldy, int M,
                             int N, int K, int epilogue, void* work, size_t work_bytes,
                             void* stream) {
    if (!x || !x_scales || !q_tiles || !s_rows || !y || M <= 0 || N <= 0 || K <= 0)
        return QLM_ERR_ARG;
    if (epilogue < EPI_STORE || epilogue > EPI_SWIGLU || ldx < K || ldy < N) return QLM_ERR_ARG;
    if (K % 64 != 0 || K >= 1 << 17 || ldx % 16 != 0 || ldx >= 1 << 23) return QLM_ERR_SHAPE;
    if (((uintptr_t)x | (uintptr_t)q_tiles | (uintptr_t)work) & 15u) return QLM_ERR_SHAPE;
    const size_t need = qlm_matmul_a8_workspace_bytes(M, N, K, epilogue);
    if (need && (!work || work_bytes < need)) return QLM_ERR_ARG;
    const A8Args a{x, x_scales, q_tiles, s_rows, y, ldx, ldy, M, N, K, (N + 15) / 16};
    hipStream_t st = as_stream(stream);
    if (epilogue == EPI_SWIGLU)
        launch<EPI_SWIGLU>(a, st);
    else if (epilogue == EPI_RESID)
        launch<EPI_RESID>(a, st);
    else
        launch<EPI_STORE>(a, st);
    return qlm_launch_status();
}

// Loads this file's code object on the current device now; the runtime
// otherwise loads it at the first launch of one of its kernels.
hipError_t qlm_load_gemm_a8() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>((k_a8_stream<EPI_STORE, 1, 8>)));
}
