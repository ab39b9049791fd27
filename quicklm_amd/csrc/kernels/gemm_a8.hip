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
// Forms, taken by what each is reckoned to cost (plan_of):
//   k_a8_stream  few workgroups' worth of tiles: bound by the way of the bytes
//                to the CUs; every wave streams its share of K by itself.
//   k_a8_tile    as 128 x 128 tiles, two workgroups a CU, K in slices if they
//                are few: bound by the bytes' way too;
//                as 128 x 256 tiles, one workgroup a CU;
//                as 256 x 256 tiles: bound by LDS and the matrix cores, both
//                busy 0.43 us of a block's 0.5 to 0.64, and by the writing of
//                the outputs at a round's end (a quarter of a round of K 4096).
// Measured on an MI355X, operands cold in the caches, us (and the larger of
// the bytes' time at a 4 GiB copy's 4.75 TB/s and the products' at the 2134
// TOP/s of an 8192-wide int8 library product): 1 x 9728 x 2560 SwiGLU 11.6
// (10.5), 16 x 2560 x 9728 10.7 (5.4), 64 x 2560 x 9728 16.0 (5.7), 512 x 2560 x
// 2560 18.5 (3.9), 1000 x 2560 x 2560 19 (6.1), 1000 x 6144 x 2560 28 (14.7),
// 2048 x 9728 x 2560 SwiGLU 104 to 110 from card to card (96), 4096 x 12288 x
// 4096 178 to 190 (193), 8192 x 8192 x 8192 424 (515; 2.6 POP/s).

#include <algorithm>

#include "common.hpp"

namespace {

enum { EPI_STORE = 0, EPI_RESID = 1, EPI_SWIGLU = 2 };
enum { OUT_PART = 3 };  // beside the epilogues: a slice's sums, joined by k_a8_join
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
    int tiles;    // 16-row weight tiles (of a half, for SwiGLU)
    int t_first;  // the launch's first output tile
    int gx, gy, blocks, per_xcd;  // column and row blocks, all (slices too), a XCD's share
    int* part;                    // the slices' sums [slice][M][halves][16 tiles]
    int bslice;                   // 64-column blocks a slice (even), all of them: one slice
};

// Scales of four neighbouring channels (those past the last are copies of it).
__device__ __forceinline__ f32x4u load_scales(const float* sw, int n, int N) {
    if (n + 4 <= N) return *reinterpret_cast<const f32x4u*>(sw + n);
    f32x4u v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = sw[min(n + i, N - 1)];
    return v;
}

// g / (1 + exp(-g)) in a third of the instructions of expf and a division:
// exp2 of the product with log2 e, whose rounding error is put back, and a
// reciprocal with one Newton step; off by 3 + 1 + 1 + 1 roundings at most (the
// exponential, the sum, the reciprocal, the product) down to kDeepGate. The
// epilogue of a 2048 x 9728 SwiGLU took 10 us of a round's 40 with the library's.
// Every fused multiply-add is written out, so all forms give the same bits.
constexpr float kDeepGate = -80.0f;
__device__ __forceinline__ float silu_fast(float g) {
#pragma clang fp contract(off)
    constexpr float kLog2e = 1.44269502e0f, kRest = 1.92596303e-8f, kLn2 = 0.693147182f;
    const float c = fminf(g, 200.0f);  // (an infinite one has no rounding error)
    const float hi = c * -kLog2e;
    const float lo = fmaf(-c, kRest, fmaf(c, -kLog2e, -hi));
    float e = __builtin_amdgcn_exp2f(hi);
    e = fmaf(e * kLn2, lo, e);
    const float d = 1.0f + e;
    float r = __builtin_amdgcn_rcpf(d);
    r = fmaf(fmaf(-d, r, 1.0f), r, r);
    return g * r;
}

// silu(g) * u for a gate below kDeepGate, where 1 + exp(-g) is exp(-g) to fp32
// and soon past its range, its reciprocal below the normal range and flushed:
// g exp(g) u with the exponential as the fourth power of exp(g / 4), multiplied
// in an order in which nothing but the result can leave the range. Off by 8
// roundings of the exponentials and 5 of the products, and by half the spacing
// of subnormal numbers where it is one; 0 for -inf.
__device__ __forceinline__ float silu_deep_mul(float g, float u) {
#pragma clang fp contract(off)
    const float c = fmaxf(g, -300.0f);  // 300 exp(-300) times anything is 0
    const float h = expf(0.25f * c);
    return (c * h) * (u * h * h) * h;
}

// Four results of one row from their sums (SwiGLU: gate and up sums).
template <int EPI>
__device__ __forceinline__ f32x4u scaled(v4i s0, v4i s1, float sx, f32x4u w0, f32x4u w1) {
#pragma clang fp contract(off)
    f32x4u v, u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = (float)s0[i] * sx * w0[i];
        if constexpr (EPI == EPI_SWIGLU) u[i] = (float)s1[i] * sx * w1[i];
    }
    if constexpr (EPI == EPI_SWIGLU) {
        f32x4u y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = silu_fast(v[i]) * u[i];
        if (fminf(fminf(v.x, v.y), fminf(v.z, v.w)) < kDeepGate) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (v[i] < kDeepGate) y[i] = silu_deep_mul(v[i], u[i]);
        }
        return y;
    }
    return v;
}

// What is added to, and a result: rounded as product and as sum in every form.
// Contracted to a fused multiply-add, as the compiler does it in some forms and
// for some columns, a row's bits would depend on the number of rows.
__device__ __forceinline__ float added(float old, float v) {
#pragma clang fp contract(off)
    return old + v;
}
__device__ __forceinline__ f32x4u added(f32x4u old, f32x4u v) {
    return f32x4u{added(old.x, v.x), added(old.y, v.y), added(old.z, v.z), added(old.w, v.w)};
}

// Stores (EPI_RESID: adds) the first `left` of four results.
template <int EPI>
__device__ __forceinline__ void put(float* dst, f32x4u v, int left) {
    if (left >= 4) {
        if constexpr (EPI == EPI_RESID) v = added(*reinterpret_cast<const f32x4u*>(dst), v);
        *reinterpret_cast<f32x4u*>(dst) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (i < left) dst[i] = EPI == EPI_RESID ? added(dst[i], v[i]) : v[i];
}

// Buffer descriptor of a uniform base: a load then takes a lane's 32-bit
// offset and a scalar one, no vector arithmetic on addresses. Reads past
// `bytes` return 0.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* p, unsigned bytes) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return __builtin_amdgcn_make_buffer_rsrc(
        reinterpret_cast<void*>(((uint64_t)hi << 32) | lo), 0, (int)bytes, 0x00027000);
}

// 16 bytes a lane straight into LDS, lane after lane from `to` (uniform).
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t r, char* to, int lane_off,
                                            int uniform_off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)to, 16,
                                             lane_off, uniform_off, 0, 0);
}

// MT 16-row tiles of x against NT weight tiles (SwiGLU: NT gate tiles and
// their up tiles) a workgroup. NW waves take units of two 64-column blocks of K
// in turn, each through a ring of D units of its own in LDS, so nothing waits
// for another wave before the end, when the sums are added in LDS (integers:
// in any order). Loads go straight to LDS in whole cache lines: a lane's 16
// bytes of a row of x straight into the matrix instruction's registers put
// neighbouring lanes on different rows, which the L1 serves four times slower
// (64 x 2560 x 9728 24 us).
template <int EPI, int MT, int NT, int NW, int D>
__global__ __launch_bounds__(NW* QLM_WAVE) void k_a8_stream(A8Args a) {
    constexpr int H = EPI == EPI_SWIGLU ? 2 : 1, F = H * NT;
    constexpr int UNIT = (MT + F) * 2048, L = 2 * (MT + F);  // a unit's bytes and loads
    static_assert(F * MT * 1024 <= NW * D * UNIT, "the sums take the rings' place");
    __shared__ __attribute__((aligned(1024))) char smem[NW * D * UNIT];
    const int lane = threadIdx.x & (QLM_WAVE - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / QLM_WAVE);
    const int nblk = a.K >> 6, t0 = blockIdx.x * NT, m0 = blockIdx.y * (16 * MT);
    const int nunit = (nblk + 1) >> 1, units = (nunit - wave + NW - 1) / NW;  // of this wave

    // x: 8 rows x 128 columns a load, row r's 16-byte piece p at
    // r * 128 + (p ^ (r & 7)) * 16 of its 8-row group. Rows past the last are
    // copies of it, and so are pieces past K (of those before), never multiplied.
    const int rows = min(a.M - m0, 16 * MT);
    const __amdgpu_buffer_rsrc_t rx = make_rsrc(a.x + (size_t)m0 * a.ldx,
                                                (unsigned)(rows - 1) * (unsigned)a.ldx + a.K);
    const int piece = (lane & 7) ^ (lane >> 3);
    const int past = piece >= 4 ? 64 : 0;
    int xoff[2 * MT];
#pragma unroll
    for (int g = 0; g < 2 * MT; ++g)
        xoff[g] = min(8 * g + (lane >> 3), rows - 1) * (int)a.ldx + piece * 16;
    __amdgpu_buffer_rsrc_t rw[F];
#pragma unroll
    for (int f = 0; f < F; ++f)
        rw[f] = make_rsrc(a.q + ((size_t)(f / NT) * a.tiles + min(t0 + f % NT, a.tiles - 1)) *
                                    nblk * 1024,
                          (unsigned)nblk * 1024);
    char* ring = smem + wave * (D * UNIT);
    auto fetch = [&](int i) {  // the wave's unit i
        const int u = wave + i * NW;
        char* to = ring + (i % D) * UNIT;
        const int back = 2 * u + 1 >= nblk ? past : 0;
        const int b1 = min(2 * u + 1, nblk - 1);
#pragma unroll
        for (int f = 0; f < F; ++f) {
            load_to_lds(rw[f], to + f * 2048, lane * 16, u * 2048);
            load_to_lds(rw[f], to + f * 2048 + 1024, lane * 16, b1 * 1024);
        }
#pragma unroll
        for (int g = 0; g < 2 * MT; ++g)
            load_to_lds(rx, to + F * 2048 + g * 1024, xoff[g] - back, u * 128);
    };
    v4i acc[F][MT];
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[f][t] = v4i{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < D; ++i)
        if (i < units) fetch(i);
    const int xl = F * 2048 + ((lane & 15) >> 3) * 1024 + (lane & 7) * 128 +
                   ((lane >> 4) ^ (lane & 7)) * 16;
#pragma unroll 1
    for (int i = 0; i < units; ++i) {
        if (units - i >= D)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(L * (D - 1)) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const char* at = ring + (i % D) * UNIT;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (h && 2 * (wave + i * NW) + 1 >= nblk) break;
            v4i w[F], x[MT];
#pragma unroll
            for (int f = 0; f < F; ++f)
                w[f] = *reinterpret_cast<const v4i*>(at + f * 2048 + h * 1024 + lane * 16);
#pragma unroll
            for (int t = 0; t < MT; ++t)
                x[t] = *reinterpret_cast<const v4i*>(at + (xl ^ (h << 6)) + t * 2048);
#pragma unroll
            for (int f = 0; f < F; ++f)
#pragma unroll
                for (int t = 0; t < MT; ++t)
                    acc[f][t] =
                        __builtin_amdgcn_mfma_i32_16x16x64_i8(w[f], x[t], acc[f][t], 0, 0, 0);
        }
        // the unit is read: its place takes the unit after the ring's last
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (i + D < units) fetch(i + D);
    }
    int* sums = reinterpret_cast<int*>(smem);
    __syncthreads();  // every ring is read
    for (int i = threadIdx.x; i < F * MT * 256; i += NW * QLM_WAVE) sums[i] = 0;
    __syncthreads();
    // lane l holds outputs n = 4 (l >> 4) + i of row m = l & 15
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                atomicAdd(&sums[((f * MT + t) * 4 + i) * QLM_WAVE + lane], acc[f][t][i]);
    __syncthreads();
    for (int p = wave; p < NT * MT; p += NW) {
        const int f = p / MT, t = p % MT;
        v4i s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                s[h][i] = sums[(((f + (h & (H - 1)) * NT) * MT + t) * 4 + i) * QLM_WAVE + lane];
        const int m = m0 + 16 * t + (lane & 15), n = 16 * (t0 + f) + 4 * (lane >> 4);
        if (m < a.M && n < a.N) {
            const f32x4u w0 = load_scales(a.sw, n, a.N);
            const f32x4u w1 = H == 2 ? load_scales(a.sw + a.N, n, a.N) : w0;
            put<EPI>(a.y + (size_t)m * a.ldy + n, scaled<EPI>(s[0], s[1], a.sx[m], w0, w1),
                     a.N - n);
        }
    }
}

__device__ __forceinline__ void mma(v4i& acc, v4i w, v4i x) {
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, acc, 0, 0, 0);
}

// BM = 16 WM FM rows of x and BN = 16 WN FN weight rows a workgroup, WM x WN
// waves of FM x FN fragments each.
//
// LDS holds WD blocks (64 columns) of weight fragments and XU units (128
// columns) of x. A load of x takes 8 rows x 128 columns, whole cache lines:
// loads of 16 rows x 64 columns, the fragments themselves, took half as long
// again. Row r's 16-byte piece p lies at r * 128 + (p ^ (r & 7)) * 16 of its
// 8-row group, so that the 8 lanes of an LDS access meet every bank once.
template <int EPI, bool SW, int WM, int WN, int FM, int FN, int WD, int XU>
__global__ __launch_bounds__(WM* WN* QLM_WAVE, 2) void k_a8_tile(A8Args a) {
    constexpr int NW = WM * WN, BF = WN * FN, AF = WM * FM;  // fragments of a block
    constexpr int OF = SW ? FN / 2 : FN;  // output fragments of a wave
    constexpr int LX = AF / NW, LW = BF / NW, L = LX + LW;  // a wave's loads a block
    static_assert(AF % NW == 0 && BF % NW == 0 && FN % 2 == 0 && FN / 2 <= FM, "tile shape");
    constexpr int XUNIT = AF * 2048, WBLK = BF * 1024, W0 = XU * XUNIT;
    __shared__ __attribute__((aligned(1024))) char smem[XU * XUNIT + WD * WBLK];
    const int lane = threadIdx.x & (QLM_WAVE - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / QLM_WAVE);
    const int wm = wave / WN, wn = wave % WN;
    // Workgroups go to the 8 XCDs in turn: XCD i takes the i-th eighth of the
    // blocks, in bands of BAND row blocks (column by column inside a band).
    constexpr int BAND = 4;
    int t = (int)(blockIdx.x & 7) * a.per_xcd + (int)(blockIdx.x >> 3);
    if (t >= a.blocks) return;
    const int slice = t / (a.gx * a.gy);
    t -= slice * a.gx * a.gy;
    const int band = t / (BAND * a.gx);
    const int bh = min(BAND, a.gy - BAND * band);
    t -= band * BAND * a.gx;
    const int m0 = (BAND * band + t % bh) * AF * 16;
    const int t0 = a.t_first + (t / bh) * WN * OF;  // first output tile
    // this slice's blocks of K
    const int b0 = slice * a.bslice, kblk = a.K >> 6, nblk = min(kblk - b0, a.bslice);

    // x: the unit's 8-row groups, LX of each half of them a wave. Rows past the
    // last are copies of it; where K ends in the middle of a unit, so are the
    // pieces past it (of those before), and none of them is multiplied.
    const int rows = min(a.M - m0, AF * 16);
    const __amdgpu_buffer_rsrc_t rx = make_rsrc(
        a.x + (size_t)m0 * a.ldx + b0 * 64, (unsigned)(rows - 1) * (unsigned)a.ldx + a.K - b0 * 64);
    const int piece = (lane & 7) ^ (lane >> 3);
    const int past = piece >= 4 ? 64 : 0;
    int xoff[LX], xstep[LX];  // first half of the groups, and on to the second
#pragma unroll
    for (int l = 0; l < LX; ++l) {
        const int r = 8 * (wave * LX + l) + (lane >> 3);
        xoff[l] = min(r, rows - 1) * (int)a.ldx + piece * 16;
        xstep[l] = min(r + 8 * AF, rows - 1) * (int)a.ldx + piece * 16 - xoff[l];
    }
    // weights: staged fragments in the waves' order (gate tiles, up tiles)
    __amdgpu_buffer_rsrc_t rw[LW];
#pragma unroll
    for (int l = 0; l < LW; ++l) {
        const int f = wave * LW + l, w = f / FN, j = f % FN, h = SW ? j / OF : 0;
        const int tl = min(t0 + w * OF + (SW ? j % OF : j), a.tiles - 1);
        rw[l] = make_rsrc(a.q + (((size_t)h * a.tiles + tl) * kblk + b0) * 1024,
                          (unsigned)nblk * 1024);
    }
    const int woff = lane * 16;
    const int last_unit = (nblk - 1) >> 1;
    // load l of half unit `half` of x into unit slot `slot`, of block b's weights
    auto fetch_x1 = [&](int l, int half, int slot) {
        const int h = half & 1, u = min(half >> 1, last_unit);
        const int back = u == last_unit && (nblk & 1) ? past : 0;
        load_to_lds(rx, smem + slot * XUNIT + (h * AF + wave * LX + l) * 1024,
                    xoff[l] + (xstep[l] & -h) - back, u * 128);
    };
    auto fetch_w1 = [&](int l, int b, int slot) {
        load_to_lds(rw[l], smem + W0 + slot * WBLK + (wave * LW + l) * 1024, woff,
                    min(b, nblk - 1) * 1024);
    };
    auto fetch_x = [&](int half, int slot) {
#pragma unroll
        for (int l = 0; l < LX; ++l) fetch_x1(l, half, slot);
    };
    v4i acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = v4i{0, 0, 0, 0};

    // fragment i of x: row r = lane & 15, piece lane >> 4 of the block's half
    const int xl = ((wm * FM * 2) + ((lane & 15) >> 3)) * 1024 + (lane & 7) * 128 +
                   ((lane >> 4) ^ (lane & 7)) * 16;
    auto read_x = [&](int at, int i) {
        return *reinterpret_cast<const v4i*>(smem + at + i * 2048);
    };
    auto read_w = [&](int at, int j) {
        return *reinterpret_cast<const v4i*>(smem + at + j * 1024);
    };
    const int wl = W0 + wn * FN * 1024 + lane * 16;

    // A wave's fragments of block b sit in one set of registers. Its columns
    // are multiplied in two halves; a register is read anew, for block b + 1,
    // as soon as its last product is issued:
    //   first half   the upper columns' weights of block b
    //   barrier b    block b is read by everyone, block b + 1 has arrived
    //   second half  the lower columns' weights and x of block b + 1
    // so every read has half a block of products to return. Weights of block
    // b + WD and half a unit of x are requested after barrier b, spread over a
    // block's length: a burst of them holds up the products behind it.
    constexpr int HN = FN / 2;
    constexpr int XH = 2 * XU - 1;  // iteration b requests x's half unit b + XH
    // iterations whose requests may be under way when block b + 1 is needed
    constexpr int AHEAD = (WD - 1 < 2 * XU - 3 ? WD - 1 : 2 * XU - 3) - 1;
    static_assert(AHEAD >= 0, "ring depths");
    constexpr int L1 = L / 4;  // a block's requests in its second half; the others follow it
    v4i x[FM], w[FN];
#pragma unroll
    for (int h = 0; h < XH - WD; ++h) fetch_x(h, (h >> 1) % XU);
#pragma unroll
    for (int b = -WD; b < 0; ++b)
#pragma unroll
        for (int l = 0; l < (b < -1 ? L : L1); ++l) {
            if (l < LW)
                fetch_w1(l, b + WD, b + WD);
            else if (b + XH >= 0)
                fetch_x1(l - LW, b + XH, ((b + XH) >> 1) % XU);
        }
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(L * AHEAD) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < FM; ++i) {  // in the order of the second half below
        if (2 * i < HN) w[2 * i] = read_w(wl, 2 * i);
        if (2 * i + 1 < HN) w[2 * i + 1] = read_w(wl, 2 * i + 1);
        x[i] = read_x(xl, i);
    }
    int ws = 0;               // slot of block b's weights
    int xs = 0;               // slot of block b's unit of x
    int xf = (XH >> 1) % XU;  // slot of half unit b + XH
    int ws0 = WD - 1, xf0 = ((XH - 1) >> 1) % XU;  // those that block b - 1 requests into
#pragma unroll 1
    for (int b = 0; b < nblk; ++b) {
        auto request = [&](int l, int b0) {
            if (l < LW)
                fetch_w1(l, b0 + WD, ws0);
            else
                fetch_x1(l - LW, b0 + XH, xf0);
        };
        int wa = wl + ws * WBLK;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
#pragma unroll
            for (int j = 0; j < HN; ++j) mma(acc[i][j], w[j], x[i]);
            if (i < HN) w[HN + i] = read_w(wa, HN + i);
#pragma unroll
            for (int l = L1 + i * (L - L1) / FM; l < L1 + (i + 1) * (L - L1) / FM; ++l)
                request(l, b - 1);
            __builtin_amdgcn_sched_barrier(0);
        }
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(L * AHEAD) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        ws0 = ws;
        xf0 = xf;
        if ((b + XH) & 1) xf = xf + 1 == XU ? 0 : xf + 1;
        ws = ws + 1 == WD ? 0 : ws + 1;
        if (b & 1) xs = xs + 1 == XU ? 0 : xs + 1;
        wa = wl + ws * WBLK;
        const int xa = (xl ^ (((b + 1) & 1) << 6)) + xs * XUNIT;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
#pragma unroll
            for (int j = 0; j < HN; ++j) mma(acc[i][HN + j], w[HN + j], x[i]);
            if (2 * i < HN) w[2 * i] = read_w(wa, 2 * i);
            if (2 * i + 1 < HN) w[2 * i + 1] = read_w(wa, 2 * i + 1);
            x[i] = read_x(xa, i);
#pragma unroll
            for (int l = i * L1 / FM; l < (i + 1) * L1 / FM; ++l) request(l, b);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing lands after the end
    const int ml = m0 + wm * FM * 16 + (lane & 15);
    const int nl = (t0 + wn * OF) * 16 + 4 * (lane >> 4);
    if constexpr (EPI == OUT_PART) {
        const int ldp = 16 * a.tiles, H = SW ? 2 : 1;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            int* p = a.part + ((size_t)slice * a.M + ml + 16 * i) * H * ldp + nl;
#pragma unroll
            for (int j = 0; j < FN; ++j)
                if (ml + 16 * i < a.M && nl + 16 * (j % OF) < ldp)
                    *reinterpret_cast<v4i*>(p + (j / OF) * ldp + 16 * (j % OF)) = acc[i][j];
        }
        return;
    }
    // every scale is requested before the first output is formed
    float sx[FM];
#pragma unroll
    for (int i = 0; i < FM; ++i) sx[i] = a.sx[min(ml + 16 * i, a.M - 1)];
    f32x4u s0[OF], s1[OF];
#pragma unroll
    for (int j = 0; j < OF; ++j) {
        s0[j] = load_scales(a.sw, nl + 16 * j, a.N);
        if constexpr (SW) s1[j] = load_scales(a.sw + a.N, nl + 16 * j, a.N);
    }
    // inside the matrix nothing of a load or store is conditional; what is added
    // to is requested half the rows at a time (row by row each waits in turn:
    // 2862 x 3428 x 2048 47 us)
    const bool inside = m0 + AF * 16 <= a.M && (t0 + WN * OF) * 16 <= a.N;
    constexpr int G = FM / 2;
#pragma unroll
    for (int g = 0; g < FM; g += G) {
        f32x4u old[G][OF];
        float* y = a.y + (size_t)(ml + 16 * g) * a.ldy + nl;
        if constexpr (EPI == EPI_RESID) {
            if (inside) {
#pragma unroll
                for (int i = 0; i < G; ++i)
#pragma unroll
                    for (int j = 0; j < OF; ++j)
                        old[i][j] =
                            *reinterpret_cast<const f32x4u*>(y + 16 * i * a.ldy + 16 * j);
            }
        }
#pragma unroll
        for (int i = 0; i < G; ++i) {
#pragma unroll
            for (int j = 0; j < OF; ++j) {
                const f32x4u v = scaled<EPI>(acc[g + i][j], acc[g + i][SW ? j + OF : j], sx[g + i],
                                             s0[j], SW ? s1[j] : s0[j]);
                if (inside)
                    *reinterpret_cast<f32x4u*>(y + 16 * j) =
                        EPI == EPI_RESID ? added(old[i][j], v) : v;
                else if (ml + 16 * (g + i) < a.M)
                    put<EPI>(y + 16 * j, v, a.N - (nl + 16 * j));
            }
            y += 16 * a.ldy;
        }
    }
}

// The slices' sums of four neighbouring outputs a thread, in 32-bit integers
// (order does not matter), then the epilogue.
constexpr int kJoinThreads = 256;
template <int EPI>
__global__ __launch_bounds__(kJoinThreads) void k_a8_join(A8Args a, int slices) {
    constexpr int H = EPI == EPI_SWIGLU ? 2 : 1;
    const int q4 = 4 * a.tiles;  // groups of four of a row
    const long long i = (long long)blockIdx.x * kJoinThreads + threadIdx.x;
    if (i >= (long long)a.M * q4) return;
    const int m = (int)(i / q4), n = 4 * (int)(i - (long long)m * q4);
    const int ldp = 16 * a.tiles;
    const int* p = a.part + (size_t)m * H * ldp + n;
    const size_t step = (size_t)a.M * H * ldp;
    v4i s[2] = {v4i{0, 0, 0, 0}, v4i{0, 0, 0, 0}};
    constexpr int U = 4;  // slices in flight
    for (int k = 0; k < slices; k += U) {
        v4i v[U][H];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < H; ++h)
                v[u][h] = *reinterpret_cast<const v4i*>(p + min(k + u, slices - 1) * step + h * ldp);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < H; ++h)
                if (k + u < slices) s[h] += v[u][h];
    }
    if (n >= a.N) return;
    const f32x4u w0 = load_scales(a.sw, n, a.N);
    const f32x4u w1 = H == 2 ? load_scales(a.sw + a.N, n, a.N) : w0;
    put<EPI>(a.y + (size_t)m * a.ldy + n, scaled<EPI>(s[0], s[1], a.sx[m], w0, w1), a.N - n);
}

int ceil_div(int a, int b) { return (a + b - 1) / b; }

// A streaming form: 16-row tiles of x and weight tiles a workgroup, its waves
// and the units of their rings; its time by the plan's reckoning.
struct StreamShape {
    int mt, nt, waves, depth;
    double us;
};

// The form of a call. A workgroup reads all of its rows of x and weights, and a
// CU takes in 62 KB a us of them, whoever shares it; beyond one workgroup a CU,
// those whose rings fill the LDS also wait for each other. Measured on an
// MI355X with operands cold (2560 x 2560 weights, us): 64 rows 5.9 in groups of
// 16, 5.5 in one of 64; 128 rows 7.2 in groups of 64 x 2 tiles, 9.1 of 16; 400
// rows 11.4 in groups of 48 x 2 tiles, 13.8 of 64 x 2, 20 of 16.
StreamShape stream_shape(int M, int tiles, int K, int halves) {
    // Long rows of tiles: workgroups that share a CU (16 x 2 x 9728 x 2560:
    // 11.9 us with 4 waves, 14.6 with 8), and with thousands of tiles two of
    // them a workgroup, to read x half as often (16 x 151936 x 2560: 75, 80).
    const bool many = tiles * halves > 512, most = M > 1 && tiles * halves >= 4096;
    StreamShape best{0, 0, 0, 0, 1e30};
    auto offer = [&](int mt, int nt, int waves, int depth) {
        const double groups = (double)ceil_div(tiles, nt) * ceil_div(M, 16 * mt);
        const double kb = K * 16.0 * (mt + nt * halves) / 1024;
        const bool shares = waves * depth * (mt + nt * halves) * 2 <= 40;  // KB of LDS
        const double rounds = groups <= 256 ? 1 : groups / 256 + (shares ? 0 : 0.4);
        // (a workgroup's own start and end, and its outputs' way to memory)
        const double us = 2.6 + rounds * kb / (halves > 1 ? 48 : 62) + 1.2 * (rounds - 1) +
                          2e-7 * 4 * M * tiles * 16;
        if (us < best.us) best = {mt, nt, waves, depth, us};
    };
    if (most && M <= 32) {
        M <= 16 ? offer(1, 2, 4, 2) : offer(2, 2, 2, 2);
        return best;
    }
    offer(1, 1, many ? 4 : 8, 2);
    if (M > 16) offer(2, 1, many ? 4 : 8, 2);
    if (M > 32) offer(3, 1, 4, many ? 1 : 2);
    if (M > 48) offer(4, 1, many ? 2 : 4, 2);
    if (M > 64) offer(3, 2, 4, 1);
    if (M > 64 && halves == 1) offer(4, 2, 8, 1);
    return best;
}

// How a call runs. Times in us, measured on an MI355X with operands cold in
// the caches; kblk 64-column blocks of K.
enum { K_STREAM = 0, K_T128 = 1, K_WIDE = 2, K_T256 = 3 };  // (wide: 128 x 256)
struct Plan {
    int kind;
    int cols, rest;      // K_T256: of the first columns (256 each), the others' kind
    int slices, bslice;  // of K, and 64-column blocks in each (K_T128 alone)
};

constexpr int kMaxRows = 1 << 20, kMaxOutputs = 1 << 23;  // tile numbers fit 32 bits
constexpr int kSliceMinRows = 32, kSliceMinBlocks = 8, kSliceMost = 8, kSliceTiles = 256;

// 128 x 128 tiles, two workgroups a CU: alone on its CU a workgroup takes
// 0.275 a block, beside another twice as long; after the first 512 tiles the
// CUs are no longer in step. (Its 16 KB a block come in at 60 KB a us, as in
// the streaming form. Eight waves a workgroup, four on every other block, gain
// a tenth with the GPU half empty and lose a fifth with it full; deeper rings
// and a wave that touches the lines ahead gain nothing.)
double cost128(int n, int kblk) {
    const int full = n / 512, rest = n % 512;
    const double round = 9.5 + 0.57 * kblk;
    if (rest <= 256) return full * round + (rest ? 6.5 + 0.275 * kblk : 0);
    return full * round + (full ? rest / 512.0 * round : rest <= 384 ? 9 + 0.5 * kblk : round);
}
// 128 x 256 tiles, one workgroup a CU: the outputs of two of the above for
// three quarters of their bytes (512 x 9728 x 2560 26.7 us instead of 30.2).
double cost_wide(int n, int kblk) {
    const int full = n / 256, rest = n % 256;
    return full * (10.5 + 0.42 * kblk) + (rest ? 10.5 + (0.35 + 0.07 * rest / 256.0) * kblk : 0);
}
// 256 x 256 tiles, one workgroup a CU: 0.51 a block while the other CUs idle,
// 0.64 with all of them.
double cost256(int n, int kblk) {
    return ceil_div(n, 256) * (16.5 + (0.5 + 0.14 * std::min(1.0, n / 256.0)) * kblk);
}

Plan plan_of(int M, int N, int K, int epilogue) {
    const int halves = epilogue == EPI_SWIGLU ? 2 : 1, kblk = K / 64;
    const int tiles = ceil_div(N, 16);
    Plan best{K_STREAM, 0, 0, 1, kblk};
    double least = 1e30;
    const int gx1 = ceil_div(tiles, 8 / halves), gy1 = ceil_div(M, 128);
    const int gx2 = ceil_div(tiles, 16 / halves), gy2 = ceil_div(M, 256);
    auto offer = [&](double us, Plan p) {
        if (us < least) least = us, best = p;
    };
    offer(stream_shape(M, tiles, K, halves).us, best);
    if (M > kSliceMinRows) {
        for (int s = 1; s <= kSliceMost; s *= 2) {
            if (s > 1 && (gx1 * gy1 * s > kSliceTiles || kblk < kSliceMinBlocks * s)) break;
            // the slices' sums are written and read back, 3.3 MB a us
            const double join = s == 1 ? 0 : 2.5 + 1.2e-6 * s * M * halves * N;
            const int bs = s == 1 ? kblk : ceil_div(ceil_div(kblk, s), 2) * 2;
            offer(cost128(gx1 * gy1 * s, bs) + join, Plan{K_T128, 0, 0, ceil_div(kblk, bs), bs});
        }
        offer(cost_wide(gx2 * gy1, kblk), Plan{K_WIDE, 0, 0, 1, kblk});
    }
    if (M > 128) {
        offer(cost256(gx2 * gy2, kblk), Plan{K_T256, gx2, 0, 1, kblk});
        // full rounds of 256 tiles, and the columns left over as smaller ones
        const int full = gx2 * gy2 / 256 * 256 / gy2;
        if (full > 0 && full < gx2) {
            const double most = cost256(full * gy2, kblk);
            offer(most + cost128((gx1 - 2 * full) * gy1, kblk), Plan{K_T256, full, K_T128, 1, kblk});
            offer(most + cost_wide((gx2 - full) * gy1, kblk), Plan{K_T256, full, K_WIDE, 1, kblk});
        }
    }
    return best;
}

// Bytes that a sliced call writes of its workspace.
size_t part_bytes(const Plan& p, int M, int N, int epilogue) {
    return (size_t)p.slices * M * (epilogue == EPI_SWIGLU ? 2 : 1) * (ceil_div(N, 16) * 16) * 4;
}

// Columns [first, last), 256 each, as tiles of the kind.
template <int EPI, int KIND>
void launch_tile(A8Args a, const Plan& p, int first, int last, hipStream_t st) {
    constexpr bool SW = EPI == EPI_SWIGLU;
    constexpr int WIDTH = KIND == K_T128 ? 128 : 256, OT = WIDTH / 16 / (SW ? 2 : 1);
    a.t_first = first * (16 / (SW ? 2 : 1));
    a.gx = ceil_div(std::min(a.tiles, last * (16 / (SW ? 2 : 1))) - a.t_first, OT);
    a.gy = ceil_div(a.M, KIND == K_T256 ? 256 : 128);
    a.blocks = a.gx * a.gy * p.slices;
    a.per_xcd = ceil_div(a.blocks, 8);
    a.bslice = p.bslice;
    const dim3 grid(8 * a.per_xcd), threads((KIND == K_T128 ? 4 : 8) * QLM_WAVE);
    if constexpr (KIND == K_T256) {
        hipLaunchKernelGGL((k_a8_tile<EPI, SW, 2, 4, 8, 4, 4, 3>), grid, threads, 0, st, a);
    } else if constexpr (KIND == K_WIDE) {
        hipLaunchKernelGGL((k_a8_tile<EPI, SW, 2, 4, 4, 4, 4, 4>), grid, threads, 0, st, a);
    } else if (p.slices == 1) {
        hipLaunchKernelGGL((k_a8_tile<EPI, SW, 2, 2, 4, 4, 4, 3>), grid, threads, 0, st, a);
    } else {
        hipLaunchKernelGGL((k_a8_tile<OUT_PART, SW, 2, 2, 4, 4, 4, 3>), grid, threads, 0, st, a);
        const long long groups = (long long)a.M * 4 * a.tiles;
        hipLaunchKernelGGL((k_a8_join<EPI>),
                           dim3((unsigned)((groups + kJoinThreads - 1) / kJoinThreads)),
                           dim3(kJoinThreads), 0, st, a, p.slices);
    }
}

template <int EPI, int MT, int NT, int NW, int D>
void launch_stream(const A8Args& a, hipStream_t st) {
    hipLaunchKernelGGL((k_a8_stream<EPI, MT, NT, NW, D>),
                       dim3(ceil_div(a.tiles, NT), ceil_div(a.M, 16 * MT)), dim3(NW * QLM_WAVE), 0,
                       st, a);
}

template <int EPI>
void launch(const A8Args& a, const Plan& p, hipStream_t st) {
    const int all = ceil_div(a.tiles, EPI == EPI_SWIGLU ? 8 : 16);
    if (p.kind == K_T256) {
        launch_tile<EPI, K_T256>(a, p, 0, p.cols, st);
        if (p.rest == K_T128) launch_tile<EPI, K_T128>(a, p, p.cols, all, st);
        if (p.rest == K_WIDE) launch_tile<EPI, K_WIDE>(a, p, p.cols, all, st);
        return;
    }
    if (p.kind == K_WIDE) return launch_tile<EPI, K_WIDE>(a, p, 0, all, st);
    if (p.kind == K_T128) return launch_tile<EPI, K_T128>(a, p, 0, all, st);
    const StreamShape f = stream_shape(a.M, a.tiles, a.K, EPI == EPI_SWIGLU ? 2 : 1);
    if (f.mt == 1 && f.nt == 2) return launch_stream<EPI, 1, 2, 4, 2>(a, st);
    if (f.mt == 1 && f.waves == 8) return launch_stream<EPI, 1, 1, 8, 2>(a, st);
    if (f.mt == 1) return launch_stream<EPI, 1, 1, 4, 2>(a, st);
    if (f.mt == 2 && f.nt == 2) return launch_stream<EPI, 2, 2, 2, 2>(a, st);
    if (f.mt == 2 && f.waves == 8) return launch_stream<EPI, 2, 1, 8, 2>(a, st);
    if (f.mt == 2) return launch_stream<EPI, 2, 1, 4, 2>(a, st);
    if (f.mt == 3 && f.nt == 2) return launch_stream<EPI, 3, 2, 4, 1>(a, st);
    if (f.mt == 3 && f.depth == 2) return launch_stream<EPI, 3, 1, 4, 2>(a, st);
    if (f.mt == 3) return launch_stream<EPI, 3, 1, 4, 1>(a, st);
    if (f.nt == 2) {  // (not SwiGLU: see stream_shape)
        if constexpr (EPI != EPI_SWIGLU) launch_stream<EPI, 4, 2, 8, 1>(a, st);
        return;
    }
    if (f.waves == 4) return launch_stream<EPI, 4, 1, 4, 2>(a, st);
    launch_stream<EPI, 4, 1, 2, 2>(a, st);
}

}  // namespace

extern "C" size_t qlm_matmul_a8_workspace_bytes(int M, int N, int K, int epilogue) {
    if (M <= 0 || N <= 0 || K <= 0 || K % 64 != 0 || epilogue < EPI_STORE || epilogue > EPI_SWIGLU)
        return 0;
    // Slices are cut for at most 256 tiles of 128 x 128 sums in all, at most 8
    // of a call: a bound that never falls with M.
    if (M <= kSliceMinRows || K / 64 < 2 * kSliceMinBlocks) return 0;
    const size_t sums = (size_t)M * (epilogue == EPI_SWIGLU ? 2 : 1) * (((size_t)N + 15) / 16 * 16);
    const size_t most = (size_t)kSliceTiles * 128 * 128;
    return 4 * (kSliceMost * sums < most ? kSliceMost * sums : most);
}

extern "C" int qlm_matmul_a8(const int8_t* x, int ldx, const float* x_scales,
                             const int8_t* q_tiles, const float* s_rows, float* y, int ldy, int M,
                             int N, int K, int epilogue, void* work, size_t work_bytes,
                             void* stream) {
    if (!x || !x_scales || !q_tiles || !s_rows || !y || M <= 0 || N <= 0 || K <= 0)
        return QLM_ERR_ARG;
    if (epilogue < EPI_STORE || epilogue > EPI_SWIGLU || ldx < K || ldy < N) return QLM_ERR_ARG;
    if (K % 64 != 0 || K >= 1 << 17 || ldx % 16 != 0 || ldx >= 1 << 23) return QLM_ERR_SHAPE;
    if (M >= kMaxRows || N >= kMaxOutputs) return QLM_ERR_SHAPE;
    if (((uintptr_t)x | (uintptr_t)q_tiles | (uintptr_t)work) & 15u) return QLM_ERR_SHAPE;
    const Plan p = plan_of(M, N, K, epilogue);
    const size_t need = qlm_matmul_a8_workspace_bytes(M, N, K, epilogue);
    if (need && (!work || work_bytes < need)) return QLM_ERR_ARG;
    if (p.slices > 1 && part_bytes(p, M, N, epilogue) > work_bytes) return QLM_ERR_ARG;
    A8Args a{};
    a.x = x;
    a.sx = x_scales;
    a.q = q_tiles;
    a.sw = s_rows;
    a.y = y;
    a.ldx = ldx;
    a.ldy = ldy;
    a.M = M;
    a.N = N;
    a.K = K;
    a.tiles = (N + 15) / 16;
    a.part = static_cast<int*>(work);
    hipStream_t st = as_stream(stream);
    if (epilogue == EPI_SWIGLU)
        launch<EPI_SWIGLU>(a, p, st);
    else if (epilogue == EPI_RESID)
        launch<EPI_RESID>(a, p, st);
    else
        launch<EPI_STORE>(a, p, st);
    return qlm_launch_status();
}

// Loads this file's code object on the current device now; the runtime
// otherwise loads it at the first launch of one of its kernels.
hipError_t qlm_load_gemm_a8() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(k_a8_join<EPI_STORE>));
}
