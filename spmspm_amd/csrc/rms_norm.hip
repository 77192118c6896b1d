// RMS_Norm, W8_Quantize (w8_api.h): a row of 16-bit numbers is read once, held in registers, reduced and written.
//
// Mathematics.  With t = h w the codes of a normed row are those of t itself, since the division by the rms scales all of a row
// alike: rint(127 t / max|t|).  So they do not depend on the sum of squares, whose rounding varies with its order, and one pass
// takes the sum of h^2 and the maximum of |t| together.
//
// Bound by memory: 2 bytes for x, 2 for the residual and 2 for h, 2 or 1 for the result of every element.  4099 rows of 9216 with a
// residual: 54 us and 5.6 TB/s into 16 bits, 52 us and 5.1 TB/s into 8; 4096 rows of 20480 to 8 bits 43 us, 5.9 TB/s; one row of
// 5120 3.2 us, which is latency.
#include "w8_common.hiph"

#include <algorithm>

namespace decode {
namespace {

struct NormArgs {
    const uint16_t *x, *residual, *weight;
    uint16_t *      h, *y;
    int8_t*         codes;
    float*          scales;
    int64_t         x_stride, r_stride, h_stride, y_stride, c_stride;
    int             N, K;
    float           eps;
};

__device__ __forceinline__ void store8(uint16_t* p, shortx8 v, int left)
{
    if (left >= 8) {
        *reinterpret_cast<loose8*>(p) = v;
        return;
    }
    for (int i = 0; i < 7; ++i)
        if (i < left)
            p[i] = v[i];
}

template <bool BF16>
__device__ __forceinline__ float up(uint16_t v)
{
    return from16(v, BF16);
}

template <bool BF16>
__device__ __forceinline__ uint16_t down(float x)
{
    return BF16 ? __builtin_bit_cast(uint16_t, (__bf16)x) : __builtin_bit_cast(uint16_t, (_Float16)x);
}

// Sum of `a` and maximum of `b` over the WAVES waves of a row, in every lane.
template <int WAVES>
__device__ __forceinline__ void reduce(float& a, unsigned& b, float (*sum)[16], unsigned (*top)[16], int turn)
{
    for (int d = 32; d > 0; d >>= 1) {
        a += __shfl_xor(a, d);
        b = max(b, (unsigned)__shfl_xor((int)b, d));
    }
    if constexpr (WAVES > 1) {
        const int wave = threadIdx.x / kWave;
        if (threadIdx.x % kWave == 0)
            sum[turn][wave] = a, top[turn][wave] = b;
        __syncthreads();
        a = 0.f, b = 0;
        for (int w = 0; w < WAVES; ++w)
            a += sum[turn][w], b = max(b, top[turn][w]);
    }
}

// One row by WAVES waves, V vectors of eight elements a lane in registers; V = 0: a row of any length, read twice.  Without NORM the row
// is only rounded to 8 bits.
template <bool BF16, bool NORM, bool QUANT, int WAVES, int V>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * kWave) void rms_norm(NormArgs a)
{
    constexpr int      kThreads = WAVES * kWave, kHeld = V > 0 ? V : 1;
    __shared__ float    sum[2][16];
    __shared__ unsigned top[2][16];
    const int           lane = WAVES == 1 ? threadIdx.x % kWave : threadIdx.x;
    const int64_t       row  = WAVES == 1 ? (int64_t)blockIdx.x * 4 + threadIdx.x / kWave : (int64_t)blockIdx.x;
    if (WAVES == 1 && row >= a.N)
        return;
    const uint16_t* x = a.x + row * a.x_stride;
    const uint16_t* r = a.residual + row * a.r_stride;
    uint16_t*       h = a.h + row * a.h_stride;
    const int       n = V > 0 ? V : (a.K + kThreads * 8 - 1) / (kThreads * 8);

    shortx8 held[kHeld], gain[kHeld];
    // The vector at element e as the norm sees it; what lies behind the row is 0.
    auto fetch = [&](int e) {
        shortx8 v = load8(x, e, a.K);
        if (NORM && a.residual != nullptr) {
            const shortx8 d = load8(r, e, a.K);
            for (int i = 0; i < 8; ++i)
                v[i] = down<BF16>(up<BF16>(v[i]) + up<BF16>(d[i]));
        }
        return v;
    };
    float    squares = 0.f;
    unsigned most    = 0; // bits of max |t|: an infinity or a NaN is larger than every number
    auto     take    = [&](float& sum, shortx8 v, shortx8 w) {
        for (int i = 0; i < 8; ++i) {
            const float f = up<BF16>(v[i]), t = NORM ? f * up<BF16>(w[i]) : f;
            if (NORM)
                sum = __builtin_fmaf(f, f, sum);
            if (QUANT)
                most = max(most, __float_as_uint(t) & 0x7fffffffu);
        }
    };
    // Rows that are read twice have up to 2048 vectors a lane: sums of vectors, of 32 of those, and of these, since in one sum the
    // roundings of thousands of additions of like numbers go one way (2^24 of them: off by 2.4e-4).
    float sums = 0.f;
    auto  fold = [&](float& total, float sum, int j) {
        sums += sum;
        if (j % 32 == 31 || j == n - 1)
            total += sums, sums = 0.f;
    };
#pragma unroll kHeld
    for (int j = 0; j < n; ++j) {
        const int e = (j * kThreads + lane) * 8, k = V > 0 ? j : 0;
        held[k] = 0, gain[k] = 0;
        if (e < a.K) {
            held[k] = fetch(e);
            if (NORM)
                gain[k] = load8(a.weight, e, a.K);
        }
        if (NORM && a.h != nullptr && e < a.K)
            store8(h + e, held[k], a.K - e);
        if (V == 0) {
            float sum = 0.f;
            take(sum, held[0], gain[0]);
            fold(squares, sum, j);
        }
    }
    if (V > 0) { // behind all loads: h may take x's place
#pragma unroll
        for (int j = 0; j < V; ++j) {
            take(squares, held[j], gain[j]);
        }
    }
    // The row once more, for rows that are not held: h where it was written (it may have taken x's place), x and the residual otherwise.
    auto again = [&](int j, int e) {
        if (V > 0)
            return held[V > 0 ? j : 0];
        return NORM && a.h != nullptr ? load8(h, e, a.K) : fetch(e);
    };
    reduce<WAVES>(squares, most, sum, top, 0);

    float inverse_rms = 1.f;
    if constexpr (NORM) {
        float mean = squares / (float)a.K, unit = 1.f;
        if (BF16 && !(squares < INFINITY)) { // squares of bf16 numbers from 2^64 on: once more with h / 2^96
            float    small = 0.f;
            unsigned none  = 0;
            for (int j = 0; j < n; ++j) {
                const int e   = (j * kThreads + lane) * 8;
                float     sum = V > 0 ? small : 0.f;
                if (e < a.K) {
                    const shortx8 v = again(j, e);
                    for (int i = 0; i < 8; ++i) {
                        const float f = up<BF16>(v[i]) * 0x1p-96f;
                        sum           = __builtin_fmaf(f, f, sum);
                    }
                }
                if (V > 0)
                    small = sum;
                else
                    fold(small, sum, j);
            }
            reduce<WAVES>(small, none, sum, top, 1);
            mean = small / (float)a.K, unit = 0x1p-96f;
        }
        inverse_rms = 1.f / sqrtf(mean + (unit == 1.f ? a.eps : 0.f)) * unit;
    }
    const Row8 r8(most);
    if (QUANT && lane == 0)
        a.scales[row] = r8.scale * inverse_rms;
    int8_t* codes = a.codes + row * a.c_stride;
    uintx2  end   = 0; // codes of the vector that the row ends in
#pragma unroll kHeld
    for (int j = 0; j < n; ++j) {
        const int e = (j * kThreads + lane) * 8;
        if (e >= a.K)
            continue;
        const shortx8 v = again(j, e);
        shortx8       w = gain[V > 0 ? j : 0];
        if (V == 0 && NORM)
            w = load8(a.weight, e, a.K);
        if constexpr (QUANT) {
            float t[8];
            for (int i = 0; i < 8; ++i)
                t[i] = r8.none ? 0.f : (NORM ? up<BF16>(v[i]) * up<BF16>(w[i]) : up<BF16>(v[i]));
            const uintx2 c = codes8(t, r8.m, r8.inverse);
            if (e + 8 <= a.K)
                *reinterpret_cast<uintx2*>(codes + e) = c;
            else
                end = c;
        } else {
            shortx8 y;
            for (int i = 0; i < 8; ++i)
                y[i] = down<BF16>(up<BF16>(v[i]) * inverse_rms * up<BF16>(w[i]));
            store8(a.y + row * a.y_stride + e, y, a.K - e);
        }
    }
    // What a caller keeps behind a row's codes stays.
    if (QUANT && a.K % 8 != 0 && lane == a.K / 8 % kThreads)
        for (int i = 0; i < 7; ++i)
            if (i < a.K % 8)
                codes[a.K / 8 * 8 + i] = (int8_t)(end[i / 4] >> (8 * (i % 4)));
}

template <bool BF16, bool NORM, bool QUANT, int WAVES, int V>
int start(hipStream_t stream, const NormArgs& a)
{
    constexpr int kMost = 1 << 21; // rows of a launch: its threads are counted in 32 bits
    NormArgs      b     = a;
    for (int64_t first = 0; first < a.N; first += kMost) {
        b.N = (int)std::min<int64_t>(kMost, a.N - first);
        const int e = launch(rms_norm<BF16, NORM, QUANT, WAVES, V>, dim3((unsigned)(WAVES == 1 ? (b.N + 3) / 4 : b.N), 1, 1),
                             dim3(WAVES == 1 ? 256 : WAVES * kWave, 1, 1), stream, b);
        if (e != 0)
            return e;
        b.x += kMost * b.x_stride;
        b.residual = b.residual != nullptr ? b.residual + kMost * b.r_stride : nullptr;
        b.h        = b.h != nullptr ? b.h + kMost * b.h_stride : nullptr;
        b.y        = b.y != nullptr ? b.y + kMost * b.y_stride : nullptr;
        b.codes    = b.codes != nullptr ? b.codes + kMost * b.c_stride : nullptr;
        b.scales   = b.scales != nullptr ? b.scales + kMost : nullptr;
    }
    return 0;
}

// Waves to a row and vectors to a lane.  Many rows: few waves, as many vectors as leave few lanes without one, since rows in flight
// hide each other's latency (us, and with sixteen waves: 1777 rows of 5121 8.9, 13.1; 4096 of 5120 to 8 bits 29.8, 32.6; 4099 of 9216
// 52, 55).  Few rows: all the waves there are (64 rows of 7168 4.3, four waves with four vectors 6.2).  Longer rows than registers
// hold are read twice.
template <bool BF16, bool NORM, bool QUANT>
int start(hipStream_t stream, const NormArgs& a)
{
    const int vectors = (a.K + 7) / 8;
    if (vectors > 4096) {
        if constexpr (!NORM) // no weights to hold
            if (vectors <= 8192)
                return start<BF16, NORM, QUANT, 16, 8>(stream, a);
        return start<BF16, NORM, QUANT, 16, 0>(stream, a);
    }
    if (a.N < 256 && vectors > 256) {
        if (vectors <= 1024)
            return start<BF16, NORM, QUANT, 16, 1>(stream, a);
        if (vectors <= 2048)
            return start<BF16, NORM, QUANT, 16, 2>(stream, a);
        return start<BF16, NORM, QUANT, 16, 4>(stream, a);
    }
    if (vectors <= 64)
        return start<BF16, NORM, QUANT, 1, 1>(stream, a);
    if (vectors <= 128)
        return start<BF16, NORM, QUANT, 1, 2>(stream, a);
    switch ((vectors + 255) / 256) { // to a lane of four waves
    case 1: return start<BF16, NORM, QUANT, 4, 1>(stream, a);
    case 2: return start<BF16, NORM, QUANT, 4, 2>(stream, a);
    case 3: return start<BF16, NORM, QUANT, 4, 3>(stream, a);
    case 4: return start<BF16, NORM, QUANT, 4, 4>(stream, a);
    case 5: return start<BF16, NORM, QUANT, 4, 5>(stream, a);
    case 6: return start<BF16, NORM, QUANT, 4, 6>(stream, a);
    }
    switch ((vectors + 511) / 512) { // to a lane of eight
    case 4: return start<BF16, NORM, QUANT, 8, 4>(stream, a);
    case 5: return start<BF16, NORM, QUANT, 8, 5>(stream, a);
    case 6: return start<BF16, NORM, QUANT, 8, 6>(stream, a);
    default: return start<BF16, NORM, QUANT, 8, 8>(stream, a);
    }
}

int start(hipStream_t stream, const NormArgs& a, int dtype)
{
    if (a.weight == nullptr)
        return dtype == DECODE_BF16 ? start<true, false, true>(stream, a) : start<false, false, true>(stream, a);
    if (a.codes != nullptr)
        return dtype == DECODE_BF16 ? start<true, true, true>(stream, a) : start<false, true, true>(stream, a);
    return dtype == DECODE_BF16 ? start<true, true, false>(stream, a) : start<false, true, false>(stream, a);
}

int check_sizes(int N, int K, int most, int dtype)
{
    if (N < 0 || K < 1 || K > most)
        return refuse("%d rows of %d numbers (1 to %d)", N, K, most);
    if (dtype != DECODE_FP16 && dtype != DECODE_BF16)
        return refuse("unknown element type %d", dtype);
    return 0;
}

} // namespace

int run_quantize(hipStream_t stream, const void* x, int64_t x_stride, int N, int K, int8_t* codes, int64_t codes_stride,
                 float* scales, int dtype)
{
    NormArgs a{};
    a.x = static_cast<const uint16_t*>(x), a.x_stride = x_stride;
    a.codes = codes, a.c_stride = codes_stride, a.scales = scales;
    a.N = N, a.K = K;
    return start(stream, a, dtype);
}

} // namespace decode

using namespace decode;

extern "C" int RMS_Norm(hipStream_t stream, const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                        const void* weight, float eps, int N, int K, void* h_out, int64_t h_stride, void* y, int64_t y_stride,
                        int8_t* codes, int64_t codes_stride, float* scales, int dtype)
{
    if (int e = check_sizes(N, K, codes != nullptr || scales != nullptr ? kMaxK8 : 1 << 24, dtype))
        return e;
    if (!(eps >= 1e-20f) || !(eps < INFINITY))
        return refuse("eps %g: 1e-20 or more", (double)eps);
    if (N == 0)
        return 0;
    if ((codes != nullptr) == (y != nullptr))
        return refuse("a norm writes either 16-bit rows or codes");
    if (bad_pointer(x, 2) || bad_pointer(weight, 2) || (residual != nullptr && bad_pointer(residual, 2)) ||
        (h_out != nullptr && bad_pointer(h_out, 2)) || (y != nullptr && bad_pointer(y, 2)))
        return refuse("a null or misaligned x, residual, weight, h or y (2 bytes)");
    if (codes != nullptr && bad_codes(codes, codes_stride, scales, N, K))
        return refuse("codes null or misaligned (16 bytes, rows too), or scales (4)");
    if (N > 1 && ((h_out != nullptr && h_stride < K) || (y != nullptr && y_stride < K)))
        return refuse("rows of an output less than %d numbers apart", K);
    NormArgs a{};
    a.x = static_cast<const uint16_t*>(x), a.x_stride = x_stride;
    a.residual = static_cast<const uint16_t*>(residual), a.r_stride = residual_stride;
    a.weight = static_cast<const uint16_t*>(weight);
    a.h = static_cast<uint16_t*>(h_out), a.h_stride = h_stride;
    a.y = static_cast<uint16_t*>(y), a.y_stride = y_stride;
    a.codes = codes, a.c_stride = codes_stride, a.scales = scales;
    a.N = N, a.K = K, a.eps = eps;
    return start(stream, a, dtype);
}

extern "C" int W8_Quantize(hipStream_t stream, const void* x, int64_t x_stride, int N, int K, int8_t* codes, int64_t codes_stride,
                           float* scales, int dtype)
{
    if (int e = check_sizes(N, K, kMaxK8, dtype))
        return e;
    if (N == 0)
        return 0;
    if (bad_pointer(x, 2) || bad_codes(codes, codes_stride, scales, N, K))
        return refuse("x null or misaligned (2 bytes), codes (16, rows too) or scales (4)");
    return run_quantize(stream, x, x_stride, N, K, codes, codes_stride, scales, dtype);
}
