// Linear with 4-bit weights: W4_Pack, W4_Linear (decode_api.h).
//
// Mathematics.  Within a group of K a row's scale s and zero point z are constant, so
//   sum_k x_k s (w_k - z) = s * (sum_k x_k w_k - z * sum_k x_k):
// the matrix cores multiply activations by the codes themselves, the sums of x come from a product with ones, and scale and
// zero point are applied to a group's sums in float32.
// For fp16 a code masked out of its dword in place is the subnormal w * 2^-22 (bits 2..5 of a half) or w * 2^-18 (bits
// 6..9): one AND per two codes, one rotation per eight.  v_mfma_f32_16x16x32_f16 multiplies subnormals as they are, but
// aligns its sums by exponent fields, so that a code's distance from the top of the mantissa costs precision: hence bits
// 2..9 and not 0..7, and ones for the sums of x that are normal numbers.  The two kinds go into products of their own,
// since x itself may not be scaled by 1/16 without loss.  bf16 has no mantissa to spare for that: there a code is put
// into the mantissa of 16 (16 + w is exact) and 16 sum x is taken off with the zero point.
#include "decode_common.hiph"

namespace decode {

constexpr int kBlockK = 128; // columns of W in a block: 16 rows x 128 columns, 16 bytes a lane

// Packed weights: codes [row tile of 16][block of 128 columns][lane][4 dwords], then words [row tile][group][16 rows], the
// bits of a float32 scale (the 16-bit types' values fit its upper 20 bits) with the zero point in its four lowest.
// Lane r + 16 h of a block holds, of row r, for each half p of 64 columns the dwords A = 2p, B = 2p + 1:
//   columns 64 p + 8 h + 0..7        nibbles 0 4 2 6 of A, then of B
//   columns 64 p + 32 + 8 h + 0..7   nibbles 1 5 3 7 of A, then of B
// and the dwords are rotated left by 2 bits (fp16) or 3 (bf16), to where the kernel masks them out.
__host__ __device__ inline int64_t code_bytes(int M, int K)
{
    return (int64_t)((M + 15) / 16) * ((K + kBlockK - 1) / kBlockK) * 1024;
}

__global__ __launch_bounds__(64) void w4_pack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int M,
                                              int K, int group, int bf16, uint8_t* packed)
{
    const int lane = threadIdx.x, r = lane & 15, h = lane >> 4, blocks = (K + kBlockK - 1) / kBlockK, groups = K / group;
    const int tile = blockIdx.y, kb = blockIdx.x, row = tile * 16 + r;
    constexpr int kNibble[8] = {0, 4, 2, 6, 0, 4, 2, 6};
    uintx4        out{0, 0, 0, 0};
    for (int p = 0; p < 2; ++p)
        for (int x = 0; x < 8; ++x)
            for (int q = 0; q < 2; ++q) {
                const int k = kb * kBlockK + 64 * p + 32 * q + 8 * h + x;
                if (row < M && k < K)
                    out[2 * p + (x >> 2)] |= (codes[(int64_t)row * K + k] & 15u) << (4 * (kNibble[x] + q));
            }
    const int turn = bf16 ? 3 : 2;
    for (int i = 0; i < 4; ++i)
        out[i] = out[i] << turn | out[i] >> (32 - turn);
    reinterpret_cast<uintx4*>(packed)[((int64_t)tile * blocks + kb) * 64 + lane] = out;
    unsigned* words = reinterpret_cast<unsigned*>(packed + code_bytes(M, K));
    for (int g = kb * kBlockK / group + h; g < groups && g < (kb + 1) * kBlockK / group; g += 4) {
        unsigned w = 0;
        if (row < M)
            w = (__float_as_uint(from16(scales[(int64_t)row * groups + g], bf16)) & ~15u) | (zeros[(int64_t)row * groups + g] & 15u);
        words[((int64_t)tile * groups + g) * 16 + r] = w;
    }
}

struct LinearArgs {
    const uint8_t*  packed;
    const uint16_t* x;
    int64_t         x_stride;
    uint16_t*       y;
    const uint16_t* bias;
    int             M, N, K, groups, act;
};

template <bool BF16>
struct Types;
template <>
struct Types<false> {
    using vec = half8;
    static __device__ __forceinline__ floatx4 mfma(vec a, vec b, floatx4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Types<true> {
    using vec = bf8;
    static __device__ __forceinline__ floatx4 mfma(vec a, vec b, floatx4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

__device__ __forceinline__ float activate(float y, int act)
{
    if (act == 1)
        return fmaxf(y, 0.f) + (y != y ? y : 0.f); // a NaN stays one
    if (act == 2) { // y * sigmoid(2u) = y/2 (1 + tanh u); large |u| ends at 0 and y
        const float u = 0.7978845608028654f * (y + 0.044715f * y * y * y);
        return y / (1.f + __expf(-2.f * u));
    }
    return y;
}

// One workgroup: R row tiles of 16 rows and NT column tiles of 16 columns, the blocks of K dealt to its waves in turn; the
// waves' sums are joined through LDS.  G: group size.
template <int NT, int R, int G, bool BF16, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void w4_linear(LinearArgs a)
{
    using T   = Types<BF16>;
    using vec = typename T::vec;
    constexpr int      kGroups = kBlockK / G; // groups of a block
    constexpr unsigned kLow = 0x003c003cu, kHigh = 0x03c003c0u, kBf16 = 0x00780078u, k16 = 0x41804180u;
    __shared__ float join[WAVES][R * 16 * NT * 16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, h = lane >> 4;
    const int tiles = (a.M + 15) / 16, blocks = (a.K + kBlockK - 1) / kBlockK;
    const int tile0 = blockIdx.x * R, n0 = blockIdx.y * 16 * NT;

    const uintx4* codes[R];
    const unsigned* words[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int tile = min(tile0 + r, tiles - 1); // a tile past the end is computed again and not stored
        codes[r]       = reinterpret_cast<const uintx4*>(a.packed) + (int64_t)tile * blocks * 64 + lane;
        words[r]       = reinterpret_cast<const unsigned*>(a.packed + code_bytes(a.M, a.K)) + (int64_t)tile * a.groups * 16 + 4 * h;
    }
    const uint16_t* x[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
        x[n] = a.x + (int64_t)min(n0 + 16 * n + c, a.N - 1) * a.x_stride + 8 * h;

    floatx4 y[R][NT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
            y[r][n] = floatx4{0.f, 0.f, 0.f, 0.f};
    const unsigned one = BF16 ? 0x3f803f80u : 0x04000400u; // 1, or the smallest normal number 2^-14
    const vec      ones = __builtin_bit_cast(vec, uintx4{one, one, one, one});

    uintx4 wn[R], sn[R][kGroups];
    auto   fetch = [&](int kb) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            wn[r] = __builtin_nontemporal_load(codes[r] + (int64_t)kb * 64);
#pragma unroll
            for (int g = 0; g < kGroups; ++g)
                sn[r][g] = *reinterpret_cast<const uintx4*>(words[r] + min(kb * kGroups + g, a.groups - 1) * 16);
        }
    };
    int kb = wave;
    if (kb < blocks)
        fetch(kb);
    for (; kb < blocks; kb += WAVES) {
        uintx4 w[R], sw[R][kGroups];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            w[r] = wn[r];
#pragma unroll
            for (int g = 0; g < kGroups; ++g)
                sw[r][g] = sn[r][g];
        }
        vec xv[4][NT]; // columns 32 j + 8 h + 0..7 of the block
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int  k      = kb * kBlockK + 32 * j;
            const bool inside = k < a.K; // K is a multiple of 32
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uintx4 raw = *reinterpret_cast<const uintx4*>(x[n] + (inside ? k : 0));
                if (!inside)
                    raw = uintx4{0, 0, 0, 0};
                xv[j][n] = __builtin_bit_cast(vec, raw);
            }
        }
        fetch(min(kb + WAVES, blocks - 1));
        floatx4 lo[R][NT], up[R][NT], xs[NT];
        const floatx4 zero{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) { // 32 columns: lower nibbles for even j, upper ones for odd
            constexpr int kSteps = G / 32;
            const bool    first  = j % kSteps == 0;
            if (first) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    xs[n] = zero;
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        lo[r][n] = up[r][n] = zero;
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
                xs[n] = T::mfma(ones, xv[j][n], xs[n]);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const unsigned A = w[r][j & 2], B = w[r][(j & 2) + 1];
                uintx4         raw;
                if constexpr (BF16) {
                    auto part = [](unsigned v, int n) { return (__builtin_amdgcn_alignbit(v, v, n) & kBf16) | k16; };
                    const int n = (j & 1) * 4;
                    raw = uintx4{part(A, n), part(A, n + 8), part(B, n), part(B, n + 8)};
                } else {
                    const unsigned m = (j & 1) ? kHigh : kLow;
                    raw = uintx4{A & m, __builtin_amdgcn_alignbit(A, A, 8) & m, B & m, __builtin_amdgcn_alignbit(B, B, 8) & m};
                }
                const vec wv = __builtin_bit_cast(vec, raw);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    floatx4& acc = !BF16 && (j & 1) ? up[r][n] : lo[r][n];
                    acc          = T::mfma(wv, xv[j][n], acc);
                }
            }
            if (j % kSteps == kSteps - 1) {
                const int g = j / kSteps;
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const unsigned word = sw[r][g][i];
                        // the zero point's bits change the scale by less than 2^-19 of it, a 256th of the output's rounding
                        const float s = __uint_as_float(word) * (BF16 ? 1.f : 0x1p22f);
                        const float z = BF16 ? (float)(word & 15u) + 16.f : (float)(word & 15u) * 0x1p-8f;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            float t = lo[r][n][i];
                            if constexpr (!BF16) {
                                if (G == 32)
                                    t = (j & 1) ? up[r][n][i] * 0.0625f : t;
                                else
                                    t = __builtin_fmaf(up[r][n][i], 0.0625f, t);
                            }
                            y[r][n][i] = __builtin_fmaf(__builtin_fmaf(-z, xs[n][i], t), s, y[r][n][i]);
                        }
                    }
            }
        }
    }

#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
            *reinterpret_cast<floatx4*>(&join[wave][((n * 16 + c) * R + r) * 16 + 4 * h]) = y[r][n];
    __syncthreads();
    for (int at = threadIdx.x; at < R * 16 * NT * 16; at += 64 * WAVES) {
        const int m = tile0 * 16 + at % (R * 16), n = n0 + at / (R * 16);
        if (m >= a.M || n >= a.N)
            continue;
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < WAVES; ++v)
            sum += join[v][at];
        if (a.bias != nullptr)
            sum += from16(a.bias[m], BF16);
        a.y[(int64_t)n * a.M + m] = to16(activate(sum, a.act), BF16);
    }
}

namespace {

template <int NT, int R, int WAVES>
int run_linear(hipStream_t stream, const LinearArgs& a, int group, bool bf16)
{
    const int  tiles = (a.M + 15) / 16;
    const dim3 grid((unsigned)((tiles + R - 1) / R), (unsigned)((a.N + 16 * NT - 1) / (16 * NT)), 1), block(64 * WAVES, 1, 1);
    if (group == 32)
        return bf16 ? launch(w4_linear<NT, R, 32, true, WAVES>, grid, block, stream, a)
                    : launch(w4_linear<NT, R, 32, false, WAVES>, grid, block, stream, a);
    if (group == 64)
        return bf16 ? launch(w4_linear<NT, R, 64, true, WAVES>, grid, block, stream, a)
                    : launch(w4_linear<NT, R, 64, false, WAVES>, grid, block, stream, a);
    return bf16 ? launch(w4_linear<NT, R, 128, true, WAVES>, grid, block, stream, a)
                : launch(w4_linear<NT, R, 128, false, WAVES>, grid, block, stream, a);
}

int check_weights(int M, int K, int group, int dtype)
{
    if (group != 32 && group != 64 && group != 128)
        return refuse("a group of %d columns: 32, 64 or 128", group);
    if (M < 1 || M > 16 * 65535 || K < group || K % group != 0)
        return refuse("weights of %d rows (at most 16 * 65535) and %d columns (a multiple of %d)", M, K, group);
    if (dtype != DECODE_FP16 && dtype != DECODE_BF16)
        return refuse("unknown element type %d", dtype);
    return 0;
}

} // namespace
} // namespace decode

using namespace decode;

extern "C" size_t W4_PackedBytes(int M, int K, int group)
{
    if ((group != 32 && group != 64 && group != 128) || M < 1 || M > 16 * 65535 || K < group || K % group != 0)
        return 0;
    return (size_t)code_bytes(M, K) + (size_t)((M + 15) / 16) * (K / group) * 64;
}

extern "C" int W4_Pack(hipStream_t stream, const uint8_t* codes, const void* scales, const uint8_t* zeros, int M, int K,
                       int group, int dtype, void* packed)
{
    if (int e = check_weights(M, K, group, dtype))
        return e;
    if (codes == nullptr || zeros == nullptr || bad_pointer(scales, 2) || bad_pointer(packed, 16))
        return refuse("a null or misaligned codes, scales, zeros (1, 2, 1 bytes) or packed (16)");
    const dim3 grid((unsigned)((K + kBlockK - 1) / kBlockK), (unsigned)((M + 15) / 16), 1);
    return launch(w4_pack, grid, dim3(64, 1, 1), stream, codes, static_cast<const uint16_t*>(scales), zeros, M, K, group,
                  dtype == DECODE_BF16, static_cast<uint8_t*>(packed));
}

extern "C" int W4_Linear(hipStream_t stream, const void* packed, const void* X, int64_t x_stride, void* Y, int M, int N,
                         int K, int group, const void* bias, int activation, int dtype)
{
    if (int e = check_weights(M, K, group, dtype))
        return e;
    if (N < 0 || N > 65535 * 64)
        return refuse("%d columns (0 to 64 * 65535)", N);
    if (activation < 0 || activation > 2)
        return refuse("unknown activation %d (0 none, 1 ReLU, 2 GELU)", activation);
    if (N == 0)
        return 0;
    if (bad_pointer(packed, 16) || bad_pointer(X, 16) || bad_pointer(Y, 2) || (bias != nullptr && bad_pointer(bias, 2)) ||
        (N > 1 && x_stride < K) || x_stride % 8 != 0)
        return refuse("a null or misaligned weight, X (16 bytes, rows too), Y or bias (2)");
    const LinearArgs a{static_cast<const uint8_t*>(packed), static_cast<const uint16_t*>(X), x_stride,
                       static_cast<uint16_t*>(Y),           static_cast<const uint16_t*>(bias), M, N, K, K / group, activation};
    const bool       bf16 = dtype == DECODE_BF16;
    if (N <= 16)
        return run_linear<1, 1, 8>(stream, a, group, bf16);
    if (N <= 32)
        return run_linear<2, 1, 8>(stream, a, group, bf16);
    return run_linear<4, 1, 8>(stream, a, group, bf16);
}
