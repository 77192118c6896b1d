// Linear with 4-bit weights: W4_Pack, W4_Linear (decode_api.h).
//
// Mathematics.  Within a group of K a row's scale s and zero point z are constant, so
//   sum_k x_k s (w_k - z) = s * (sum_k x_k (16 + w_k) - (16 + z) * sum_k x_k):
// the matrix cores multiply activations by the codes themselves, put into the mantissa of 16 (16 + w is exact in fp16 and
// in bf16; an OR with a mask and, for three codes of four, a rotation), the sums of x come from a product with ones, and
// scale and zero point are applied to a group's sums in float32.
#include "decode_common.hiph"

namespace decode {

constexpr int kBlockK = 128; // columns of W in a block: 16 rows x 128 columns, 16 bytes a lane

// Packed weights: codes [row tile of 16][block of 128 columns][lane][4 dwords], scales [row tile][group][16 rows] in 16
// bits, zero points [row tile][block][h][group of the block][rows 4 h .. 4 h + 3] in 4.  Lane r + 16 h of a block holds, of row r, for each half p of 64 columns
// the dwords A = 2p, B = 2p + 1:
//   columns 64 p + 8 h + 0..7        nibbles 0 4 2 6 of A, then of B
//   columns 64 p + 32 + 8 h + 0..7   nibbles 1 5 3 7 of A, then of B
// and the dwords are rotated left to where the kernel masks the first nibbles out: by 6 bits for fp16, 3 for bf16.
struct Layout {
    int     tiles, blocks, groups;
    int64_t scales, zeros, bytes; // offsets, size
};

__host__ __device__ inline Layout layout_of(int M, int K, int group)
{
    Layout l;
    l.tiles  = (M + 15) / 16;
    l.blocks = (K + kBlockK - 1) / kBlockK;
    l.groups = K / group;
    l.scales = (int64_t)l.tiles * l.blocks * 1024;
    l.zeros  = l.scales + (int64_t)l.tiles * l.groups * 32;
    l.bytes  = (l.zeros + (int64_t)l.tiles * l.blocks * (kBlockK / group) * 8 + 15) / 16 * 16;
    return l;
}

__global__ __launch_bounds__(64) void w4_pack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int M,
                                              int K, int group, int bf16, uint8_t* packed)
{
    const int    lane = threadIdx.x, r = lane & 15, h = lane >> 4;
    const Layout l = layout_of(M, K, group);
    const int    tile = blockIdx.y, kb = blockIdx.x, row = tile * 16 + r, turn = bf16 ? 3 : 6;
    constexpr int kNibble[8] = {0, 4, 2, 6, 0, 4, 2, 6};
    uintx4        out{0, 0, 0, 0};
    for (int p = 0; p < 2; ++p)
        for (int x = 0; x < 8; ++x)
            for (int q = 0; q < 2; ++q) {
                const int k = kb * kBlockK + 64 * p + 32 * q + 8 * h + x;
                if (row < M && k < K)
                    out[2 * p + (x >> 2)] |= (codes[(int64_t)row * K + k] & 15u) << (4 * (kNibble[x] + q));
            }
    for (int i = 0; i < 4; ++i)
        out[i] = out[i] << turn | out[i] >> (32 - turn);
    reinterpret_cast<uintx4*>(packed)[((int64_t)tile * l.blocks + kb) * 64 + lane] = out;
    const int per = kBlockK / group;
    for (int g = h; g < per; g += 4) {
        const int     gk   = kb * per + g;
        const bool    live = row < M && gk < l.groups;
        const int64_t src  = (int64_t)row * l.groups + gk;
        if (gk < l.groups)
            reinterpret_cast<uint16_t*>(packed + l.scales)[((int64_t)tile * l.groups + gk) * 16 + r] = live ? scales[src] : (uint16_t)0;
        if ((r & 1) == 0) { // rows r and r + 1 of rows 4 (r / 4) ..
            const unsigned z0 = live ? zeros[src] & 15u : 0u, z1 = live && row + 1 < M ? zeros[src + l.groups] & 15u : 0u;
            packed[l.zeros + ((((int64_t)tile * l.blocks + kb) * 4 + (r >> 2)) * per + g) * 2 + (r >> 1 & 1)] = (uint8_t)(z0 | z1 << 4);
        }
    }
}

struct LinearArgs {
    const uint8_t*  packed;
    const uint16_t* x;
    int64_t         x_stride;
    uint16_t*       y;
    const uint16_t* bias;
    int             M, N, K, act;
};

template <bool BF16>
struct Types;
template <>
struct Types<false> {
    using vec = half8;
    static constexpr unsigned kMask = 0x03c003c0u, k16 = 0x4c004c00u, kOne = 0x3c003c00u;
    static __device__ __forceinline__ floatx4 mfma(vec a, vec b, floatx4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Types<true> {
    using vec = bf8;
    static constexpr unsigned kMask = 0x00780078u, k16 = 0x41804180u, kOne = 0x3f803f80u;
    static __device__ __forceinline__ floatx4 mfma(vec a, vec b, floatx4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

__device__ __forceinline__ float activate(float y, int act)
{
    if (act == 1)
        return y < 0.f ? 0.f : y; // a NaN stays one
    if (act == 2) { // y * sigmoid(2u) = y/2 (1 + tanh u); large |u| ends at 0 and y
        const float u = 0.7978845608028654f * (y + 0.044715f * y * y * y);
        return y / (1.f + __expf(-2.f * u));
    }
    return y;
}

// One workgroup: R row tiles of 16 rows and NT column tiles of 16 columns, the blocks of K dealt to its WAVES waves in turn;
// the waves' sums are joined through LDS.  G: group size.
template <int NT, int R, int G, bool BF16, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void w4_linear(LinearArgs a)
{
    using T   = Types<BF16>;
    using vec = typename T::vec;
    constexpr int kGroups = kBlockK / G; // groups of a block
    __shared__ float join[WAVES][R * 16 * NT * 16];
    const int    lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, h = lane >> 4;
    const Layout l = layout_of(a.M, a.K, G);
    const int    tile0 = blockIdx.x * R, n0 = blockIdx.y * 16 * NT;

    const uintx4*   codes[R];
    const uint16_t* scales[R];
    const uint8_t*  zeros[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t tile = min(tile0 + r, l.tiles - 1); // a tile past the end is computed again and not stored
        codes[r]  = reinterpret_cast<const uintx4*>(a.packed) + tile * l.blocks * 64 + lane;
        scales[r] = reinterpret_cast<const uint16_t*>(a.packed + l.scales) + tile * l.groups * 16 + 4 * h;
        zeros[r]  = a.packed + l.zeros + (tile * l.blocks * 4 + h) * kGroups * 2;
    }
    const uint16_t* x[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
        x[n] = a.x + (int64_t)min(n0 + 16 * n + c, a.N - 1) * a.x_stride + 8 * h;

    const floatx4 zero{0.f, 0.f, 0.f, 0.f};
    floatx4       y[R][NT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
            y[r][n] = zero;
    const vec ones = __builtin_bit_cast(vec, uintx4{T::kOne, T::kOne, T::kOne, T::kOne});

    // two sets of registers: the loads of a wave's next block are in flight while it works on one
    struct Block {
        uintx4   w[R];
        uintx2   s[R][kGroups];
        unsigned z[R][(kGroups + 1) / 2];
        vec      x[4][NT];
    } set[2];
    auto fetch = [&](Block& b, int kb) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            b.w[r] = __builtin_nontemporal_load(codes[r] + (int64_t)kb * 64);
#pragma unroll
            for (int g = 0; g < kGroups; ++g)
                b.s[r][g] = *reinterpret_cast<const uintx2*>(scales[r] + min(kb * kGroups + g, l.groups - 1) * 16);
            const uint8_t* z = zeros[r] + (int64_t)kb * 8 * kGroups;
            if constexpr (kGroups == 1)
                b.z[r][0] = *reinterpret_cast<const uint16_t*>(z);
            else
#pragma unroll
                for (int g = 0; g < kGroups / 2; ++g)
                    b.z[r][g] = reinterpret_cast<const unsigned*>(z)[g];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) { // columns past the end as zeros (K is a multiple of 32)
            const int  k      = kb * kBlockK + 32 * j;
            const bool inside = k < a.K;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uintx4 raw = *reinterpret_cast<const uintx4*>(x[n] + (inside ? k : 0));
                if (!inside)
                    raw = uintx4{0, 0, 0, 0};
                b.x[j][n] = __builtin_bit_cast(vec, raw);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto work = [&](const Block& b) {
        floatx4 acc[R][NT], xs[NT];
#pragma unroll
        for (int j = 0; j < 4; ++j) { // 32 columns: nibbles 0 4 2 6 of two dwords, or 1 5 3 7
            constexpr int kSteps = G / 32;
            if (j % kSteps == 0) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    xs[n] = zero;
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        acc[r][n] = zero;
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
                xs[n] = T::mfma(ones, b.x[j][n], xs[n]);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const unsigned A = b.w[r][j & 2], B = b.w[r][(j & 2) + 1];
                const int      n0 = 4 * (j & 1);
                auto part = [](unsigned v, int n) { return (__builtin_amdgcn_alignbit(v, v, n) & T::kMask) | T::k16; };
                const vec wv = __builtin_bit_cast(vec, uintx4{part(A, n0), part(A, n0 + 8), part(B, n0), part(B, n0 + 8)});
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    acc[r][n] = T::mfma(wv, b.x[j][n], acc[r][n]);
            }
            if (j % kSteps == kSteps - 1) {
                const int g = j / kSteps;
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float sc = from16((uint16_t)(b.s[r][g][i >> 1] >> (16 * (i & 1))), BF16);
                        const float zp = (float)((b.z[r][g >> 1] >> (16 * (g & 1) + 4 * i)) & 15u) + 16.f;
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            y[r][n][i] = __builtin_fmaf(__builtin_fmaf(-zp, xs[n][i], acc[r][n][i]), sc, y[r][n][i]);
                    }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    if (wave < l.blocks) {
        int kb = wave;
        fetch(set[0], kb);
        while (true) {
            fetch(set[1], min(kb + WAVES, l.blocks - 1)); // the last one is fetched again and not used
            work(set[0]);
            if ((kb += WAVES) >= l.blocks)
                break;
            fetch(set[0], min(kb + WAVES, l.blocks - 1));
            work(set[1]);
            if ((kb += WAVES) >= l.blocks)
                break;
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
    return (size_t)layout_of(M, K, group).bytes;
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
                       static_cast<uint16_t*>(Y),           static_cast<const uint16_t*>(bias), M, N, K, activation};
    const bool       bf16 = dtype == DECODE_BF16;
    if (N <= 16)
        return run_linear<1, 1, 8>(stream, a, group, bf16);
    if (N <= 32)
        return run_linear<2, 1, 8>(stream, a, group, bf16);
    return run_linear<4, 1, 8>(stream, a, group, bf16);
}
