// Linear with 4-bit weights: W4_Pack, W4_Linear (decode_api.h).
//
// Mathematics.  Within a group of K a row's scale s and zero point z are constant, so
//   sum_k x_k s (w_k - z) = s * (sum_k x_k (16 + w_k) - (16 + z) * sum_k x_k):
// the matrix cores multiply activations by the codes themselves, put into the mantissa of 16 (16 + w is exact in fp16 and
// in bf16; an OR with a mask and, for three codes of four, a rotation), the sums of x come from a product with ones, and
// scale and zero point are applied to a group's sums in float32.
#include "decode_common.hiph"

#include <algorithm>

namespace decode {

constexpr int kBlockK     = 128;        // columns of W in a block: 16 rows x 128 columns, 16 bytes a lane
constexpr int kWaves      = 8;          // waves of a workgroup of w4_linear
constexpr int kMaxColumns = 16 * 65535; // column tiles are the y dimension of the grid
constexpr int kMaxK       = 1 << 30;    // column numbers of the last block, and of those fetched behind it, are ints

// Packed weights: codes [row tile of 16][block of 128 columns][lane][4 dwords], scales [row tile][group][16 rows] in 16
// bits, zero points plus 16 [row tile][block][h][group of the block][rows 4 h .. 4 h + 3] in 8.  Lane r + 16 h of a block holds, of row r, for each half p of 64 columns
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
    l.bytes  = (l.zeros + (int64_t)l.tiles * l.blocks * (kBlockK / group) * 16 + 15) / 16 * 16;
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
        packed[l.zeros + ((((int64_t)tile * l.blocks + kb) * 4 + (r >> 2)) * per + g) * 4 + (r & 3)] =
            (uint8_t)(16 + (live ? zeros[src] & 15 : 0));
    }
}

struct LinearArgs {
    const uint8_t*  packed;
    const uint16_t* x;
    int64_t         x_stride;
    uint16_t*       y;
    const uint16_t* bias;
    float*          part;
    int             M, N, K, act, splits;
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

// What a lane loads of one block of R row tiles.
template <int R, int G>
struct Weights {
    static constexpr int kGroups = kBlockK / G; // groups of a block
    uintx4   w[R];
    uintx2   s[R][kGroups];
    unsigned z[R][kGroups];
};

template <int R, int G>
struct Source {
    const uintx4*   codes[R];
    const uint16_t* scales[R];
    const uint8_t*  zeros[R];
    int             groups;

    // Row tiles from tile0 on; one past the end is the last one again (it is computed and not stored).
    __device__ __forceinline__ Source(const LinearArgs& a, const Layout& l, int tile0, int lane)
    {
        constexpr int kGroups = kBlockK / G;
        const int     h       = lane >> 4;
        groups                = l.groups;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t tile = min(tile0 + r, l.tiles - 1);
            codes[r]  = reinterpret_cast<const uintx4*>(a.packed) + tile * l.blocks * 64 + lane;
            scales[r] = reinterpret_cast<const uint16_t*>(a.packed + l.scales) + tile * l.groups * 16 + 4 * h;
            zeros[r]  = a.packed + l.zeros + (tile * l.blocks * 4 + h) * kGroups * 4;
        }
    }

    template <bool ZEROS>
    __device__ __forceinline__ void fetch(Weights<R, G>& b, int kb) const
    {
        constexpr int kGroups = kBlockK / G;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            b.w[r] = __builtin_nontemporal_load(codes[r] + (int64_t)kb * 64);
#pragma unroll
            for (int g = 0; g < kGroups; ++g) // a group past the end meets zeros of X
                b.s[r][g] = *reinterpret_cast<const uintx2*>(scales[r] + min(kb * kGroups + g, groups - 1) * 16);
            const unsigned* z = reinterpret_cast<const unsigned*>(zeros[r] + (int64_t)kb * 16 * kGroups);
            if constexpr (!ZEROS) {
            } else if constexpr (kGroups == 1) {
                b.z[r][0] = z[0];
            } else if constexpr (kGroups == 2) {
                const uintx2 v = *reinterpret_cast<const uintx2*>(z);
                b.z[r][0] = v[0], b.z[r][1] = v[1];
            } else {
                const uintx4 v = *reinterpret_cast<const uintx4*>(z);
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    b.z[r][g] = v[g];
            }
        }
    }
};

// y += W X of one block; x(j, n) gives the lane's operand for columns 32 j .. 32 j + 31 of column tile n.  Without ZEROS the 16 and
// the zero points stay in the sums.
template <int NT, int R, int G, bool BF16, bool ZEROS, typename X>
__device__ __forceinline__ void multiply(floatx4 (&y)[R][NT], const Weights<R, G>& b, X x)
{
    using T   = Types<BF16>;
    using vec = typename T::vec;
    constexpr int kSteps = G / 32;
    const floatx4 zero{0.f, 0.f, 0.f, 0.f};
    const vec     ones = __builtin_bit_cast(vec, uintx4{T::kOne, T::kOne, T::kOne, T::kOne});
    floatx4       acc[R][NT], xs[NT];
    unsigned      mask = T::kMask;
    asm("" : "+v"(mask)); // in a register: an instruction takes one literal, and with two a code's AND and OR are two instructions
#pragma unroll
    for (int j = 0; j < 4; ++j) { // 32 columns: nibbles 0 4 2 6 of two dwords, or 1 5 3 7
        if (j % kSteps == 0) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                xs[n] = zero;
#pragma unroll
                for (int r = 0; r < R; ++r)
                    acc[r][n] = zero;
            }
        }
        vec xv[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            xv[n] = x(j, n);
            if constexpr (ZEROS)
                xs[n] = T::mfma(ones, xv[n], xs[n]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const unsigned A = b.w[r][j & 2], B = b.w[r][(j & 2) + 1];
            const int      n0 = 4 * (j & 1);
            auto part = [&](unsigned v, int n) { return (__builtin_amdgcn_alignbit(v, v, n) & mask) | T::k16; };
            const vec wv = __builtin_bit_cast(vec, uintx4{part(A, n0), part(A, n0 + 8), part(B, n0), part(B, n0 + 8)});
#pragma unroll
            for (int n = 0; n < NT; ++n)
                acc[r][n] = T::mfma(wv, xv[n], acc[r][n]);
        }
        if (j % kSteps == kSteps - 1) {
            const int g = j / kSteps;
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float sc = from16((uint16_t)(b.s[r][g][i >> 1] >> (16 * (i & 1))), BF16);
                    if constexpr (ZEROS) {
                        const float zp = (float)((b.z[r][g] >> (8 * i)) & 255u);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            y[r][n][i] = __builtin_fmaf(__builtin_fmaf(-zp, xs[n][i], acc[r][n][i]), sc, y[r][n][i]);
                    } else {
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            y[r][n][i] = __builtin_fmaf(acc[r][n][i], sc, y[r][n][i]);
                    }
                }
        }
    }
}

// Sums that came out infinite or NaN are computed once more, with w - z itself as the operand: an infinity of X, met by 16 + w, would
// be taken off again as NaN, and bf16 values near the type's end overflow on the way (here they go in 2^16 times smaller).  Other
// sums keep their bits.  Bit 4 (r NT + n) + i of a lane: y[r][n][i] is such a sum; a look at the sums where there are none.  28672x7168,
// N = 16, with no such value in X / a row of NaN / one infinity in a row 25 / 35 / 65 us, 9216x36864, N = 64, 80 / 83 / 259.
template <int NT, int R>
__device__ __forceinline__ unsigned infinite_sums(const floatx4 (&y)[R][NT])
{
    static_assert(4 * R * NT <= 32, "");
    float none = 0.f; // NaN with an infinity or a NaN
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                none = __builtin_fmaf(y[r][n][i], 0.f, none);
    unsigned bad = 0;
    if (__builtin_expect(__any(none != 0.f), 0)) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    bad |= fabsf(y[r][n][i]) < __builtin_inff() ? 0u : 1u << (4 * (r * NT + n) + i);
    }
    return bad;
}

// Rows 4 h .. 4 h + 3 of a tile and column n0 + c over blocks first, first + step .. below last, until those that bit i of `bad` asks
// for are NaN, as they are from the first one in X on.  By whole waves.
template <int G, bool BF16>
__device__ floatx4 sum_again(const LinearArgs& a, const Layout& l, unsigned bad, int tile, int n0, int first, int last, int step, int lane)
{
    using T   = Types<BF16>;
    using vec = typename T::vec;
    constexpr int   kGroups = kBlockK / G, kTurn = BF16 ? 3 : 6;
    constexpr float kDown = BF16 ? 0x1p-16f : 1.f;
    const int       c = lane & 15, h = lane >> 4;
    const int64_t   at = min(tile, l.tiles - 1);
    const uintx4*   codes = reinterpret_cast<const uintx4*>(a.packed) + at * l.blocks * 64 + lane;
    const uint16_t* scales = reinterpret_cast<const uint16_t*>(a.packed + l.scales) + at * l.groups * 16 + 4 * h;
    const uint8_t*  zeros = a.packed + l.zeros + (at * l.blocks * 4 + (c >> 2)) * kGroups * 4 + (c & 3); // of row c
    const uint16_t* x = a.x + (int64_t)min(n0 + c, a.N - 1) * a.x_stride + 8 * h;
    floatx4         sum{0.f, 0.f, 0.f, 0.f};
    for (int kb = first; kb < last; kb += step) {
        const uintx4 w = codes[(int64_t)kb * 64];
        for (int j = 0; j < 4; ++j) {
            const int k = kb * kBlockK + 32 * j, g = 32 * j / G;
            if (k >= a.K)
                break;
            const uintx4 raw = *reinterpret_cast<const uintx4*>(x + k);
            const float  z   = (float)zeros[(kb * 4 * kGroups + g) * 4] - 16.f;
            vec          wv, xv;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                constexpr int  kNibble[8] = {0, 4, 2, 6, 0, 4, 2, 6};
                const unsigned dword = j < 2 ? (e < 4 ? w[0] : w[1]) : (e < 4 ? w[2] : w[3]);
                const unsigned code  = __builtin_amdgcn_alignbit(dword, dword, (4 * (kNibble[e] + (j & 1)) + kTurn) & 31) & 15u;
                const float    xe    = from16((uint16_t)(raw[e >> 1] >> (16 * (e & 1))), BF16) * kDown;
                if constexpr (BF16)
                    wv[e] = (__bf16)((float)code - z), xv[e] = (__bf16)xe;
                else
                    wv[e] = (_Float16)((float)code - z), xv[e] = (_Float16)xe;
            }
            const floatx4 acc = T::mfma(wv, xv, floatx4{0.f, 0.f, 0.f, 0.f});
            const uintx2  s   = *reinterpret_cast<const uintx2*>(scales + (kb * kGroups + g) * 16);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                sum[i] = __builtin_fmaf(acc[i] * from16((uint16_t)(s[i >> 1] >> (16 * (i & 1))), BF16), 1.f / kDown, sum[i]);
        }
        unsigned numbers = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            numbers |= sum[i] == sum[i] ? 1u << i : 0u;
        if (!__any((numbers & bad) != 0))
            break;
    }
    return sum;
}

// Few columns.  One workgroup: R row tiles of 16 rows and 16 columns, a share of K's blocks dealt to its waves in turn; the waves'
// sums are joined through LDS.  G: group size.  Bound by memory where it has one workgroup for every CU: 28672x7168, N = 16,
// groups of 128, in 24.6 us is 4.3 TB/s of weights (a large copy moves 4.9); 5120x5120, N = 1 takes 7.4, a launch, two
// rounds of loads and the join, where its bytes are 2.8.  What it took: two sets of registers, so that no
// wait for X includes the weights behind it; X from the cache as rarely as the registers allow (R tiles per read of it).
template <int R, int G, bool BF16>
__global__ __launch_bounds__(64 * kWaves) void w4_linear(LinearArgs a)
{
    using vec = typename Types<BF16>::vec;
    __shared__ float join[kWaves][R * 256];
    const int    lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, h = lane >> 4;
    const Layout l = layout_of(a.M, a.K, G);
    const int    tile0 = blockIdx.x * R, n0 = blockIdx.y * 16;
    const Source<R, G> source(a, l, tile0, lane);
    const uint16_t*    x = a.x + (int64_t)min(n0 + c, a.N - 1) * a.x_stride + 8 * h;

    floatx4 y[R][1];
#pragma unroll
    for (int r = 0; r < R; ++r)
        y[r][0] = floatx4{0.f, 0.f, 0.f, 0.f};
    // two sets of registers: the loads of a wave's next block are in flight while it works on one
    struct Block {
        Weights<R, G> w;
        vec           x[4];
    } set[2];
    auto fetch = [&](Block& b, int kb) {
        source.template fetch<true>(b.w, kb);
#pragma unroll
        for (int j = 0; j < 4; ++j) { // columns past the end as zeros (K is a multiple of 32)
            const int  k      = kb * kBlockK + 32 * j;
            const bool inside = k < a.K;
            uintx4     raw    = *reinterpret_cast<const uintx4*>(x + (inside ? k : 0));
            if (!inside)
                raw = uintx4{0, 0, 0, 0};
            b.x[j] = __builtin_bit_cast(vec, raw);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto work = [&](const Block& b) {
        multiply<1, R, G, BF16, true>(y, b.w, [&](int j, int) { return b.x[j]; });
        __builtin_amdgcn_sched_barrier(0);
    };
    const int per = (l.blocks + a.splits - 1) / a.splits, last = min((int)(blockIdx.z + 1) * per, l.blocks);
    if ((int)blockIdx.z * per + wave < last) {
        int kb = (int)blockIdx.z * per + wave;
        fetch(set[0], kb);
        while (true) {
            fetch(set[1], min(kb + kWaves, last - 1)); // the last one is fetched again and not used
            work(set[0]);
            if ((kb += kWaves) >= last)
                break;
            fetch(set[0], min(kb + kWaves, last - 1));
            work(set[1]);
            if ((kb += kWaves) >= last)
                break;
        }
    }

#pragma unroll
    for (int r = 0; r < R; ++r)
        *reinterpret_cast<floatx4*>(&join[wave][(c * R + r) * 16 + 4 * h]) = y[r][0];
    if (const unsigned bad = infinite_sums<1, R>(y); __builtin_expect(__any(bad != 0), 0)) {
        for (int r = 0; r < R; ++r) {
            if (!__any((bad >> (4 * r) & 15u) != 0))
                continue;
            const floatx4 sum = sum_again<G, BF16>(a, l, bad >> (4 * r) & 15u, tile0 + r, n0, (int)blockIdx.z * per + wave, last, kWaves, lane);
            for (int i = 0; i < 4; ++i)
                if (bad >> (4 * r + i) & 1u)
                    join[wave][(c * R + r) * 16 + 4 * h + i] = sum[i];
        }
    }
    __syncthreads();
    for (int at = threadIdx.x; at < R * 256; at += 64 * kWaves) {
        const int m = tile0 * 16 + at % (R * 16), n = n0 + at / (R * 16);
        if (m >= a.M || n >= a.N)
            continue;
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < kWaves; ++v)
            sum += join[v][at];
        if (a.splits > 1) {
            a.part[((int64_t)blockIdx.z * a.N + n) * (l.tiles * 16) + m] = sum;
            continue;
        }
        if (a.bias != nullptr)
            sum += from16(a.bias[m], BF16);
        a.y[(int64_t)n * a.M + m] = to16(activate(sum, a.act), BF16);
    }
}

// Many columns.  One workgroup: WAVES waves of R row tiles each and NT column tiles, over a share of K's blocks; the X of a
// block goes through LDS, once for all waves.  Partial sums of a split K go to `part` [split][column][row].  9216x36864, N = 64,
// bf16, groups of 64, seven shares: 76.9 us with the sum of the shares (5), 2.4 TB/s of weights.  Without its products the
// kernel takes 57, without its loads of weights 69 (of 76.4), and two waves a SIMD hide the one behind the other only in part; loads two and
// three blocks ahead, operands a step ahead, vector instructions dealt between the products and XCDs with shares of their own did not help.
// w4_linear, which reads X from the cache for every wave, takes 190 to 240 there.
template <int NT, int R, int G, bool BF16, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void w4_linear_wide(LinearArgs a)
{
    using vec = typename Types<BF16>::vec;
    constexpr int kThreads = 64 * WAVES, kChunks = NT * 16 * 16 / kThreads; // 16-byte chunks of X a thread moves per block
    static_assert(kChunks * kThreads == NT * 256, "");
    __shared__ uintx4 slab[2][4 * NT * 64];
    const int    lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, h = lane >> 4;
    const Layout l = layout_of(a.M, a.K, G);
    const int    tile0 = (blockIdx.x * WAVES + wave) * R, n0 = blockIdx.y * 16 * NT;
    const int    per = (l.blocks + a.splits - 1) / a.splits, first = blockIdx.z * per, last = min(first + per, l.blocks);
    const Source<R, G> source(a, l, tile0, lane);

    floatx4 y[R][NT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
            y[r][n] = floatx4{0.f, 0.f, 0.f, 0.f};

    // chunk q of a thread: 8 columns k0 .. of row `row` of the slab; sixteen threads read a row's 256 bytes.  In LDS an operand's
    // sixteen rows are permuted by its place in the block, which spreads the sixteen chunks of a row over the banks.
    const int       ch = threadIdx.x & 15, k0 = 8 * ch;
    const uint16_t* xsrc[kChunks];
    int             xdst[kChunks];
#pragma unroll
    for (int q = 0; q < kChunks; ++q) {
        const int row = (threadIdx.x >> 4) + q * (kThreads / 16);
        xsrc[q] = a.x + (int64_t)min(n0 + row, a.N - 1) * a.x_stride + k0;
        xdst[q] = ((ch >> 2) * NT + (row >> 4)) * 64 + (ch & 3) * 16 + ((row & 15) ^ ch);
    }
    uintx4 xr[kChunks];
    auto   fetch_x = [&](int kb) {
        const bool inside = kb * kBlockK + k0 < a.K;
#pragma unroll
        for (int q = 0; q < kChunks; ++q) {
            xr[q] = *reinterpret_cast<const uintx4*>(xsrc[q] + (inside ? kb * kBlockK : -k0));
            if (!inside)
                xr[q] = uintx4{0, 0, 0, 0};
        }
    };
    auto store_x = [&](int buf) {
#pragma unroll
        for (int q = 0; q < kChunks; ++q)
            slab[buf][xdst[q]] = xr[q];
    };
    // The 16 and the zero points go off a group's products with the sum of X from a product with ones, of which every wave makes its
    // own; finer groups than 128 leave them in, and a product in float32 takes them off two blocks at once.  Measured with / without
    // the latter: 9216x36864, N = 64, groups of 64 76.4 / 83.4 us; groups of 128, 20480x5120, N = 24 23.9 / 22.7, 4096x11008,
    // N = 48 18.1 / 17.6.
    constexpr bool kZeros = G == 128;
    Weights<R, G> set[2];
    auto          work = [&](const Weights<R, G>& w, int buf) {
        multiply<NT, R, G, BF16, kZeros>(y, w, [&](int j, int n) {
            return __builtin_bit_cast(vec, slab[buf][(j * NT + n) * 64 + h * 16 + (c ^ (4 * j + h))]);
        });
    };
    // A span, two blocks (one with groups of 32), has four sums of X for every column, over 64 (32) columns of W each.  A wave
    // makes two products' worth of a block's for all; `correct` takes them off, times (16 + z) scale of row c and sum h (exact in
    // float32), a step after the span, when a barrier has made them everybody's.
    static_assert(2 * NT == WAVES, "");
    constexpr int kSums = G == 32 ? 4 : 2, kSpan = 4 / kSums; // sums of a block, blocks of a span
    __shared__ float sums[2][4][16 * NT];
    const uint16_t*  coef_s[R];
    const uint8_t*   coef_z[R];
    uint16_t         scale[R];
    uint8_t          zero[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t tile = min(tile0 + r, l.tiles - 1);
        coef_s[r] = reinterpret_cast<const uint16_t*>(a.packed + l.scales) + tile * l.groups * 16 + c;
        coef_z[r] = a.packed + l.zeros + (tile * l.blocks * 4 + (c >> 2)) * (kBlockK / G) * 4 + (c & 3);
        scale[r] = 0, zero[r] = 0;
    }
    auto fetch_coef = [&](int kb) {
        constexpr int kGroups = kBlockK / G;
        const int     block = min(kb + h / kSums, l.blocks - 1), g = h % kGroups;
#pragma unroll
        for (int r = 0; r < R; ++r) { // a group past the end meets zeros of X
            scale[r] = coef_s[r][min(block * kGroups + g, l.groups - 1) * 16];
            zero[r]  = coef_z[r][(block * 4 * kGroups + g) * 4];
        }
    };
    auto add_up = [&](int slot, int buf, int block) {
        const vec ones = __builtin_bit_cast(vec, uintx4{Types<BF16>::kOne, Types<BF16>::kOne, Types<BF16>::kOne, Types<BF16>::kOne});
        const int n = wave >> 1, j = 2 * (wave & 1);
        const vec x0 = __builtin_bit_cast(vec, slab[buf][(j * NT + n) * 64 + h * 16 + (c ^ (4 * j + h))]);
        const vec x1 = __builtin_bit_cast(vec, slab[buf][((j + 1) * NT + n) * 64 + h * 16 + (c ^ (4 * j + 4 + h))]);
        const floatx4 none{0.f, 0.f, 0.f, 0.f};
        floatx4       s0 = Types<BF16>::mfma(ones, x0, none);
        if constexpr (G == 32) {
            const floatx4 s1 = Types<BF16>::mfma(ones, x1, none);
            if (h == 0)
                sums[slot][j][n * 16 + c] = s0[0], sums[slot][j + 1][n * 16 + c] = s1[0];
        } else {
            s0 = Types<BF16>::mfma(ones, x1, s0);
            if (h == 0)
                sums[slot][2 * block + (wave & 1)][n * 16 + c] = s0[0];
        }
    };
    auto correct = [&](const float (&coef)[R], int slot, int kb) {
        const int  block = kb + h / kSums;
        const bool there = block >= first && block < last;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float xs = sums[slot][h][n * 16 + c];
#pragma unroll
            for (int r = 0; r < R; ++r)
                y[r][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(coef[r], there ? xs : 0.f, y[r][n], 0, 0, 0);
        }
    };
    auto coefs = [&](float (&coef)[R]) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            coef[r] = -(float)zero[r] * from16(scale[r], BF16);
    };
    int  kb   = first;
    auto step = [&](const Weights<R, G>& now, Weights<R, G>& next, int buf) { // block kb is in slab `buf`, X of the next in registers
        source.template fetch<kZeros>(next, min(kb + 1, last - 1));
        store_x(buf ^ 1);
        fetch_x(min(kb + 2, last - 1));
        const int  at    = kb - first, slot = at / kSpan & 1;
        const bool start = kSpan == 1 || buf == 0; // of a span
        float      coef[R];
        if (!kZeros && start) {
            coefs(coef); // of the span before, zeros at first
            fetch_coef(kb);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (!kZeros)
            add_up(slot, buf, at % kSpan);
        work(now, buf);
        if (!kZeros && start)
            correct(coef, slot ^ 1, kb - kSpan);
        __syncthreads();
        ++kb;
    };
    if (first < last) {
        fetch_x(kb);
        source.template fetch<kZeros>(set[0], kb);
        store_x(0);
        fetch_x(min(kb + 1, last - 1));
        __syncthreads();
        while (true) {
            step(set[0], set[1], 0);
            if (kb >= last)
                break;
            step(set[1], set[0], 1);
            if (kb >= last)
                break;
        }
        if (!kZeros) {
            const int span = (last - first - 1) / kSpan;
            float     coef[R];
            coefs(coef);
            correct(coef, span & 1, first + span * kSpan);
        }
    }
    const unsigned bad = infinite_sums<NT, R>(y);
    auto           finish = [&](int col, int m, float sum) {
        if (a.bias != nullptr)
            sum += from16(a.bias[m], BF16);
        a.y[(int64_t)col * a.M + m] = to16(activate(sum, a.act), BF16);
    };
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int col = n0 + n * 16 + c;
        if (col >= a.N)
            continue;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int m = (tile0 + r) * 16 + 4 * h;
            if (a.splits > 1) { // the slabs' rows are padded to whole tiles
                if (tile0 + r < l.tiles)
                    *reinterpret_cast<floatx4*>(a.part + ((int64_t)blockIdx.z * a.N + col) * (l.tiles * 16) + m) = y[r][n];
                continue;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (m + i < a.M)
                    finish(col, m + i, y[r][n][i]);
        }
    }
    if (__builtin_expect(__any(bad != 0), 0)) {
        for (int at = 0; at < R * NT; ++at) {
            const int r = at / NT, n = at % NT, col = n0 + n * 16 + c;
            if (!__any((bad >> (4 * at) & 15u) != 0))
                continue;
            const floatx4 sum = sum_again<G, BF16>(a, l, bad >> (4 * at) & 15u, tile0 + r, n0 + n * 16, first, last, 1, lane);
            for (int i = 0; i < 4; ++i) {
                const int m = (tile0 + r) * 16 + 4 * h + i;
                if ((bad >> (4 * at + i) & 1u) == 0 || col >= a.N || tile0 + r >= l.tiles)
                    continue;
                if (a.splits > 1)
                    a.part[((int64_t)blockIdx.z * a.N + col) * (l.tiles * 16) + m] = sum[i];
                else if (m < a.M)
                    finish(col, m, sum[i]);
            }
        }
    }
}

// Sums the slabs of a split K: four rows of a column per thread, and the slabs dealt to the workgroup's waves, whose sums meet
// in LDS (66 slabs of 529x50 one after the other in every thread: 20 us more).
constexpr int kJoinWaves = 4;

__global__ __launch_bounds__(64 * kJoinWaves) void w4_join(LinearArgs a, int bf16)
{
    __shared__ floatx4 sums[kJoinWaves][64];
    const int     lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int     quads = (a.M + 15) / 16 * 4;
    const int     at = blockIdx.x * 64 + lane, col = at / quads, m = at % quads * 4;
    const int64_t slab = (int64_t)a.N * (quads * 4);
    floatx4       sum{0.f, 0.f, 0.f, 0.f};
    if (col < a.N) {
        const float* part = a.part + (int64_t)at * 4;
#pragma unroll 4
        for (int s = wave; s < a.splits; s += kJoinWaves)
            sum += *reinterpret_cast<const floatx4*>(part + s * slab);
    }
    sums[wave][lane] = sum;
    __syncthreads();
    if (wave != 0 || col >= a.N)
        return;
#pragma unroll
    for (int w = 1; w < kJoinWaves; ++w)
        sum += sums[w][lane];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (m + i < a.M)
            a.y[(int64_t)col * a.M + m + i] =
                to16(activate(sum[i] + (a.bias != nullptr ? from16(a.bias[m + i], bf16) : 0.f), a.act), bf16);
}

namespace {

// How a call runs: w4_linear with `row_tiles` tiles a workgroup, or w4_linear_wide with `column_tiles` tiles a workgroup and
// the blocks of K in `splits` shares.
struct Plan {
    int row_tiles;    // of w4_linear; 0: w4_linear_wide
    int column_tiles; // of w4_linear_wide, 2 or 4
    int splits;       // shares of K
};

#ifdef SPMM_KEEP_VARIANTS
Plan g_plan{0, 0, 0};
#endif

constexpr int kWideTiles = 2; // row tiles of a wave of the wide kernel
constexpr int kMostShares = 64; // of K, for the wide kernel
constexpr int wide_waves(int column_tiles) { return column_tiles == 2 ? 4 : 8; }

// The most row tiles w4_linear's registers hold (finer groups have more scales).
constexpr int most_tiles(int group) { return group == 128 ? 7 : (group == 64 ? 5 : 4); }

// The cheapest by a model of a call's time in microseconds, fitted to calls of 512x1024 to 28672x7168 and 9216x36864 with 1 to
// 64 columns.  w4_linear's workgroups are counted in rounds of 256, one for every CU.  That is what the registers leave from three row
// tiles on (two in groups of 32); of fewer a CU holds two or three, which the model does not count.  A step, a block of K for each
// of a workgroup's 8 waves, takes 0.4 for a row tile and 0.6 for X: 28672x7168, N = 16, fp16, groups of 128, with 7 / 4 / 2 / 1 row tiles 26.7 / 33.9 /
// 40.7 / 59.5 us.  K in shares, so that few rows fill the CUs with many row tiles each: 5120x20480, N = 16 22.6 us with five
// row tiles in four shares, 32.5 at best in one; 7168x28672, N = 8 26.7 (seven in four) and 29.4; 4096x11008, N = 4 15.6 at
// best in shares, 13.3 in one.  Columns past 16 are workgroups of their own.
// The wide kernel takes a block of K in step[0] with two column tiles and one workgroup on a CU, in step[1] with two on it, and in
// step[2] with four column tiles, 5 for launch and ends, and with shares 2 for the second launch and their bytes: 5120x5120,
// N = 32, groups of 128 12.9 (w4_linear 12.6); 20480x5120, N = 24 22.0 (29.8) and N = 64 29.2 with four, 36.6 with two column
// tiles (57.0); 640x8192, N = 64, groups of 64 10.2 with 16 shares, 12.7 with 8 and 14.5 with 64 (11.0); 529x25184, N = 50,
// groups of 32 17.2 with 24 shares of two column tiles, 20.8 with 66 of four (24.0); 512x1024 with N = 64 8.6 (4.0).
Plan plan_of(int M, int N, int K, int group)
{
#ifdef SPMM_KEEP_VARIANTS // the tests' build: every kernel at small sizes
    if (g_plan.splits > 0 && g_plan.row_tiles <= most_tiles(group))
        return g_plan;
#endif
    const int64_t tiles = (M + 15) / 16, blocks = (K + kBlockK - 1) / kBlockK;
    auto          up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    Plan          p{1, 0, 1};
    double        best = 1e30;
    for (int r = 1; r <= most_tiles(group); ++r)
        for (int s = 1; s <= 8 && 16 * s <= std::max<int64_t>(16, blocks); ++s) {
            double us = 3.0 + (double)(up(up(tiles, r) * up(N, 16) * s, 256) * up(up(blocks, s), 8)) * (0.4 * r + 0.6);
            if (s > 1) // the sum of the shares: a launch, and every share written and read
                us += 6.0 + s * (double)M * N * 8.0 / 4.9e6;
            if (us < best)
                best = us, p = Plan{r, 0, s};
        }
    if (N <= 16)
        return p;
    const double step32[3] = {1.0, 1.8, 2.3}, step64[3] = {0.74, 1.25, 1.6}, step128[3] = {0.58, 1.1, 1.25};
    const double* step = group == 32 ? step32 : (group == 64 ? step64 : step128);
    for (int nt = 2; nt <= 4; nt += 2) {
        const int64_t groups = up(tiles, kWideTiles * wide_waves(nt)) * up(N, 16 * nt);
        for (int fill = 0; fill <= 512; fill += 256) { // shares for none, one or two workgroups on every CU
            int64_t       s   = std::max<int64_t>(1, std::min<int64_t>({fill / groups, blocks, kMostShares}));
            const int64_t per = up(blocks, s), rest = groups * up(blocks, per) % 512, full = groups * up(blocks, per) / 512;
            s                 = up(blocks, per);
            double us = 5.0;
            if (nt == 4)
                us += (double)(per * up(groups * s, 256)) * step[2];
            else
                us += (double)per * ((double)full * step[1] + (rest > 256 ? step[1] : (rest > 0 ? step[0] : 0.0)));
            if (s > 1)
                us += 2.0 + (double)s * M * N * 8.0 / 6e6;
            if (us < best)
                best = us, p = Plan{0, nt, (int)s};
        }
    }
    return p;
}

size_t workspace_of(int M, int N, const Plan& p)
{
    return p.splits > 1 ? (size_t)p.splits * N * ((M + 15) / 16 * 16) * sizeof(float) : 0;
}

int run_join(hipStream_t stream, const LinearArgs& a, bool bf16)
{
    const int64_t quads = (int64_t)((a.M + 15) / 16) * 4 * a.N;
    return launch(w4_join, dim3((unsigned)((quads + 63) / 64), 1, 1), dim3(64 * kJoinWaves, 1, 1), stream, a, (int)bf16);
}

template <int R, int G, bool BF16>
int run_narrow(hipStream_t stream, int row_tiles, const LinearArgs& a)
{
    if constexpr (R > 1)
        if (row_tiles < R)
            return run_narrow<R - 1, G, BF16>(stream, row_tiles, a);
    const unsigned tiles = (unsigned)(a.M + 15) / 16;
    const int      err   = launch(w4_linear<R, G, BF16>, dim3((tiles + R - 1) / R, (unsigned)(a.N + 15) / 16, (unsigned)a.splits),
                                  dim3(64 * kWaves, 1, 1), stream, a);
    return err != 0 || a.splits == 1 ? err : run_join(stream, a, BF16);
}

template <int NT, int G, bool BF16>
int run_wide(hipStream_t stream, const LinearArgs& a)
{
    constexpr int      W = wide_waves(NT);
    constexpr unsigned kRows = W * kWideTiles;
    const unsigned     tiles = (unsigned)(a.M + 15) / 16;
    const int          err   = launch(w4_linear_wide<NT, kWideTiles, G, BF16, W>,
                                      dim3((tiles + kRows - 1) / kRows, (unsigned)(a.N + 16 * NT - 1) / (16 * NT), (unsigned)a.splits),
                                      dim3(64 * W, 1, 1), stream, a);
    return err != 0 || a.splits == 1 ? err : run_join(stream, a, BF16);
}

template <int G, bool BF16>
int run_linear(hipStream_t stream, const Plan& p, const LinearArgs& a)
{
    if (p.row_tiles > 0)
        return run_narrow<most_tiles(G), G, BF16>(stream, p.row_tiles, a);
    return p.column_tiles == 2 ? run_wide<2, G, BF16>(stream, a) : run_wide<4, G, BF16>(stream, a);
}

int check_weights(int M, int K, int group, int dtype)
{
    if (group != 32 && group != 64 && group != 128)
        return refuse("a group of %d columns: 32, 64 or 128", group);
    if (M < 1 || M > 16 * 65535 || K < group || K > kMaxK || K % group != 0)
        return refuse("weights of %d rows (at most 16 * 65535) and %d columns (a multiple of %d, at most 2^30)", M, K, group);
    if (dtype != DECODE_FP16 && dtype != DECODE_BF16)
        return refuse("unknown element type %d", dtype);
    return 0;
}

} // namespace
} // namespace decode

using namespace decode;

#ifdef SPMM_KEEP_VARIANTS
// Every later call runs as the plan says (see Plan); splits 0: as the library chooses.
extern "C" int W4_Debug_SetPlan(int row_tiles, int column_tiles, int splits)
{
    if (row_tiles < 0 || splits < 0 || splits > kMostShares || (splits > 0 && row_tiles == 0 && column_tiles != 2 && column_tiles != 4))
        return 1;
    g_plan = Plan{row_tiles, column_tiles, splits};
    return 0;
}
#endif

extern "C" size_t W4_PackedBytes(int M, int K, int group)
{
    if ((group != 32 && group != 64 && group != 128) || M < 1 || M > 16 * 65535 || K < group || K > kMaxK || K % group != 0)
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

extern "C" size_t W4_WorkspaceBytes(int M, int N, int K, int group)
{
    if (W4_PackedBytes(M, K, group) == 0 || N < 1 || N > kMaxColumns)
        return 0;
    return workspace_of(M, N, plan_of(M, N, K, group));
}

extern "C" int W4_Linear(hipStream_t stream, const void* packed, const void* X, int64_t x_stride, void* Y, int M, int N,
                         int K, int group, const void* bias, int activation, void* workspace, size_t workspace_bytes,
                         int dtype)
{
    if (int e = check_weights(M, K, group, dtype))
        return e;
    if (N < 0 || N > kMaxColumns)
        return refuse("%d columns of X (0 to %d)", N, kMaxColumns);
    if (activation < 0 || activation > 2)
        return refuse("unknown activation %d (0 none, 1 ReLU, 2 GELU)", activation);
    if (N == 0)
        return 0;
    if (bad_pointer(packed, 16) || bad_pointer(X, 16) || bad_pointer(Y, 2) || (bias != nullptr && bad_pointer(bias, 2)) ||
        (N > 1 && x_stride < K) || x_stride % 8 != 0)
        return refuse("a null or misaligned weight, X (16 bytes, rows too), Y or bias (2)");
    const Plan   p    = plan_of(M, N, K, group);
    const size_t need = workspace_of(M, N, p);
    if (need > 0 && (bad_pointer(workspace, 16) || workspace_bytes < need))
        return refuse("workspace of %zu bytes (16-byte aligned), %zu needed", workspace == nullptr ? (size_t)0 : workspace_bytes, need);
    LinearArgs a{};
    a.packed = static_cast<const uint8_t*>(packed), a.x = static_cast<const uint16_t*>(X), a.x_stride = x_stride;
    a.y = static_cast<uint16_t*>(Y), a.bias = static_cast<const uint16_t*>(bias), a.part = static_cast<float*>(workspace);
    a.M = M, a.N = N, a.K = K, a.act = activation, a.splits = p.splits;
    const bool bf16 = dtype == DECODE_BF16;
    if (group == 32)
        return bf16 ? run_linear<32, true>(stream, p, a) : run_linear<32, false>(stream, p, a);
    if (group == 64)
        return bf16 ? run_linear<64, true>(stream, p, a) : run_linear<64, false>(stream, p, a);
    return bf16 ? run_linear<128, true>(stream, p, a) : run_linear<128, false>(stream, p, a);
}
