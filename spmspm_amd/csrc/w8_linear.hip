// Linears of 8-bit integers: W8_Pack, W8_Linear, W8_Gated (w8_api.h).
//
// Mathematics.  Y[n][m] = act(sx[n] sw[m] sum_k cx[n][k] cw[m][k] + b[m]): the matrix cores take the sums in whole numbers, exactly and
// in any order, so that K may be split among waves and workgroups at will without a result changing; scales, bias and
// activation are applied to a sum in float32.
//
// Packed weights.  Blocks of 16 rows x 64 columns, 1 KB, in the order in which v_mfma_i32_16x16x64_i8 takes its first operand: 16 bytes a
// lane, lane r + 16 q has columns 16 q .. 16 q + 15 of row r.  Four row tiles make a group of 64 rows, whose order is chosen for the
// results: after the product a lane r + 16 q holds, of column r of X, rows 4 q .. 4 q + 3 of every tile.  Row 16 q + 4 t + i of the group
// is put at row 4 q + i of tile t, so that these are 16 consecutive outputs, 32 bytes of Y.  In gated weights tiles 0 and 1 hold 32
// rows of the gate (row 8 q + 4 t + i), tiles 2 and 3 the same rows of up: both sums of an output meet in one lane.
// K is filled up with zeros to a multiple of 128: what X has there does not matter.  Of every 128 columns the groups lie one behind the
// other, 8 KB each, two steps of four tiles: workgroups that are equally far along K read one stretch of memory, where rows that
// lay whole would be a power of two apart and meet on the same channels.
#include "w8_common.hiph"

#include <algorithm>
#include <type_traits>

namespace decode {
namespace {

constexpr int kMaxRows8 = 1 << 24;
constexpr int kGroup8   = 8192; // bytes of a group's 128 columns
constexpr int kMaxN8    = 16 * 65535;

struct Layout8 {
    int     groups, steps; // groups of 64 packed rows, steps of 64 columns (an even number)
    int64_t scales, bytes; // offset of the scales (float32; of the gate, then of up), size
};

__host__ __device__ inline Layout8 layout8(int M, int K, bool gated)
{
    Layout8 l;
    l.groups = gated ? (M + 31) / 32 : (M + 63) / 64;
    l.steps  = (K + 127) / 128 * 2;
    l.scales = (int64_t)l.groups * l.steps * 4096;
    l.bytes  = l.scales + (int64_t)l.groups * 64 * 4;
    return l;
}

struct PackArgs {
    const int8_t *w, *up;
    const float * scales, *up_scales;
    int64_t       w_stride, up_stride;
    int           M, K;
    uint8_t*      packed;
};

// A workgroup lays out the 128 columns of a group, a wave a row tile's.
__global__ __launch_bounds__(256) void w8_pack(PackArgs a)
{
    const bool    gated = a.up != nullptr;
    const Layout8 l     = layout8(a.M, a.K, gated);
    const int     lane = threadIdx.x % kWave, tile = threadIdx.x / kWave, r = lane & 15, q = lane >> 4;
    const int     group = blockIdx.x % l.groups, block = blockIdx.x / l.groups;
    const bool    second = gated && tile >= 2;
    const int     row = gated ? group * 32 + (r >> 2) * 8 + (tile & 1) * 4 + (r & 3) : group * 64 + (r >> 2) * 16 + tile * 4 + (r & 3);
    const int8_t* src = second ? a.up + row * a.up_stride : a.w + row * a.w_stride;
    uintx4*       to  = reinterpret_cast<uintx4*>(a.packed + (int64_t)blockIdx.x * kGroup8) + tile * 64 + lane;
    for (int step = 0; step < 2; ++step) {
        const int k   = block * 128 + step * 64 + q * 16;
        uintx4    out = 0;
        if (row < a.M && k + 16 <= a.K)
            out = *reinterpret_cast<const loose_bytes16*>(src + k);
        else if (row < a.M)
            for (int b = 0; b < 16; ++b)
                if (k + b < a.K)
                    out[b / 4] |= (unsigned)(uint8_t)src[k + b] << (8 * (b % 4));
        to[step * 256] = out;
    }
    if (block == 0 && tile == 0) { // 64 scales: of the group's rows, or of 32 rows of the gate and of up
        const int  per = gated ? 32 : 64, m = group * per + lane % per;
        const bool u = gated && lane >= 32;
        reinterpret_cast<float*>(a.packed + l.scales)[(u ? (int64_t)l.groups * 32 : 0) + m] =
            m < a.M ? (u ? a.up_scales[m] : a.scales[m]) : 0.f;
    }
}

struct ProductArgs {
    const uint8_t* packed;
    const int8_t*  x;
    const float*   x_scales;
    int64_t        x_stride;
    uint16_t*      y;
    const uint16_t *bias, *up_bias;
    int*           part; // sums of the shares of K (part_of); null where K is not split
    int            M, N, K, act, bf16;
    int            shares, per; // shares of K, blocks of 128 columns in each but the last
    int            row_tiles, column_tiles; // of w8_tiles
};

// The kernel's arguments, read from memory once more where a tile begins and ends: kept in registers from the kernel's start they would
// leave too few scalars for its loop.
__device__ __forceinline__ ProductArgs late_args8()
{
    typedef const __attribute__((address_space(4))) ProductArgs* Pointer;
    Pointer p = (Pointer)(uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    ProductArgs a{};
    a.packed = p->packed, a.x = p->x, a.x_scales = p->x_scales, a.x_stride = p->x_stride, a.y = p->y, a.bias = p->bias;
    a.up_bias = p->up_bias, a.part = p->part, a.M = p->M, a.N = p->N, a.K = p->K, a.act = p->act, a.bf16 = p->bf16, a.shares = p->shares;
    a.per = p->per, a.row_tiles = p->row_tiles, a.column_tiles = p->column_tiles;
    return a;
}

// ReLU, GELU (tanh form) or SiLU of W sums.  The last two are y / (1 + exp(-z)), with z = 2 sqrt(2/pi) (y + 0.044715 y^3), since
// (1 + tanh u) / 2 = 1 / (1 + exp(-2 u)), or z = y; far from 0 they end at 0 and y.  The exponential is one of 2, with -log2(e) in z's
// coefficients; the reciprocal's last bit is far below 16 bits.
template <int W>
__device__ __forceinline__ void activate8(float* y, int act)
{
    constexpr float kLog2e = 1.4426950408889634f, kOne = -kLog2e * 1.5957691216057308f, kCube = kOne * 0.044715f;
    if (act == 1) {
        for (int i = 0; i < W; ++i)
            y[i] = y[i] < 0.f ? 0.f : y[i]; // a NaN stays one
    } else if (act == 2) {
        for (int i = 0; i < W; ++i)
            y[i] *= __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(y[i] * (kOne + kCube * y[i] * y[i])));
    } else if (act == 3) {
        for (int i = 0; i < W; ++i)
            y[i] *= __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2e * y[i]));
    }
}

template <int W>
struct Loose { // W 16-bit numbers at any alignment of theirs
    typedef uint16_t type __attribute__((ext_vector_type(W)));
    typedef type __attribute__((aligned(2))) loose;
};

// What W consecutive outputs from row `m` on have in common over the columns.
template <bool GATED, int W>
struct Tail8 {
    float sw[W], su[W], b[W], bu[W];
    int   m, left;

    static __device__ __forceinline__ void biases(float* to, const uint16_t* p, int left, bool bf16)
    {
        typename Loose<W>::type v = 0;
        if (p != nullptr && left >= W)
            v = *reinterpret_cast<const typename Loose<W>::loose*>(p);
        else if (p != nullptr)
            for (int i = 0; i < W - 1; ++i)
                if (i < left)
                    v[i] = p[i];
        for (int i = 0; i < W; ++i)
            to[i] = from16(v[i], bf16);
    }

    __device__ __forceinline__ Tail8(const ProductArgs& a, const Layout8& l, int row) : m(row), left(a.M - row)
    {
        if (left <= 0)
            return;
        const float* s = reinterpret_cast<const float*>(a.packed + l.scales) + m; // the layout's rows go past M
        biases(b, a.bias == nullptr ? nullptr : a.bias + m, left, a.bf16);
        if (GATED)
            biases(bu, a.up_bias == nullptr ? nullptr : a.up_bias + m, left, a.bf16);
        for (int i = 0; i < W; ++i) {
            sw[i] = s[i];
            if (GATED)
                su[i] = s[i + (int64_t)l.groups * 32];
        }
    }

    // From LDS: scales, and biases as 32-bit words of 16 bits; those of up `up` words behind the gate's.
    __device__ __forceinline__ Tail8(const ProductArgs& a, int row, const float* s, const unsigned* bias, int up) : m(row), left(a.M - row)
    {
        for (int i = 0; i < W; ++i) {
            sw[i] = s[i], b[i] = a.bias != nullptr ? from16((uint16_t)bias[i], a.bf16) : 0.f;
            if (GATED)
                su[i] = s[up + i], bu[i] = a.up_bias != nullptr ? from16((uint16_t)bias[up + i], a.bf16) : 0.f;
        }
    }

    // What a column's sums, of the gate in a gated product, are ahead of the activation; sx is the scale of its row of X.
    __device__ __forceinline__ void scale(float* y, const int* sum, float sx) const
    {
        for (int i = 0; i < W; ++i)
            y[i] = (float)sum[i] * sw[i] * sx + b[i];
    }

    // The gate's times the sums of up.
    __device__ __forceinline__ void times(float* y, const int* up, float sx) const
    {
        for (int i = 0; i < W; ++i)
            y[i] *= (float)up[i] * su[i] * sx + bu[i];
    }

    // Into column n.
    __device__ __forceinline__ void put(const ProductArgs& a, int n, const float* y) const
    {
        if (left <= 0)
            return;
        typename Loose<W>::type out;
        if (a.bf16)
            for (int i = 0; i < W; ++i)
                out[i] = __builtin_bit_cast(uint16_t, (__bf16)y[i]);
        else
            for (int i = 0; i < W; ++i)
                out[i] = __builtin_bit_cast(uint16_t, (_Float16)y[i]);
        uint16_t* to = a.y + (int64_t)n * a.M + m;
        if (left >= W) {
            *reinterpret_cast<typename Loose<W>::loose*>(to) = out;
            return;
        }
        for (int i = 0; i < W - 1; ++i)
            if (i < left)
                to[i] = out[i];
    }

    // The three of one column; `up` is read by gated products only.
    __device__ __forceinline__ void store(const ProductArgs& a, int n, float sx, const int* sum, const int* up) const
    {
        if (left <= 0)
            return;
        float y[W];
        scale(y, sum, sx);
        activate8<W>(y, a.act);
        if constexpr (GATED)
            times(y, up, sx);
        put(a, n, y);
    }
};

// The sums of a share of K go to memory as the matrix cores leave them: of a group and a tile of 16 columns, four tiles of 1 KB.
__device__ __forceinline__ intx4* part_of(const ProductArgs& a, int groups, int share, int columns, int group, int column)
{
    return reinterpret_cast<intx4*>(a.part) + (((int64_t)share * columns + column) * groups + group) * 256;
}

// Shares of K: a second launch and their bytes, 9216x36864 with 193 columns in seven shares 10 us for 54 MB.
// A wave ends half a group, tiles h and h + 2 of a gated product, 2 h and 2 h + 1 otherwise, of 16 columns from the sums of all shares.
template <bool GATED>
__global__ __launch_bounds__(256) void w8_join(ProductArgs a)
{
    const Layout8 l = layout8(a.M, a.K, GATED);
    const int     lane = threadIdx.x % kWave, columns = (a.N + 15) / 16;
    const int64_t unit = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
    const int     h = (int)(unit & 1), group = (int)(unit / 2 % l.groups), column = (int)(unit / 2 / l.groups);
    const int     n = column * 16 + (lane & 15), q = lane >> 4;
    if (n >= a.N)
        return;
    const intx4*  p    = part_of(a, l.groups, 0, columns, group, column) + (GATED ? h : 2 * h) * 64 + lane;
    const int64_t next = (int64_t)columns * l.groups * 256;
    intx4         sum[2] = {0, 0};
#pragma unroll 8
    for (int s = 0; s < a.shares; ++s)
        for (int t = 0; t < 2; ++t)
            sum[t] += p[s * next + t * (GATED ? 128 : 64)];
    int v[8];
    for (int i = 0; i < 8; ++i)
        v[i] = sum[i / 4][i % 4];
    if constexpr (GATED)
        Tail8<true, 4>(a, l, group * 32 + 8 * q + 4 * h).store(a, n, a.x_scales[n], v, v + 4);
    else
        Tail8<false, 8>(a, l, group * 64 + 16 * q + 8 * h).store(a, n, a.x_scales[n], v, nullptr);
}

// Few columns: a workgroup of kNarrowWaves waves takes R row tiles and NT column tiles, its waves every kNarrowWaves-th block of 128 columns of
// its share of K.  W is read once and goes from memory into the matrix operands as it is packed.  X comes eight rows of 128 bytes to a
// load and takes the operands' order in a corner of LDS that the wave has for itself (read in that order, 16 rows at once, a load
// keeps the address unit four times as long: 2.3 us for every 16 columns of 5120).  A wave has D blocks of both in flight.  The
// waves' sums meet in LDS.  A gated product has rows of the gate and of up in every workgroup: tiles t and t + 2 with R = 2.
// X16: X holds 16-bit rows, eight at most, which every workgroup rounds to 8 bits for itself: a launch less.  Its first blocks of W are
// asked for ahead of the rows, whose maxima therefore wait for them (5120x5120, N = 1 9.2 us of a Python caller, 7.5 on given codes).
// Bound by memory: 28672x7168 with 16 columns 34 us, 6.0 TB/s of W; 13696x5120 gate and up of one token 25 us, 5.6 TB/s.
constexpr int kNarrowWaves = 8;
constexpr int kRows16      = 8;

// What a wave wrote to LDS is there for its other lanes, and what they read may be written over: no instruction, the wave's
// accesses keep their order.
__device__ __forceinline__ void wave_handoff8()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <bool GATED, int R, int NT, int D, bool X16>
__global__ __launch_bounds__(64 * kNarrowWaves) void w8_narrow(ProductArgs a, int column_tiles)
{
    static_assert((!GATED || R >= 2) && (!X16 || NT == 1));
    __shared__ unsigned top[X16 ? kRows16 : 1][kNarrowWaves];
    __shared__ int   total[R * NT][kWave][4];
    __shared__ intx4 turned[kNarrowWaves][NT][2][kWave]; // X: 8 rows a KB, row r's chunk c at place 8 r + (c ^ r)
    const Layout8  l    = layout8(a.M, a.K, GATED);
    const int      lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), c = lane & 15, q = lane >> 4;
    const int      unit = blockIdx.x / column_tiles, n0 = blockIdx.x % column_tiles * (NT * 16), share = blockIdx.y;
    const int      group = unit * R / 4, first = unit % (4 / R) * (GATED ? 1 : R), apart = GATED && R == 2 ? 2 : 1; // of its row tiles
    const int      from = share * a.per, to = min(from + a.per, l.steps / 2);
    const int      last = (a.K - 1) / 16 * 16;
    for (int i = threadIdx.x; i < R * NT * kWave; i += 64 * kNarrowWaves)
        reinterpret_cast<intx4*>(total)[i] = 0;
    if constexpr (!X16)
        __syncthreads();

    const intx4*  w = reinterpret_cast<const intx4*>(a.packed + (int64_t)group * kGroup8) + first * 64 + lane;
    const int8_t* x[NT][2];
    for (int u = 0; u < NT; ++u) // rows behind the last are the last again
        for (int s = 0; s < 2; ++s)
            x[u][s] = a.x + (int64_t)min(n0 + u * 16 + s * 8 + (lane >> 3), a.N - 1) * a.x_stride * (X16 ? 2 : 1);
    struct Block {
        intx4   w[2][R], x[X16 ? 1 : NT][2];
        shortx8 x16[2];
    };
    Block held[D];
    auto  fetch = [&](Block& h, int block) {
        if constexpr (X16)
            for (int i = 0; i < 2; ++i)
                h.x16[i] = load8(reinterpret_cast<const uint16_t*>(x[0][0]), block * 128 + 16 * (lane & 7) + 8 * i, a.K);
        for (int u = 0; u < (X16 ? 0 : NT); ++u) // behind the last 16 columns of X the weights are 0
            for (int s = 0; s < 2; ++s)
                h.x[u][s] = *reinterpret_cast<const intx4*>(x[u][s] + min(block * 128 + 16 * (lane & 7), last));
        for (int s = 0; s < 2; ++s)
            for (int t = 0; t < R; ++t)
                h.w[s][t] = __builtin_nontemporal_load(w + (int64_t)block * l.groups * (kGroup8 / 16) + (s * 4 + t * apart) * 64);
    };
    intx4 sum[R][NT];
    for (int t = 0; t < R; ++t)
        for (int u = 0; u < NT; ++u)
            sum[t][u] = 0;
    for (int d = 0; d < D; ++d)
        if (from + wave + d * kNarrowWaves < to)
            fetch(held[d], from + wave + d * kNarrowWaves);
    Row8 mine{};
    auto row8 = [&](int n) { // what the codes of row n are made with
        unsigned bits = 0;
        for (int w = 0; w < kNarrowWaves; ++w)
            bits = max(bits, top[X16 ? n : 0][w]);
        return Row8(bits);
    };
    if constexpr (X16) {
        for (int n = 0; n < a.N; ++n) {
            const uint16_t* row  = reinterpret_cast<const uint16_t*>(a.x) + n * a.x_stride;
            unsigned        bits = 0; // of the largest magnitude: an infinity or a NaN is larger than every number
            for (int e = threadIdx.x * 8; e < a.K; e += 512 * kNarrowWaves) {
                const shortx8 v = load8(row, e, a.K);
                for (int i = 0; i < 8; ++i)
                    bits = max(bits, __float_as_uint(from16(v[i], a.bf16)) & 0x7fffffffu);
            }
            for (int d = 32; d > 0; d >>= 1)
                bits = max(bits, (unsigned)__shfl_xor((int)bits, d));
            if (lane == 0)
                top[n][wave] = bits;
        }
        __syncthreads();
        mine = row8(min(lane >> 3, a.N - 1));
    }
    for (int block = from + wave; block < to;) {
#pragma unroll
        for (int d = 0; d < D; ++d, block += kNarrowWaves) {
            if (block >= to)
                break;
            if constexpr (X16) { // columns past the eighth are not there: what they are multiplied by does not matter
                uintx4 code;
                for (int i = 0; i < 2; ++i) {
                    float t[8];
                    for (int j = 0; j < 8; ++j)
                        t[j] = mine.none ? 0.f : from16(held[d].x16[i][j], a.bf16);
                    const uintx2 c8 = codes8(t, mine.m, mine.inverse);
                    code[2 * i] = c8[0], code[2 * i + 1] = c8[1];
                }
                turned[wave][0][0][(lane & 56) | ((lane & 7) ^ (lane >> 3))] = __builtin_bit_cast(intx4, code);
            }
            for (int u = 0; u < (X16 ? 0 : NT); ++u)
                for (int s = 0; s < 2; ++s)
                    turned[wave][u][s][(lane & 56) | ((lane & 7) ^ (lane >> 3))] = held[d].x[u][s];
            wave_handoff8();
            for (int s = 0; s < 2; ++s)
                for (int u = 0; u < NT; ++u) {
                    const intx4 b = turned[wave][u][c >> 3][(c & 7) * 8 + ((4 * s + q) ^ (c & 7))];
                    for (int t = 0; t < R; ++t)
                        sum[t][u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(held[d].w[s][t], b, sum[t][u], 0, 0, 0);
                }
            wave_handoff8();
            if (block + D * kNarrowWaves < to)
                fetch(held[d], block + D * kNarrowWaves);
        }
    }
    for (int t = 0; t < R; ++t)
        for (int u = 0; u < NT; ++u)
            for (int i = 0; i < 4; ++i)
                __hip_atomic_fetch_add(&total[t * NT + u][lane][i], sum[t][u][i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    __syncthreads();
    if (wave >= NT) // wave u ends column tile u
        return;
    const int n = n0 + wave * 16 + c;
    int       v[4 * R];
    for (int t = 0; t < R; ++t) {
        const intx4 s = *reinterpret_cast<const intx4*>(total[t * NT + wave][lane]);
        if (a.part != nullptr && n0 + wave * 16 < a.N)
            part_of(a, l.groups, share, (a.N + 15) / 16, group, n0 / 16 + wave)[(first + t * apart) * 64 + lane] = s;
        for (int i = 0; i < 4; ++i)
            v[4 * t + i] = s[i];
    }
    if (a.part != nullptr || n >= a.N)
        return;
    constexpr int W  = GATED ? 2 * R : (R == 1 ? 4 : 8); // consecutive outputs of a lane
    const float   sx = X16 ? row8(n).scale : a.x_scales[n];
    const int     m  = GATED ? group * 32 + 8 * q + 4 * first : group * 64 + 16 * q + 4 * first;
    for (int i = 0; i < (GATED ? 1 : R * 4 / W); ++i)
        Tail8<GATED, W>(a, l, m + i * W).store(a, n, sx, v + i * W, v + 2 * R);
}

// f(0) .. f(N - 1) with constants: arrays of registers have no others for an index.
template <int N, int I = 0, typename F>
__device__ __forceinline__ void each(F f)
{
    if constexpr (I < N) {
        f(std::integral_constant<int, I>());
        each<N, I + 1>(f);
    }
}

// A wave's 1 KB of 16 bytes a lane goes from global memory straight into LDS.  In assembly, since the compiler would wait for it
// ahead of the next read of LDS; the kernel waits for it itself, before the barrier that hands the tile over.  OFFSET counts for both
// addresses.
template <int OFFSET>
__device__ __forceinline__ void to_lds(unsigned lds, const void* base, unsigned offset)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3" ::"s"(lds), "v"(offset), "s"(base), "n"(OFFSET)
                 : "memory", "m0");
}

// The same of memory that is read once: the caches are kept for what is read again (36864x9216 with 64 columns 92 -> 87 us).
template <int OFFSET>
__device__ __forceinline__ void to_lds_once(unsigned lds, const void* base, unsigned offset)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3 nt" ::"s"(lds), "v"(offset), "s"(base), "n"(OFFSET)
                 : "memory", "m0");
}

// The same of one word, or of 16 bits in a word, a lane.
__device__ __forceinline__ void word_to_lds(unsigned lds, const void* address)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(address) : "memory", "m0");
}

__device__ __forceinline__ void short_to_lds(unsigned lds, const void* address)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ushort %1, off" ::"s"(lds), "v"(address) : "memory", "m0");
}

// Workgroups are dealt to the eight dies in turn, each with an L2 of its own: consecutive numbers on one die, and there a band of
// kBand row tiles by as many column tiles as run at once; shares of K one after another.
__device__ __forceinline__ void place8(const ProductArgs& a, int id, int& row, int& column, int& share)
{
    constexpr int kBand = 8;
    const int     one = a.row_tiles * a.column_tiles, total = one * a.shares, die = id % 8;
    int           at = die * (total / 8) + min(die, total % 8) + id / 8;
    share            = __builtin_amdgcn_readfirstlane(at / one);
    at -= share * one;
    const int band = at / (kBand * a.column_tiles), first = band * kBand, height = min(kBand, a.row_tiles - first);
    const int in   = at - first * a.column_tiles;
    // divisions are done by vector instructions: back to scalars, which the addresses are made of
    row = __builtin_amdgcn_readfirstlane(first + in % height), column = __builtin_amdgcn_readfirstlane(in / height);
}

// Many columns: bound by the matrix cores and, behind them, by the power that they and the way to them take.
// A workgroup of WM x WN waves takes WM MT x WN NT tiles of 16 x 16 outputs (packed rows x rows of X), a wave MT x NT of them.  K goes by in
// blocks of 128 through a ring of S places in LDS: W's blocks lie there as they are packed, one operand a KB; of X 8 rows lie in a KB,
// row r's chunk c of 16 bytes at place 8 r + (c ^ r), which the matrix operands' reads find without bank conflicts.
// While the products of a block's first half run, the second half's operands are read; then the waves meet, the place that
// all have read takes the block S further on, and the next block's first operands are read under the second half's products.
// A workgroup stays on its CU and takes every gridDim-th tile: the blocks of all its tiles are one stream, so that the next tile is
// loaded while the results of the last are written, and a tile costs its products alone.
// Measured in tiles of 256 x 256: 8192 x 8192 x 8192 398 us, 2760 TOP/s, the matrix cores busy for 65 % of the cycles at 2.0 GHz; with
// operands of zeros 337 us, 3260 TOP/s at a clock that is not throttled; products alone, from registers, reach 4000 TOP/s on random
// codes.  20480 x 5120 with 4096 columns 339 us, 2530 TOP/s.  Lines that the next die-mates miss, brought ahead into L2, help
// operands of zeros (338 -> 312) and not others (400 -> 406).  Rings of steps of 64 436, four waves of 128 x 128 each 764 (the
// accumulators are moved about).
template <bool GATED, int MT, int NT, int WM, int WN, int S>
__global__ __launch_bounds__(64 * WM * WN, 2) void w8_tiles(ProductArgs args)
{
    constexpr int kWaves = WM * WN, kRows = WM * MT, kCols = WN * NT, kStage = (kRows + kCols) * 2048; // tiles of W, of X
    constexpr int kLoads = 2 * (kRows + kCols) / kWaves;
    constexpr int kM = kRows * 16, kN = kCols * 16; // packed rows, rows of X
    constexpr int kEnds = S + 2; // loads are at most S + 1 tiles ahead of the products
    constexpr int kWLoads = 2 * kRows / kWaves, kXLoads = 2 * kCols / kWaves; // of a wave, of W and of X
    static_assert(2 * kRows % kWaves == 0 && 2 * kCols % kWaves == 0 && (kWLoads == 2 || kWLoads == 4));
    static_assert(MT % 4 == 0 && kM % 128 == 0 && kN % 64 == 0 && S >= 2);
    struct Ends { // of a tile: scales and biases of its rows (of the gate, then of up), scales of its rows of X
        float    sw[kM];
        unsigned b[kM];
        float    sx[kN];
    };
    __shared__ __attribute__((aligned(1024))) uint8_t lds[S][kStage];
    __shared__ __attribute__((aligned(16))) Ends      ends[kEnds];
    const int     lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int     q = lane >> 4, c = lane & 15, wm = wave / WN, wn = wave % WN;

    // What a wave brings of every block: kWLoads KBs of W, as they are packed, half a group's or a quarter's, then kXLoads of X.
    const uint8_t* w_now; // W's block of the next load, from the tile's first group on
    const int8_t*  x_at[kXLoads];
    unsigned       w_off, x_off[kXLoads];
    auto address = [](const void* p) { return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void*)p; };
    const unsigned lds0 = address(lds), ends0 = address(ends);
    const int      chunk = 16 * ((lane & 7) ^ (lane >> 3)), last = (args.K - 1) / 16 * 16;
    const int64_t block_bytes = (int64_t)layout8(args.M, args.K, GATED).groups * kGroup8;
    const bool    once        = args.column_tiles == 1;
    const int tiles = args.row_tiles * args.column_tiles * args.shares, apart = gridDim.x;
    // Tile of the loads, their next block and the end of the tile's, tiles seen; tile of the products, blocks of it left, tiles seen.
    int ahead = blockIdx.x - apart, ahead_block, ahead_end, ahead_turn = 0, now = blockIdx.x, left, turn = 0;
    // Turns the loads to the next tile, if there is one, and brings its ends.
    auto enter = [&] {
        if (ahead + apart >= tiles)
            return;
        ahead += apart;
        const ProductArgs a = late_args8();
        const Layout8     l = layout8(a.M, a.K, GATED);
        int               row, column, share;
        place8(a, ahead, row, column, share);
        ahead_block = share * a.per, ahead_end = min(ahead_block + a.per, l.steps / 2);
        const int tile0 = row * kRows, n0 = column * kN;
        w_now = a.packed + (int64_t)ahead_block * block_bytes + (int64_t)(tile0 / 4) * kGroup8;
        // groups and rows behind the last are the last again: computed, not stored
        w_off = min(wave * kWLoads / 8, l.groups - 1 - tile0 / 4) * kGroup8 + wave * kWLoads % 8 * 1024 + lane * 16;
        for (int i = 0; i < kXLoads; ++i) {
            const int n = min(n0 + 8 * (wave * kXLoads + i), a.N - 1);
            x_at[i]     = a.x + (int64_t)n * a.x_stride;
            x_off[i]    = min(lane >> 3, a.N - 1 - n) * (unsigned)a.x_stride;
        }
        const unsigned to = ends0 + ahead_turn++ % kEnds * (unsigned)sizeof(Ends);
        const float*   sw = reinterpret_cast<const float*>(a.packed + l.scales);
        for (int i = wave; i < kM / 64; i += kWaves) { // 64 rows, all of the gate or all of up
            const bool up = GATED && i >= kM / 128;
            const int  at = (GATED ? tile0 * 8 + (up ? i - kM / 128 : i) * 64 : tile0 * 16 + i * 64) + lane;
            const int  most = l.groups * (GATED ? 32 : 64) - 1;
            word_to_lds(to + i * 256, sw + (up ? (int64_t)l.groups * 32 : 0) + min(at, most));
            const uint16_t* bias = up ? a.up_bias : a.bias;
            if (bias != nullptr)
                short_to_lds(to + kM * 4 + i * 256, bias + min(at, a.M - 1));
        }
        for (int i = kWaves - 1 - wave; i < kN / 64; i += kWaves)
            word_to_lds(to + kM * 8 + i * 256, a.x_scales + min(n0 + i * 64 + lane, a.N - 1));
    };
    // The i-th of a wave's loads of a block.  Behind the last 16 columns of X the weights are 0: what is there does not matter.
    auto stage = [&](auto i, int place) {
        const unsigned to = lds0 + place * kStage;
        if constexpr (i < kWLoads) {
            if (kCols <= 4 && once)
                to_lds_once<i * 1024>(to + wave * kWLoads * 1024, w_now, w_off);
            else
                to_lds<i * 1024>(to + wave * kWLoads * 1024, w_now, w_off);
        } else {
            constexpr int x = i - kWLoads;
            to_lds<0>(to + (2 * kRows + wave * kXLoads + x) * 1024, x_at[x], x_off[x] + min(ahead_block * 128 + chunk, last));
        }
    };
    struct Operands {
        intx4 w[MT], x[NT];
    };
    constexpr int kReads = MT + NT, kProducts = MT * NT;
    auto fetch = [&](Operands& o, int i, int place, int half) {
        const uint8_t* p = lds[place];
        if (i < MT)
            o.w[i] = *reinterpret_cast<const intx4*>(p + ((wm * MT + i) / 4 * 8 + half * 4 + i % 4) * 1024 + lane * 16);
        else
            o.x[i - MT] = *reinterpret_cast<const intx4*>(p + (2 * kRows + (wn * NT + i - MT) * 2 + (c >> 3)) * 1024 +
                                                          (c & 7) * 128 + (((4 * half + q) ^ (c & 7)) * 16));
    };
    intx4 sum[MT][NT];
    auto clear = [&] {
        for (int t = 0; t < MT; ++t)
            for (int u = 0; u < NT; ++u)
                sum[t][u] = 0;
    };
    // The products of one half in kParts parts, with `between(part)` behind each: loads issued all at once would hold the wave up
    // ahead of its products until the memory pipe has taken them.
    constexpr int kParts = kProducts / 4;
    auto multiply = [&](const Operands& o, auto between) {
        each<kParts>([&](auto part) {
#pragma unroll
            for (int f = 4 * part; f < 4 * part + 4; ++f)
                sum[f % MT][f / MT] = __builtin_amdgcn_mfma_i32_16x16x64_i8(o.w[f % MT], o.x[f / MT], sum[f % MT][f / MT], 0, 0, 0);
            between(part);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    // f(i) for items `part` of `parts` of N.
    auto share = [](auto n, auto part, auto parts, auto f) {
        each<n * (part + 1) / parts - n * part / parts>([&](auto i) { f(std::integral_constant<int, n * part / parts + i>()); });
    };
    constexpr std::integral_constant<int, kReads> reads;
    constexpr std::integral_constant<int, kLoads> loads;
    constexpr std::integral_constant<int, kParts> parts;
    auto advance = [&] { // behind the last block there is that block again, which nobody reads: loads are made, and counted, all the same
        if (ahead_block + 1 < ahead_end)
            ++ahead_block, w_now += block_bytes;
        else
            enter();
    };
    auto begin = [&](const ProductArgs& a) { // blocks of the products' tile
        int row, column, share;
        place8(a, now, row, column, share);
        left = min(a.per, (a.K + 127) / 128 - share * a.per);
    };
    enter();
    begin(args);
    for (int s = 0; s < S; ++s) {
        each<kLoads>([&](auto i) { stage(i, s); });
        advance();
    }
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((S - 1) * kLoads) : "memory");
    Operands first, second;
    for (int i = 0; i < kReads; ++i)
        fetch(first, i, 0, 0);
    clear();
    constexpr int kEarly = kParts > 2 ? kParts * 3 / 4 : kParts; // parts under which operands are read: the rest covers their latency
    constexpr std::integral_constant<int, kEarly> early;
    constexpr int kStores = MT / 4 * NT * (GATED ? 1 : 2);  // of a wave for a tile that is full
    constexpr int kAway   = (S - 2) * kLoads;               // a wave's loads of the blocks behind the next
    static_assert(kAway + kStores < 64);
    int place = 0, relaxed = 0; // relaxed: barriers ahead of which the last results' stores may still be under way
    for (;;) {
        multiply(first, [&](auto part) {
            if constexpr (part < kEarly)
                share(reads, part, early, [&](auto i) { fetch(second, i, place, 1); });
        });
        // The next block has come.  Loads and stores are counted in their order: behind it are kAway loads, and stores.
        if (relaxed > 0)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kAway + kStores) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kAway) : "memory");
        --relaxed;
        const int next = place + 1 == S ? 0 : place + 1;
        multiply(second, [&](auto part) {
            if constexpr (part < kEarly) // behind the last block bytes that nothing takes
                share(reads, part, early, [&](auto i) { fetch(first, i, next, 0); });
            share(loads, part, parts, [&](auto i) { stage(i, place); });
        });
        advance();
        place = next;
        --left;
        if (left == 0) {
            const ProductArgs a = late_args8();
            const Layout8     l = layout8(a.M, a.K, GATED);
            int               row, column, share;
            place8(a, now, row, column, share);
            const Ends& e = ends[turn % kEnds];
            if (a.part == nullptr) {
                constexpr int kEnd = 2;
                // A group's rows at a time, whose scales and biases are read once, and two columns of tiles: their steps hide each other's latency
                // (gated 24960x256, N = 4917 187 us one by one, 154 so).  For more there are not registers enough.
                each<MT / 4>([&](auto g) {
                    const int group = wm * (MT / 4) + g;
                    each<GATED ? 1 : 2>([&](auto h) {
                        const int j = GATED ? group * 32 + 8 * q : group * 64 + 16 * q + 8 * h;
                        asm volatile("" ::: "memory");
                        const Tail8<GATED, 8> tail(a, row * (GATED ? kM / 2 : kM) + j, e.sw + j, e.b + j, kM / 2);
                        each<NT / kEnd>([&](auto part) {
                            float y[8 * kEnd], sx[kEnd];
                            int   v[8];
                            auto  of = [&](auto first, auto u) { // eight sums, from row tile `first` of the group on
                                for (int i = 0; i < 8; ++i)
                                    v[i] = sum[g * 4 + first + i / 4][part * kEnd + u][i % 4];
                            };
                            each<kEnd>([&](auto u) {
                                sx[u] = e.sx[(wn * NT + part * kEnd + u) * 16 + c];
                                of(std::integral_constant<int, 2 * h>(), u);
                                tail.scale(y + 8 * u, v, sx[u]);
                            });
                            activate8<8 * kEnd>(y, a.act);
                            each<kEnd>([&](auto u) {
                                if constexpr (GATED) {
                                    of(std::integral_constant<int, 2>(), u);
                                    tail.times(y + 8 * u, v, sx[u]);
                                }
                                const int n = column * kN + (wn * NT + part * kEnd + u) * 16 + c;
                                if (n < a.N)
                                    tail.put(a, n, y + 8 * u);
                            });
                        });
                    });
                });
                // With all its stores made: of the barriers that wait for loads older than they are.
                relaxed = (row + 1) * (GATED ? kM / 2 : kM) <= a.M && (column + 1) * kN <= a.N ? S - 1 : 0;
            } else {
                const int columns = (a.N + 15) / 16;
                each<NT>([&](auto u) {
                    const int at = column * kCols + wn * NT + u;
                    each<MT / 4>([&](auto g) {
                        const int group = row * (kM / 64) + wm * (MT / 4) + g;
                        if (at < columns && group < l.groups)
                            each<4>([&](auto t) { part_of(a, l.groups, share, columns, group, at)[t * 64 + lane] = sum[g * 4 + t][u]; });
                    });
                });
            }
            now += apart, ++turn;
            if (now >= tiles)
                break;
            begin(a);
            clear();
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // the LDS that loads are on their way to is the workgroup's until they are there
}

// How a call runs.
struct Plan8 {
    int kind;        // 0: w8_narrow, otherwise a w8_tiles of kTiles[kind - 1]
    int rows, cols;  // row and column tiles of 16 that a workgroup of w8_narrow takes
    int shares, per; // shares of K, blocks of 128 columns in each
    bool x16;        // of w8_narrow: rows of 16 bits, which its workgroups round to 8 themselves
};

// What plan8 knows of the shapes of w8_tiles: a workgroup's row and column tiles, how many fit a CU, and in microseconds what a tile costs
// beside its blocks, a block with one workgroup on the CU and with two.
struct Tiles8 {
    int    rows, cols, resident;
    double tile, block, both;
};
constexpr Tiles8 kTiles[] = {{16, 16, 1, 2.7, 1.34, 0},    {8, 16, 1, 2.4, 0.78, 0},     {16, 8, 1, 2.3, 0.73, 0},
                             {8, 8, 1, 1.8, 0.46, 0},      {8, 8, 2, 1.5, 0.59, 0.84},   {8, 4, 2, 1.5, 0.365, 0.58}};
constexpr int kShapes = sizeof kTiles / sizeof *kTiles;

#ifdef SPMM_KEEP_VARIANTS
Plan8 g_plan8{};
#endif

int64_t up8(int64_t a, int64_t b) { return (a + b - 1) / b; }

void share8(Plan8& p, int64_t blocks, int64_t shares)
{
    p.per    = (int)up8(blocks, std::max<int64_t>(1, std::min(shares, blocks)));
    p.shares = (int)up8(blocks, p.per);
}

// The cheapest by a model of a call's time in microseconds, fitted to 2912 calls of 110 shapes, from 256x256 to 36864x9216 and from 1 to 6000
// columns, on which it is 2 % off the best on average and 32 % at worst (rows of an odd length with few columns of K).  Workgroups are
// counted in rounds, one (or two) for every CU; W's and Y's bytes are added to them; K in shares costs a launch and the shares'
// bytes.  Examples, us: 5120x5120, N = 37 10.2 narrow with two row and three column tiles, 12.9 in tiles of 128 x 64;
// 20480x5120, N = 64 25.6 in tiles of 128 x 64, 30.3 narrow; 9216x36864, N = 193 97 in tiles of 256 x 256 and seven shares of K,
// 113 in tiles of 128 x 256 and three, 410 in one.
Plan8 choose8(int M, int N, int K, bool gated)
{
    const Layout8 l      = layout8(M, K, gated);
    const int64_t blocks = l.steps / 2, tiles = (int64_t)l.groups * 4;
    const double  w_mb = (double)tiles * (double)blocks * 2048e-6, part_mb = (double)tiles * (double)up8(N, 16) * 2048e-6,
                  y_mb = (double)M * N * 2e-6;
    Plan8         p{}, best{};
    double        least = 1e300;
#ifdef SPMM_KEEP_VARIANTS // the tests' build: every kernel at small sizes
    if (g_plan8.shares > 0) {
        p = g_plan8;
        share8(p, blocks, g_plan8.shares);
        return p;
    }
#endif
    auto consider = [&](double us) {
        if (p.shares > 1)
            us += 3.2 + p.shares * part_mb / 7.8;
        if (us < least)
            least = us, best = p;
    };
    if (N <= 128)
        for (p.rows = gated ? 2 : 1; p.rows <= 4; p.rows *= 2)
            for (p.cols = 1; p.cols <= std::min<int64_t>(4, up8(N, 16)); ++p.cols) {
                const int64_t columns = up8(N, 16 * p.cols), groups = tiles / p.rows * columns;
                for (int s : {1, 2, 3, 4, 6, 8, 12, 16}) {
                    if (s > 1 && (s > blocks || groups * s > 2048))
                        break;
                    share8(p, blocks, s);
                    consider(2.8 + w_mb * (double)columns / 12.6 +
                             (double)(up8(groups * p.shares, 256) * up8(p.per, 8)) * (0.19 * p.rows + 0.24 * p.cols));
                }
            }
    for (p.kind = 1; p.kind <= kShapes; ++p.kind) {
        const Tiles8& k      = kTiles[p.kind - 1];
        const int64_t groups = up8(tiles, k.rows) * up8(N, 16 * k.cols);
        p.rows = p.cols = 0;
        for (int fill = 0; fill <= k.resident; ++fill) { // shares for none, one or two workgroups on every CU
            if (fill > 0 && 256 * fill / groups < 2)
                continue;
            share8(p, blocks, fill > 0 ? std::min<int64_t>(64, 256 * fill / groups) : 1);
            const int64_t slots = 256 * k.resident, full = groups * p.shares / slots, rest = groups * p.shares % slots;
            double        us = 4.3 + w_mb / 17.3 + y_mb / 3.4;
            us += (double)full * (k.tile + p.per * (k.resident > 1 ? k.both : k.block));
            if (rest > 0)
                us += k.tile + p.per * (rest > 256 ? k.both : k.block);
            consider(us);
        }
    }
    return best;
}

// 16-bit rows are rounded within w8_narrow where few are read beside few weights: a call then is one launch and needs no workspace, 6.8
// us of a Python caller's time instead of 10.7, which is what a call takes that is not recorded.  Every workgroup reads all the rows for
// itself, one row after another, so that a second round of workgroups does it once more: several rows only where all workgroups run
// at once, one row where there are two to a CU (65536x512, N = 8 28.4 us within, 10.8 with a kernel before it; 32768x1024, N = 4 12.8 and 10.6,
// N = 1 10.0 and 10.6).  By the kernels' time, as in a graph, within and not: 1024x1024, N = 1 4.1 and 5.4, N = 4 5.3 and 5.4, N = 8
// 7.3 and 5.7; 4096x2048, N = 4 6.4 and 5.7; 4096x8192, N = 1 10.3 and 8.4; gated 1024x4096, N = 2 10.3 and 7.9.  What a graph loses so, 2.4
// us at most of 121 sizes, is the price of the shorter call.  Not where K is in shares: w8_join, which ends their sums, reads the rows'
// scales from memory, and w8_narrow writes none.
constexpr int64_t kMost16 = 8192, kMostWeights16 = 1 << 25;

Plan8 plan8(int M, int N, int K, bool gated, bool x16)
{
    const Layout8 l = layout8(M, K, gated);
    Plan8         p = choose8(M, N, K, gated);
    p.x16 = x16 && p.kind == 0 && p.cols == 1 && p.shares == 1 && N <= kRows16 && (int64_t)N * K <= kMost16 && l.scales <= kMostWeights16 &&
            (int64_t)l.groups * 4 / p.rows <= (N == 1 ? 512 : 256);
    return p;
}

size_t part_bytes8(int M, int N, int K, bool gated, const Plan8& p)
{
    return p.shares > 1 ? (size_t)p.shares * up8(N, 16) * layout8(M, K, gated).groups * 4096 : 0;
}

template <bool GATED, int MT, int NT, int WM, int WN, int S>
int run_tiles8(hipStream_t stream, ProductArgs a, int resident)
{
    a.row_tiles         = (int)up8(layout8(a.M, a.K, GATED).groups * 4, MT * WM), a.column_tiles = (int)up8(a.N, NT * WN * 16);
    const int64_t tiles = (int64_t)a.row_tiles * a.column_tiles * a.shares;
    if (tiles > 0x3fffffff)
        return refuse("%lld tiles of outputs", (long long)tiles);
    return launch(w8_tiles<GATED, MT, NT, WM, WN, S>, dim3((unsigned)std::min<int64_t>(tiles, 256 * resident), 1, 1),
                  dim3(64 * WM * WN, 1, 1), stream, a);
}

template <bool GATED, int R, int NT, int D, bool X16 = false>
int run_narrow8(hipStream_t stream, const ProductArgs& a)
{
    const int     cols  = (int)up8(a.N, NT * 16);
    const int64_t units = (int64_t)layout8(a.M, a.K, GATED).groups * (4 / R) * cols;
    if (units > 0x7fffffff)
        return refuse("%lld tiles of outputs", (long long)units);
    return launch(w8_narrow<GATED, R, NT, D, X16>, dim3((unsigned)units, (unsigned)a.shares, 1), dim3(64 * kNarrowWaves, 1, 1), stream, a, cols);
}

template <bool GATED, int R>
int run_narrow8(hipStream_t stream, const Plan8& p, const ProductArgs& a)
{
    if (p.x16)
        return run_narrow8<GATED, R, 1, R == 4 ? 3 : 4, true>(stream, a);
    if (p.cols == 1)
        return run_narrow8<GATED, R, 1, R == 4 ? 3 : 4>(stream, a);
    if (p.cols == 2)
        return run_narrow8<GATED, R, 2, R == 4 ? 3 : 4>(stream, a);
    if (p.cols == 3)
        return run_narrow8<GATED, R, 3, 2>(stream, a);
    return run_narrow8<GATED, R, 4, 2>(stream, a);
}

template <bool GATED>
int run_plan8(hipStream_t stream, const Plan8& p, const ProductArgs& a)
{
    int e;
    switch (p.kind) {
    case 0:
        if constexpr (!GATED)
            if (p.rows == 1) {
                e = run_narrow8<false, 1>(stream, p, a);
                break;
            }
        e = p.rows == 2 ? run_narrow8<GATED, 2>(stream, p, a) : run_narrow8<GATED, 4>(stream, p, a);
        break;
    case 1: e = run_tiles8<GATED, 8, 4, 2, 4, 2>(stream, a, 1); break;
    case 2: e = run_tiles8<GATED, 4, 4, 2, 4, 3>(stream, a, 1); break;
    case 3: e = run_tiles8<GATED, 4, 4, 4, 2, 3>(stream, a, 1); break;
    case 4: e = run_tiles8<GATED, 4, 2, 2, 4, 4>(stream, a, 1); break;
    case 5: e = run_tiles8<GATED, 4, 4, 2, 2, 2>(stream, a, 2); break;
    default: e = run_tiles8<GATED, 4, 2, 2, 2, 3>(stream, a, 2); break;
    }
    if (e != 0 || a.shares == 1)
        return e;
    const int64_t waves = up8(a.N, 16) * layout8(a.M, a.K, GATED).groups * 2;
    return launch(w8_join<GATED>, dim3((unsigned)up8(waves, 4), 1, 1), dim3(256, 1, 1), stream, a);
}

int check_sizes8(int M, int K)
{
    if (M < 1 || M > kMaxRows8 || K < 1 || K > kMaxK8)
        return refuse("weights of %d rows (1 to 2^24) and %d columns (1 to %d)", M, K, kMaxK8);
    return 0;
}

// Bytes from row to row of codes that the library makes room for.  From 1 KB on an odd multiple of 128: the rows of a tile then lie on
// different channels (8192 columns in rows of 8192 bytes 220 us, of 8320 209; 20480x5120, N = 4096 345 and 336).
int64_t stride8(int K)
{
    return K < 1024 ? (K + 15) / 16 * 16 : ((K + 127) / 128 | 1) * 128;
}

// Workspace of a call: sums of the shares of K; of 16-bit rows codes, then scales.
struct Space8 {
    int64_t part, codes, stride, scales, bytes; // bytes of the sums, offsets
};

Space8 space8(int M, int N, int K, bool gated, bool x16, const Plan8& p)
{
    Space8 s{};
    s.part = s.codes = s.bytes = (int64_t)part_bytes8(M, N, K, gated, p);
    if (x16) {
        s.stride = stride8(K);
        s.scales = s.codes + s.stride * N;
        s.bytes  = s.scales + ((int64_t)N * 4 + 15) / 16 * 16;
    }
    return s;
}

int run_product(hipStream_t stream, const void* packed, const void* x, int64_t x_stride, const float* x_scales, void* Y, int M, int N,
                int K, const void* bias, const void* up_bias, int activation, void* workspace, size_t workspace_bytes, int dtype,
                bool gated)
{
    if (int e = check_sizes8(M, K))
        return e;
    if (N < 0 || N > kMaxN8)
        return refuse("%d rows of X (0 to %d)", N, kMaxN8);
    if (dtype != DECODE_FP16 && dtype != DECODE_BF16)
        return refuse("unknown element type %d", dtype);
    if (activation < 0 || activation > W8_ACT_SILU)
        return refuse("unknown activation %d (0 none, 1 ReLU, 2 GELU, 3 SiLU)", activation);
    if (N == 0)
        return 0;
    if (bad_pointer(packed, 16) || bad_pointer(Y, 2) || (bias != nullptr && bad_pointer(bias, 2)) ||
        (up_bias != nullptr && bad_pointer(up_bias, 2)))
        return refuse("a null or misaligned weight (16 bytes), Y or bias (2)");
    const bool   x16 = x_scales == nullptr;
    const Plan8  p   = plan8(M, N, K, gated, x16);
    const Space8 s   = space8(M, N, K, gated, x16 && !p.x16, p);
    if (x16 ? bad_pointer(x, 2) : bad_codes(x, x_stride, x_scales, N, K))
        return refuse("X null or misaligned (16-bit rows: 2 bytes; codes: 16, rows too, scales 4)");
    const size_t need = (size_t)s.bytes;
    if (need > 0 && (bad_pointer(workspace, 16) || workspace_bytes < need))
        return refuse("workspace of %zu bytes (16-byte aligned), %zu needed", workspace == nullptr ? (size_t)0 : workspace_bytes, need);
    ProductArgs a{};
    a.packed = static_cast<const uint8_t*>(packed);
    a.x = static_cast<const int8_t*>(x), a.x_scales = x_scales, a.x_stride = x_stride;
    if (x16 && !p.x16) {
        int8_t* codes  = static_cast<int8_t*>(workspace) + s.codes;
        float*  scales = reinterpret_cast<float*>(static_cast<int8_t*>(workspace) + s.scales);
        if (int e = run_quantize(stream, x, x_stride, N, K, codes, s.stride, scales, dtype))
            return e;
        a.x = codes, a.x_scales = scales, a.x_stride = s.stride;
    }
    a.y = static_cast<uint16_t*>(Y), a.bias = static_cast<const uint16_t*>(bias), a.up_bias = static_cast<const uint16_t*>(up_bias);
    a.M = M, a.N = N, a.K = K, a.act = activation, a.bf16 = dtype == DECODE_BF16;
    a.shares = p.shares, a.per = p.per, a.part = p.shares > 1 ? static_cast<int*>(workspace) : nullptr;
    return gated ? run_plan8<true>(stream, p, a) : run_plan8<false>(stream, p, a);
}

} // namespace
} // namespace decode

using namespace decode;

#ifdef SPMM_KEEP_VARIANTS
// Every later call runs as the plan says (see Plan8); shares 0: as the library chooses.
extern "C" int W8_Debug_SetPlan(int kind, int rows, int cols, int shares)
{
    if (kind < 0 || kind > kShapes || shares < 0 ||
        (kind == 0 && shares > 0 && ((rows != 1 && rows != 2 && rows != 4) || cols < 1 || cols > 4)))
        return 1;
    g_plan8 = Plan8{kind, rows, cols, shares, 0, false};
    return 0;
}
#endif

extern "C" size_t W8_PackedBytes(int M, int K, int gated)
{
    if (M < 1 || M > kMaxRows8 || K < 1 || K > kMaxK8)
        return 0;
    return (size_t)layout8(M, K, gated != 0).bytes;
}

extern "C" int W8_Pack(hipStream_t stream, const int8_t* codes, int64_t stride, const float* scales, const int8_t* up_codes,
                       int64_t up_stride, const float* up_scales, int M, int K, void* packed)
{
    if (int e = check_sizes8(M, K))
        return e;
    const bool gated = up_codes != nullptr;
    if (codes == nullptr || bad_pointer(scales, 4) || (gated && bad_pointer(up_scales, 4)) || bad_pointer(packed, 16) ||
        (M > 1 && (stride < K || (gated && up_stride < K))))
        return refuse("null or misaligned codes, scales (4 bytes) or packed weights (16), or rows less than %d codes apart", K);
    PackArgs a{};
    a.w = codes, a.scales = scales, a.w_stride = stride;
    a.up = up_codes, a.up_scales = up_scales, a.up_stride = up_stride;
    a.M = M, a.K = K, a.packed = static_cast<uint8_t*>(packed);
    const Layout8 l = layout8(M, K, gated);
    return launch(w8_pack, dim3((unsigned)(l.groups * (l.steps / 2)), 1, 1), dim3(256, 1, 1), stream, a);
}

extern "C" size_t W8_WorkspaceBytes(int M, int N, int K, int gated, int x16)
{
    if (W8_PackedBytes(M, K, gated) == 0 || N < 1 || N > kMaxN8)
        return 0;
    const Plan8 p = plan8(M, N, K, gated != 0, x16 != 0);
    return (size_t)space8(M, N, K, gated != 0, x16 != 0 && !p.x16, p).bytes;
}

extern "C" int W8_Linear(hipStream_t stream, const void* packed, const void* x, int64_t x_stride, const float* x_scales, void* Y, int M,
                         int N, int K, const void* bias, int activation, void* workspace, size_t workspace_bytes, int dtype)
{
    return run_product(stream, packed, x, x_stride, x_scales, Y, M, N, K, bias, nullptr, activation, workspace, workspace_bytes, dtype,
                       false);
}

extern "C" int W8_Gated(hipStream_t stream, const void* packed, const void* x, int64_t x_stride, const float* x_scales, void* Y, int M,
                        int N, int K, const void* gate_bias, const void* up_bias, int activation, void* workspace,
                        size_t workspace_bytes, int dtype)
{
    return run_product(stream, packed, x, x_stride, x_scales, Y, M, N, K, gate_bias, up_bias, activation, workspace, workspace_bytes,
                       dtype, true);
}
