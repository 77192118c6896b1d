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
// K is filled up with zeros to a multiple of 128: what X has there does not matter.
#include "w8_common.hiph"

#include <algorithm>
#include <type_traits>

namespace decode {
namespace {

constexpr int kMaxRows8 = 1 << 24;

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

// One wave lays out one block of 16 rows x 64 columns.
__global__ __launch_bounds__(64) void w8_pack(PackArgs a)
{
    const bool    gated = a.up != nullptr;
    const Layout8 l     = layout8(a.M, a.K, gated);
    const int     lane = threadIdx.x, r = lane & 15, q = lane >> 4, tile = blockIdx.x & 3;
    const int64_t block = blockIdx.x;
    const int     group = (int)(block / 4 % l.groups), step = (int)(block / 4 / l.groups);
    const bool    second = gated && tile >= 2;
    const int     row = gated ? group * 32 + (r >> 2) * 8 + (tile & 1) * 4 + (r & 3) : group * 64 + (r >> 2) * 16 + tile * 4 + (r & 3);
    const int8_t* src = second ? a.up + row * a.up_stride : a.w + row * a.w_stride;
    uintx4        out = 0;
    for (int b = 0; b < 16; ++b) {
        const int k = step * 64 + q * 16 + b;
        if (row < a.M && k < a.K)
            out[b / 4] |= (unsigned)(uint8_t)src[k] << (8 * (b % 4));
    }
    reinterpret_cast<uintx4*>(a.packed)[(((int64_t)group * 4 + tile) * l.steps + step) * 64 + lane] = out;
    if (step == 0 && tile == 0) { // 64 scales: of the group's rows, or of 32 rows of the gate and of up
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
    int            M, N, K, act;
};

// ReLU, GELU (tanh form) or SiLU of eight sums.  The last two are y / (1 + exp(-z)), with z = 2 sqrt(2/pi) (y + 0.044715 y^3), since
// (1 + tanh u) / 2 = 1 / (1 + exp(-2 u)), or z = y; far from 0 they end at 0 and y.  The reciprocal's last bit is far below 16 bits.
__device__ __forceinline__ void activate8(float* y, int act)
{
    if (act == 1) {
        for (int i = 0; i < 8; ++i)
            y[i] = y[i] < 0.f ? 0.f : y[i]; // a NaN stays one
    } else if (act > 1) {
        const float cube = act == 2 ? 1.5957691216057308f * 0.044715f : 0.f, one = act == 2 ? 1.5957691216057308f : 1.f;
        for (int i = 0; i < 8; ++i) {
            const float z = y[i] * (one + cube * y[i] * y[i]);
            y[i]          = y[i] * __builtin_amdgcn_rcpf(1.f + __expf(-z));
        }
    }
}

// Eight 16-bit numbers from p on, of which `left` are there.
__device__ __forceinline__ shortx8 bias8(const uint16_t* p, int left)
{
    if (left >= 8)
        return *reinterpret_cast<const loose8*>(p);
    shortx8 v = 0;
    for (int i = 0; i < 7; ++i)
        if (i < left)
            v[i] = p[i];
    return v;
}

// What the outputs of eight consecutive rows from `m` on have in common over the columns.
template <bool BF16, bool GATED>
struct Tail8 {
    float sw[8], su[8], b[8], bu[8];
    int   m, left;

    __device__ __forceinline__ Tail8(const ProductArgs& a, const Layout8& l, int row) : m(row), left(a.M - row)
    {
        if (left <= 0)
            return;
        const float*  s  = reinterpret_cast<const float*>(a.packed + l.scales) + m; // the layout's rows go past M
        const shortx8 v  = a.bias != nullptr ? bias8(a.bias + m, left) : (shortx8)0;
        const shortx8 vu = GATED && a.up_bias != nullptr ? bias8(a.up_bias + m, left) : (shortx8)0;
        for (int i = 0; i < 8; ++i) {
            sw[i] = s[i], b[i] = from16(v[i], BF16);
            if (GATED)
                su[i] = s[i + (int64_t)l.groups * 32], bu[i] = from16(vu[i], BF16);
        }
    }

    // From LDS: scales, and biases as 32-bit words of 16 bits; those of up `up` words behind the gate's.
    __device__ __forceinline__ Tail8(const ProductArgs& a, int row, const float* s, const unsigned* bias, int up) : m(row), left(a.M - row)
    {
        for (int i = 0; i < 8; ++i) {
            sw[i] = s[i], b[i] = a.bias != nullptr ? from16((uint16_t)bias[i], BF16) : 0.f;
            if (GATED)
                su[i] = s[up + i], bu[i] = a.up_bias != nullptr ? from16((uint16_t)bias[up + i], BF16) : 0.f;
        }
    }

    // The end of the sums of column n, of its row of X the scale sx; `up` is read by gated products only.
    __device__ __forceinline__ void store(const ProductArgs& a, int n, float sx, const int* sum, const int* up) const
    {
        if (left <= 0)
            return;
        float y[8];
        for (int i = 0; i < 8; ++i)
            y[i] = (float)sum[i] * sw[i] * sx + b[i];
        activate8(y, a.act);
        if constexpr (GATED)
            for (int i = 0; i < 8; ++i)
                y[i] *= (float)up[i] * su[i] * sx + bu[i];
        shortx8 out;
        for (int i = 0; i < 8; ++i)
            out[i] = BF16 ? __builtin_bit_cast(uint16_t, (__bf16)y[i]) : __builtin_bit_cast(uint16_t, (_Float16)y[i]);
        uint16_t* to = a.y + (int64_t)n * a.M + m;
        if (left >= 8) {
            *reinterpret_cast<loose8*>(to) = out;
            return;
        }
        for (int i = 0; i < 7; ++i)
            if (i < left)
                to[i] = out[i];
    }
};

// Row of its group that a lane's outputs begin at: 16 of them, or 8 of a gated product.
template <bool GATED>
__device__ __forceinline__ int first_row8(int group, int q)
{
    return GATED ? group * 32 + 8 * q : group * 64 + 16 * q;
}

// A workgroup takes one group of 64 packed rows and 16 columns of X; its four waves take every fourth step of K and meet in LDS.
template <bool BF16, bool GATED>
__global__ __launch_bounds__(256) void w8_product(ProductArgs a)
{
    __shared__ intx4 part[4][4][64];
    const Layout8    l    = layout8(a.M, a.K, GATED);
    const int        lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int        group = blockIdx.x, n = blockIdx.y * 16 + (lane & 15), q = lane >> 4;
    const int8_t*    x     = a.x + (int64_t)min(n, a.N - 1) * a.x_stride;
    const int        last  = (a.K - 1) / 16; // the last 16 columns that X has; behind them the weights are 0
    const intx4*     w     = reinterpret_cast<const intx4*>(a.packed) + (int64_t)group * 4 * l.steps * 64 + lane;
    intx4            sum[4] = {0, 0, 0, 0};
    for (int s = wave; s < l.steps; s += 4) {
        const intx4 b = *reinterpret_cast<const intx4*>(x + 16 * min(4 * s + q, last));
        for (int t = 0; t < 4; ++t)
            sum[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[((int64_t)t * l.steps + s) * 64], b, sum[t], 0, 0, 0);
    }
    for (int t = 0; t < 4; ++t)
        part[wave][t][lane] = sum[t];
    __syncthreads();
    if (wave > 0 || n >= a.N)
        return;
    for (int t = 0; t < 4; ++t)
        for (int w = 1; w < 4; ++w)
            sum[t] += part[w][t][lane];
    int v[16];
    for (int i = 0; i < 16; ++i)
        v[i] = sum[i / 4][i % 4];
    const float sx = a.x_scales[n];
    const int   m  = first_row8<GATED>(group, q);
    Tail8<BF16, GATED>(a, l, m).store(a, n, sx, v, v + 8);
    if constexpr (!GATED)
        Tail8<BF16, false>(a, l, m + 8).store(a, n, sx, v + 8, nullptr);
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
// ahead of the next read of LDS; the kernel waits for it itself, before the barrier that hands the tile over.
__device__ __forceinline__ void to_lds(unsigned lds, const void* base, unsigned offset)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}

// The same of one word, or of 16 bits in a word, a lane.
__device__ __forceinline__ void word_to_lds(unsigned lds, const void* address)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(address) : "memory");
}

__device__ __forceinline__ void short_to_lds(unsigned lds, const void* address)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ushort %1, off" ::"s"(lds), "v"(address) : "memory");
}

// Workgroups are dealt to the eight dies in turn, each with an L2 of its own: consecutive numbers on one die, and there a band of
// kBand row tiles by as many column tiles as run at once.
__device__ __forceinline__ void place8(int id, int row_tiles, int column_tiles, int& row, int& column)
{
    constexpr int kBand = 8;
    const int     total = row_tiles * column_tiles, xcd = id % 8, rest = total % 8;
    const int     at   = xcd * (total / 8) + min(xcd, rest) + id / 8;
    const int     band = at / (kBand * column_tiles), first = band * kBand, height = min(kBand, row_tiles - first);
    const int     in   = at - first * column_tiles;
    // divisions are done by vector instructions: back to scalars, which the addresses are made of
    row = __builtin_amdgcn_readfirstlane(first + in % height), column = __builtin_amdgcn_readfirstlane(in / height);
}

// A workgroup of WM x WN waves takes WM MT x WN NT tiles of 16 x 16 outputs (packed rows x rows of X), a wave MT x NT of them.  K goes by in
// blocks of 128 through two buffers in LDS: W's blocks lie there as they are packed, one operand a KB; of X 8 rows lie in a KB,
// row r's chunk c of 16 bytes at place 8 r + (c ^ r), which the matrix operands' reads find without bank conflicts.
// While the products of a block's first half run, the second half's operands are read; then the waves meet, the buffer that
// all have read takes the block after next, and the next block's first operands are read under the second half's products.
// A workgroup stays on its CU and takes every gridDim-th tile: the blocks of all its tiles are one stream, so that the next tile is
// loaded while the results of the last are written, and a tile costs its products alone.
template <bool BF16, bool GATED, int MT, int NT, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void w8_tiles(ProductArgs a, int row_tiles, int column_tiles)
{
    constexpr int kWaves = WM * WN, kRows = WM * MT, kCols = WN * NT * 2, kStage = (2 * kRows + kCols) * 1024; // tiles of W, KBs of X
    constexpr int kLoads = (2 * kRows + kCols) / kWaves, kWLoads = 2 * kRows / kWaves;
    constexpr int kM = kRows * 16, kN = WN * NT * 16; // packed rows, rows of X
    static_assert(2 * kRows % kWaves == 0 && kCols % kWaves == 0 && MT % 4 == 0 && kM % 64 == 0 && kN % 64 == 0);
    struct Ends { // of a tile: scales and biases of its rows (of the gate, then of up), scales of its rows of X
        float    sw[kM];
        unsigned b[kM];
        float    sx[kN];
    };
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2][kStage];
    __shared__ __attribute__((aligned(16))) Ends      ends[4]; // loads are at most two tiles ahead of the products
    const Layout8 l    = layout8(a.M, a.K, GATED);
    const int     lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int     q = lane >> 4, c = lane & 15, wm = wave / WN, wn = wave % WN, blocks = l.steps / 2;
    const int     tiles = row_tiles * column_tiles;

    // What a wave brings of every block: KBs of W first, then of X.
    const uint8_t* w_at[kWLoads];
    const int8_t*  x_at[kLoads - kWLoads];
    unsigned       x_row[kLoads - kWLoads];
    auto address = [](const void* p) { return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void*)p; };
    const unsigned lds0 = address(lds), ends0 = address(ends);
    const int      chunk = 16 * ((lane & 7) ^ (lane >> 3)), last = (a.K - 1) / 16 * 16;
    // Turns the loads to a tile, the `turn`-th, and brings its ends.
    auto enter = [&](int tile, int turn) {
        int row, column;
        place8(tile, row_tiles, column_tiles, row, column);
        const int tile0 = row * kRows, n0 = column * kN;
        for (int i = 0; i < kWLoads; ++i) { // tiles behind the last are the last again: computed, not stored
            const int j = wave * kWLoads + i;
            w_at[i]     = a.packed + ((int64_t)min(tile0 + j / 2, l.groups * 4 - 1) * l.steps + j % 2) * 1024;
        }
        for (int i = 0; i < kLoads - kWLoads; ++i) {
            const int j = wave * (kLoads - kWLoads) + i;
            const int n = min(n0 + 8 * j, a.N - 1); // rows behind the last are the last again
            x_at[i]     = a.x + (int64_t)n * a.x_stride;
            x_row[i]    = min(lane >> 3, a.N - 1 - n) * (unsigned)a.x_stride;
        }
        const unsigned to = ends0 + (turn & 3) * sizeof(Ends);
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
    auto stage = [&](int i, int block, int buffer) {
        const unsigned to = lds0 + buffer * kStage;
        if (i < kWLoads)
            to_lds(to + (wave * kWLoads + i) * 1024, w_at[i] + (int64_t)block * 2048, lane * 16);
        else
            to_lds(to + (2 * kRows + wave * (kLoads - kWLoads) + i - kWLoads) * 1024,
                   x_at[i - kWLoads], x_row[i - kWLoads] + min(block * 128 + chunk, last));
    };
    struct Operands {
        intx4 w[MT], x[NT];
    };
    constexpr int kReads = MT + NT, kProducts = MT * NT;
    auto fetch = [&](Operands& o, int i, int buffer, int half) {
        const uint8_t* from = lds[buffer];
        if (i < MT)
            o.w[i] = *reinterpret_cast<const intx4*>(from + ((wm * MT + i) * 2 + half) * 1024 + lane * 16);
        else
            o.x[i - MT] = *reinterpret_cast<const intx4*>(from + (2 * kRows + (wn * NT + i - MT) * 2 + (c >> 3)) * 1024 +
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
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
#pragma unroll
            for (int f = 4 * part; f < 4 * part + 4; ++f)
                sum[f % MT][f / MT] = __builtin_amdgcn_mfma_i32_16x16x64_i8(o.w[f % MT], o.x[f / MT], sum[f % MT][f / MT], 0, 0, 0);
            between(part);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Items `part` of `parts` of n, as a range.
#define W8_SHARE(i, n, part, parts) for (int i = (n) * (part) / (parts); i < (n) * ((part) + 1) / (parts); ++i)
    Operands first, second;
    // Tile and block of the next load, and how many tiles it has seen; tile, block and number of the next products.
    int ahead_tile = blockIdx.x, ahead_block = 0, ahead_turn = 0, tile = blockIdx.x, block = 0, turn = 0;
    auto advance = [&] {
        if (++ahead_block == blocks) {
            ahead_block = 0, ahead_tile += gridDim.x, ++ahead_turn;
            if (ahead_tile < tiles)
                enter(ahead_tile, ahead_turn);
        }
    };
    enter(tile, 0);
    for (int s = 0; s < 2; ++s) {
        if (ahead_tile < tiles)
            for (int i = 0; i < kLoads; ++i)
                stage(i, ahead_block, s);
        advance();
    }
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    for (int i = 0; i < kReads; ++i)
        fetch(first, i, 0, 0);
    clear();
    constexpr int kEarly  = kParts * 3 / 4;                      // parts under which operands are read: the rest covers their latency
    constexpr int kStores = MT / 4 * NT * (GATED ? 1 : 2);       // of a wave for a tile that is full
    bool          relaxed = false;                               // the last results' stores may still be under way
    for (int buffer = 0;; buffer ^= 1) {
        const bool more = ahead_tile < tiles;
        multiply(first, [&](int part) {
            if (part < kEarly)
                W8_SHARE(j, kReads, part, kEarly)
                    fetch(second, j, buffer, 1);
        });
        // The next block has come: its loads are older than the stores, which are counted with them.
        if (relaxed)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kStores) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        relaxed = false;
        multiply(second, [&](int part) {
            if (part < kEarly)
                W8_SHARE(j, kReads, part, kEarly) // behind the last block stale bytes, which nothing takes
                    fetch(first, j, buffer ^ 1, 0);
            if (more)
                W8_SHARE(j, kLoads, part, kParts)
                    stage(j, ahead_block, buffer);
        });
        if (++block == blocks) {
            int row, column;
            place8(tile, row_tiles, column_tiles, row, column);
            const Ends& e = ends[turn & 3];
            each<MT / 4>([&](auto g) {
                const int group = wm * (MT / 4) + g;
                each<GATED ? 1 : 2>([&](auto h) {
                    const int                j = GATED ? group * 32 + 8 * q : group * 64 + 16 * q + 8 * h;
                    const Tail8<BF16, GATED> tail(a, row * (GATED ? kM / 2 : kM) + j, e.sw + j, e.b + j, kM / 2);
                    each<NT>([&](auto u) {
                        const int n = column * kN + (wn * NT + u) * 16 + c;
                        if (n >= a.N)
                            return;
                        int v[16];
                        for (int i = 0; i < 16; ++i)
                            v[i] = sum[g * 4 + i / 4][u][i % 4];
                        tail.store(a, n, e.sx[(wn * NT + u) * 16 + c], v + 8 * h, v + 8);
                    });
                });
            });
            // With all its stores made, and blocks enough that the loads of a tile's ends are waited for by another barrier.
            relaxed = (row + 1) * (GATED ? kM / 2 : kM) <= a.M && (column + 1) * kN <= a.N && blocks > 2;
            block = 0, tile += gridDim.x, ++turn;
            if (tile >= tiles)
                return;
            clear();
        }
        advance();
    }
#undef W8_SHARE
}

template <bool BF16, bool GATED>
int run_product(hipStream_t stream, const ProductArgs& a)
{
    const Layout8 l = layout8(a.M, a.K, GATED);
    if (a.N > 64) {
        const int rows = (l.groups * 4 + 15) / 16, cols = (a.N + 255) / 256;
        return launch(w8_tiles<BF16, GATED, 8, 4, 2, 4>, dim3((unsigned)std::min(rows * cols, 256), 1, 1), dim3(512, 1, 1),
                      stream, a, rows, cols);
    }
    return launch(w8_product<BF16, GATED>, dim3((unsigned)l.groups, (unsigned)(a.N + 15) / 16, 1), dim3(256, 1, 1), stream, a);
}

int check_sizes8(int M, int K)
{
    if (M < 1 || M > kMaxRows8 || K < 1 || K > kMaxK8)
        return refuse("weights of %d rows (1 to 2^24) and %d columns (1 to %d)", M, K, kMaxK8);
    return 0;
}

// Workspace of a call on 16-bit rows: codes, then scales.
struct Space8 {
    int64_t stride, scales, bytes;
};

Space8 space8(int N, int K, bool x16)
{
    Space8 s{};
    if (x16) {
        s.stride = (K + 15) / 16 * 16;
        s.scales = s.stride * N;
        s.bytes  = s.scales + ((int64_t)N * 4 + 15) / 16 * 16;
    }
    return s;
}

int run_product(hipStream_t stream, const void* packed, const W8_Codes& x, void* Y, int M, int N, int K, const void* bias,
                const void* up_bias, int activation, void* workspace, size_t workspace_bytes, int dtype, bool gated)
{
    if (int e = check_sizes8(M, K))
        return e;
    if (N < 0 || N > 16 * 65535)
        return refuse("%d rows of X (0 to %d)", N, 16 * 65535);
    if (dtype != DECODE_FP16 && dtype != DECODE_BF16)
        return refuse("unknown element type %d", dtype);
    if (activation < 0 || activation > W8_ACT_SILU)
        return refuse("unknown activation %d (0 none, 1 ReLU, 2 GELU, 3 SiLU)", activation);
    if (N == 0)
        return 0;
    if (bad_pointer(packed, 16) || bad_pointer(Y, 2) || (bias != nullptr && bad_pointer(bias, 2)) ||
        (up_bias != nullptr && bad_pointer(up_bias, 2)))
        return refuse("a null or misaligned weight (16 bytes), Y or bias (2)");
    const bool   x16 = x.scales == nullptr;
    const Space8 s   = space8(N, K, x16);
    if (x16 ? bad_pointer(x.codes, 2) : bad_codes(x, N, K) || bad_pointer(x.scales, 4))
        return refuse("X null or misaligned (16-bit rows: 2 bytes; codes: 16, rows too, scales 4)");
    const size_t need = (size_t)s.bytes;
    if (need > 0 && (bad_pointer(workspace, 16) || workspace_bytes < need))
        return refuse("workspace of %zu bytes (16-byte aligned), %zu needed", workspace == nullptr ? (size_t)0 : workspace_bytes, need);
    ProductArgs a{};
    a.packed = static_cast<const uint8_t*>(packed);
    a.x = x.codes, a.x_scales = x.scales, a.x_stride = x.stride;
    if (x16) {
        int8_t* codes  = static_cast<int8_t*>(workspace);
        float*  scales = reinterpret_cast<float*>(codes + s.scales);
        if (int e = run_quantize(stream, x.codes, x.stride, N, K, codes, s.stride, scales, dtype))
            return e;
        a.x = codes, a.x_scales = scales, a.x_stride = s.stride;
    }
    a.y = static_cast<uint16_t*>(Y), a.bias = static_cast<const uint16_t*>(bias), a.up_bias = static_cast<const uint16_t*>(up_bias);
    a.M = M, a.N = N, a.K = K, a.act = activation;
    if (gated)
        return dtype == DECODE_BF16 ? run_product<true, true>(stream, a) : run_product<false, true>(stream, a);
    return dtype == DECODE_BF16 ? run_product<true, false>(stream, a) : run_product<false, false>(stream, a);
}

} // namespace
} // namespace decode

using namespace decode;

extern "C" size_t W8_PackedBytes(int M, int K, int gated)
{
    if (M < 1 || M > kMaxRows8 || K < 1 || K > kMaxK8)
        return 0;
    return (size_t)layout8(M, K, gated != 0).bytes;
}

extern "C" int W8_Pack(hipStream_t stream, W8_Weights w, const W8_Weights* up, int M, int K, void* packed)
{
    if (int e = check_sizes8(M, K))
        return e;
    if (w.codes == nullptr || bad_pointer(w.scales, 4) || (up != nullptr && (up->codes == nullptr || bad_pointer(up->scales, 4))) ||
        bad_pointer(packed, 16) || (M > 1 && (w.w_stride < K || (up != nullptr && up->w_stride < K))))
        return refuse("null or misaligned codes, scales (4 bytes) or packed weights (16), or rows less than %d codes apart", K);
    PackArgs a{};
    a.w = w.codes, a.scales = w.scales, a.w_stride = w.w_stride;
    if (up != nullptr)
        a.up = up->codes, a.up_scales = up->scales, a.up_stride = up->w_stride;
    a.M = M, a.K = K, a.packed = static_cast<uint8_t*>(packed);
    const Layout8 l      = layout8(M, K, up != nullptr);
    const int64_t blocks = (int64_t)l.groups * l.steps * 4;
    if (blocks > 0x7fffffff)
        return refuse("weights of %d rows and %d columns: more than 2^31 blocks", M, K);
    return launch(w8_pack, dim3((unsigned)blocks, 1, 1), dim3(64, 1, 1), stream, a);
}

extern "C" size_t W8_WorkspaceBytes(int M, int N, int K, int gated, int x16)
{
    if (W8_PackedBytes(M, K, gated) == 0 || N < 1)
        return 0;
    return (size_t)space8(N, K, x16 != 0).bytes;
}

extern "C" int W8_Linear(hipStream_t stream, const void* packed, W8_Codes x, void* Y, int M, int N, int K, const void* bias,
                         int activation, void* workspace, size_t workspace_bytes, int dtype)
{
    return run_product(stream, packed, x, Y, M, N, K, bias, nullptr, activation, workspace, workspace_bytes, dtype, false);
}

extern "C" int W8_Gated(hipStream_t stream, const void* packed, W8_Codes x, void* Y, int M, int N, int K, const void* gate_bias,
                        const void* up_bias, int activation, void* workspace, size_t workspace_bytes, int dtype)
{
    return run_product(stream, packed, x, Y, M, N, K, gate_bias, up_bias, activation, workspace, workspace_bytes, dtype, true);
}
