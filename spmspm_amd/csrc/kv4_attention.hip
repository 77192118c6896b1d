// Attention over the paged 4-bit key/value cache: KV4_Attention (decode_api.h holds the format).
//
// Mathematics.  With a key's scale s and zero point z and the integer codes k,
//   q.K = s * (sum_d q_d k_d - z * sum_d q_d):
// the matrix cores multiply the codes themselves.  A code masked out of its dword in place is as an fp16 number the subnormal
// k * 2^-24 (k * 2^-20 for the second nibble of a half, whose q is 1/16 of the other's), which v_mfma_f32_16x16x32_f16
// multiplies as it is: one AND per two codes and a shift per four.  Its sums lose a few bits to that (it aligns by exponent
// fields): scores of a few units were measured within 1.7e-5 of float64 (fp16; bf16 8e-6), where kv4_attention_rows, whose operands
// are normal numbers, is within 9e-7.  The probabilities' rounding to fp16 is 2.4e-4.
// For the values v - z goes into the product, an exact small integer in fp16: the code is put into the mantissa of 1024 (of
// 64, where it is the second nibble) and 1024 + z (64 + z) is taken off, two codes at a time.  Their scale goes into the
// probabilities, p'_t = p_t s_t.  p' must fit fp16 whatever the scales are, so their exponents go into the softmax: with
// s_t = f_t 2^e_t, f_t in [1/2, 1), the running reference m follows the maximum of x_t = log2(p_t) + e_t, p'_t = 2^(x_t - m) f_t, and
// the sum of probabilities is the sum of 2^(x_t - m) 2^-e_t.
//
// Layout.  One wave works on 32 keys at a time and RT tiles of 16 query rows (the heads that share a key/value head, for
// each new token).  Scores are computed transposed, S^T = K Q^T, so that a lane owns one query row (its column) and keys
// 8h..8h+7 of the 32 (h = lane / 16): these are exactly the k indices that it has to supply for O^T = V^T P^T, so
// probabilities go from one product to the next in registers, and maxima, sums and rescaling need no exchange but the
// one between the four lanes of a row, only when the maximum rises by more than 2^8.  V^T is built from rows of V: a lane
// loads 4 bytes of each of its 8 keys and pairs their halves (v_perm); LDS is not used until the waves' results are joined.
//
// Bounds.  Few rows: memory.  32 sequences of up to 16384 keys, 64 heads over 8, D = 128: 103 us, 4.6 TB/s (a large copy moves
// 4.9); 16 of up to 2048 keys, 40 heads of their own: 36.3 us, 3.6 TB/s, the longest of one round of workgroups; 131071 keys of
// one sequence, 32 heads over 8: 32 us and 5.5 for the join.
#include "decode_common.hiph"

#include <algorithm>

namespace decode {

constexpr int   kTile   = 32;    // keys per step of a wave
constexpr int   kWaves  = 4;     // waves of a workgroup, each with every fourth tile of the workgroup's keys
constexpr float kNone   = -3.402823466e38f; // m before any key: no score is below it
// The reference m of the exponentials starts 7 below the first maximum and follows when a score passes it by more than 15:
// p' stays below 2^15 and uses fp16's range down to 2^-32 of the largest.
constexpr float kBelow = 7.f, kSlack = 15.f;

struct AttentionArgs {
    const uint8_t * k_codes, *v_codes;
    const int32_t * k_words, *v_words;
    const int *     table, *lens, *cu;
    const uint16_t* q;
    int64_t         q_token, q_head;
    uint16_t*       out;
    float*          lse;
    float*          part_o; // [split][row][D], row = token * q_heads + head
    float*          part_ml; // [split][row][2]
    float           scale_log2;
    int             num_pages, page_log2, kv_heads, q_heads, share, batch, width, stride, tokens, window, splits, bf16;
};

template <int D>
struct Shape {
    static constexpr int kSteps  = D / 32;              // MFMA steps of a score
    static constexpr int kDwords = D / 32;              // dwords of key codes per lane: D/4 elements of one key
    static constexpr int kVal    = D == 96 ? 8 : D / 16; // value elements of one key per lane (96: lanes 12..15 have none)
    static constexpr int kValBytes = kVal / 2;
    static constexpr int waves(int rt) { return D == 256 || rt == 2 ? 2 : 3; } // waves per SIMD
};

template <int D>
struct Keys {
    unsigned k[2][Shape<D>::kDwords]; // key codes of the two 16-key tiles
    unsigned v[8][(Shape<D>::kValBytes + 3) / 4];
    uintx4   kw[2], vw[2];            // words of keys 8h .. 8h+7
};

// Codes that one workgroup reads once go past the caches (measured: 3 to 6 % less time, 24 to 96 sequences of 4k to 16k keys);
// ONCE is false where other blocks of rows read them again, as the average sequence has more than one: 4 x 128 tokens over 16384
// keys, 32 heads of 256 over 4, 504 us past the caches and 468 through them; 32 x 12 tokens over 8192, 32 heads of 128 over 8, 133 and 128.
template <bool ONCE, typename T>
__device__ __forceinline__ T load_as(const uint8_t* p)
{
    return ONCE ? __builtin_nontemporal_load(reinterpret_cast<const T*>(p)) : *reinterpret_cast<const T*>(p);
}

template <bool ONCE, int N>
__device__ __forceinline__ void load_dwords(unsigned (&dst)[N], const uint8_t* p)
{
    if constexpr (N == 2) {
        const uintx2 t = load_as<ONCE, uintx2>(p);
        dst[0] = t[0], dst[1] = t[1];
    } else if constexpr (N == 3) {
        __builtin_memcpy(dst, __builtin_assume_aligned(p, 4), 12);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uintx4 t = load_as<ONCE, uintx4>(p + 4 * i);
            dst[i] = t[0], dst[i + 1] = t[1], dst[i + 2] = t[2], dst[i + 3] = t[3];
        }
    }
}

// The entry of the block table for key `pos` of the sequence, and the page that it names, or -1.
__device__ __forceinline__ int entry_at(const AttentionArgs& a, const int* row, int pos)
{
    return uniform_load(row + min(pos >> a.page_log2, a.width - 1));
}
__device__ __forceinline__ int page_of(const AttentionArgs& a, int entry, int pos)
{
    return pos >> a.page_log2 < a.width && entry >= 0 && entry < a.num_pages ? entry : -1;
}

// Loads of the 32 keys from `tile` on (a multiple of 32); p0 and p1 are the pages of its two halves of 16.
template <int D, bool ONCE>
__device__ __forceinline__ void load_keys(Keys<D>& t, const AttentionArgs& a, int head, int tile, int p0, int p1, int c, int h)
{
    const int P = 1 << a.page_log2;
    // key r of tile T is key 8 (r / 4) + 4 T + r % 4 of the 32: half 0 for r < 8
    const int      kr  = 8 * (c >> 2) + (c & 3);
    const int      kp  = max(c < 8 ? p0 : p1, 0);
    const int64_t  kat = (((int64_t)kp * a.kv_heads + head) << a.page_log2) + ((tile + kr) & (P - 1));
    const uint8_t* kc  = a.k_codes + kat * (D / 2) + h * (D / 8);
    load_dwords<ONCE>(t.k[0], kc);
    load_dwords<ONCE>(t.k[1], kc + 4 * (D / 2));
}

__device__ __forceinline__ int64_t word_index(const AttentionArgs& a, int head, int tile, int p0, int p1, int h)
{
    const int mine = h < 2 ? p0 : p1;
    return (((int64_t)max(mine, 0) * a.kv_heads + head) << a.page_log2) + ((tile + 8 * h) & ((1 << a.page_log2) - 1));
}

template <int D>
__device__ __forceinline__ void load_key_words(Keys<D>& t, const AttentionArgs& a, int head, int tile, int p0, int p1, int h)
{
    const uintx4* kw = reinterpret_cast<const uintx4*>(a.k_words + word_index(a, head, tile, p0, p1, h));
    t.kw[0] = kw[0], t.kw[1] = kw[1];
}

template <int D, bool ONCE>
__device__ __forceinline__ void load_values(Keys<D>& t, const AttentionArgs& a, int head, int tile, int p0, int p1, int c, int h)
{
    const int64_t  vat = word_index(a, head, tile, p0, p1, h);
    const uintx4*  vw  = reinterpret_cast<const uintx4*>(a.v_words + vat);
    const int      vc  = D == 96 && c >= 12 ? 0 : c;
    const uint8_t* vb  = a.v_codes + vat * (D / 2) + vc * Shape<D>::kValBytes;
    t.vw[0] = vw[0], t.vw[1] = vw[1];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (Shape<D>::kValBytes == 2)
            t.v[j][0] = *reinterpret_cast<const uint16_t*>(vb + j * (D / 2));
        else if constexpr (Shape<D>::kValBytes == 4)
            t.v[j][0] = load_as<ONCE, unsigned>(vb + j * (D / 2));
        else {
            const uintx2 w = load_as<ONCE, uintx2>(vb + j * (D / 2));
            t.v[j][0] = w[0], t.v[j][1] = w[1];
        }
    }
}

// A constant in a register: an instruction takes one literal, and with two a code's AND and OR are two instructions.
__device__ __forceinline__ unsigned in_register(unsigned v)
{
    asm("" : "+v"(v));
    return v;
}

template <int D, int RT>
struct Rows {
    half8  q[RT][Shape<D>::kSteps];
    float  qsum[RT];          // sum of the row's q, in the scores' units
    float  unit[RT];          // what a score's unit is worth, in powers of two of a probability,
    float  more[RT];          // times this: 1 but for rows with elements from 2^49 on, whose unit would not fit float32
    int    first[RT], last[RT]; // visible keys, last < first where there is none
    float  m[RT], l[RT];
    floatx4 o[RT][Shape<D>::kVal];
};

// Values whose scale is below the normal numbers, 0 in a cache that nothing was written to, are read as KV4_Append writes a
// vector of zeros: a scale of 1, codes of 0.  The exponents below are then those of normal numbers.  Seldom and by whole waves.
constexpr unsigned kLeastWord = 0x00800000u, kOneWord = 0x3f800000u;

template <int D>
__device__ __forceinline__ void zero_small(Keys<D>& t)
{
    unsigned least = t.vw[0][0];
#pragma unroll
    for (int j = 1; j < 8; ++j)
        least = min(least, t.vw[j >> 2][j & 3]);
    if (!__any(least < kLeastWord))
        return;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const bool small = t.vw[j >> 2][j & 3] < kLeastWord;
        t.vw[j >> 2][j & 3] = small ? kOneWord : t.vw[j >> 2][j & 3];
#pragma unroll
        for (int d = 0; d < (Shape<D>::kValBytes + 3) / 4; ++d)
            t.v[j][d] = small ? 0u : t.v[j][d];
    }
}

// e of a scale f 2^e, f in [1/2, 1).
__device__ __forceinline__ float exponent_of(unsigned word)
{
    return (float)__builtin_amdgcn_frexp_expf(__uint_as_float(word));
}

// Scores, softmax and product with the values for 32 keys.  The loads of the wave's next 32 are issued where the
// registers that they fill become free: the codes of the keys behind the scores, their words behind the exponents, the
// values at the end.  `edge`: some key of the tile is hidden from some row, or (`large`) some row's `more` is not 1; `gone`: the
// lane's page is not in the cache.
template <int D, int RT, typename LoadKeys, typename LoadWords, typename LoadValues>
__device__ __forceinline__ void step(Rows<D, RT>& s, Keys<D>& t, int tile, bool edge, bool large, bool gone, int h,
                                     LoadKeys load_k, LoadWords load_kw, LoadValues load_v)
{
    constexpr unsigned kLow = 0x000f000fu, kHigh = 0x00f000f0u;
    constexpr int      NV   = Shape<D>::kVal;
    floatx4 sc[2][RT];
#pragma unroll
    for (int T = 0; T < 2; ++T) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
            sc[T][r] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < Shape<D>::kSteps; ++j) {
            const unsigned w = t.k[T][j], w8 = w >> 8;
            const uintx4   raw{w & kLow, w & kHigh, w8 & kLow, w8 & kHigh};
            const half8    kk = __builtin_bit_cast(half8, raw);
#pragma unroll
            for (int r = 0; r < RT; ++r)
                sc[T][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, s.q[r][j], sc[T][r], 0, 0, 0);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    load_k();
    __builtin_amdgcn_sched_barrier(0);
    zero_small<D>(t);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned kw = t.kw[i >> 2][i & 3], vw = t.vw[i >> 2][i & 3];
        const float    zk = (float)(kw & 15u), ev = exponent_of(vw);
#pragma unroll
        for (int r = 0; r < RT; ++r) // the zero point in the scale's lowest bits is part of it
            sc[i >> 2][r][i & 3] = __builtin_fmaf(__builtin_fmaf(-zk, s.qsum[r], sc[i >> 2][r][i & 3]),
                                                  __uint_as_float(kw) * s.unit[r], ev);
    }
    __builtin_amdgcn_sched_barrier(0);
    load_kw();
    __builtin_amdgcn_sched_barrier(0);
    float f[8], il[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned vw = t.vw[i >> 2][i & 3];
        f[i]  = __builtin_amdgcn_frexp_mantf(__uint_as_float(vw));
        il[i] = __uint_as_float(0x7f000000u - (vw & 0x7f800000u)); // 2^(1 - e)
    }
    half8 pp[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        unsigned seen = 0; // bit i: the row sees key 8 h + i
        if (edge) {
            const int from = min(max(s.first[r] - tile - 8 * h, 0), 8), to = min(max(s.last[r] + 1 - tile - 8 * h, 0), 8);
            seen           = gone ? 0u : ((1u << to) - 1) & ~((1u << from) - 1);
            if (large) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float ev = exponent_of(t.vw[i >> 2][i & 3]);
                    sc[i >> 2][r][i & 3] = __builtin_fmaf(sc[i >> 2][r][i & 3] - ev, s.more[r], ev);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if ((seen >> i & 1u) == 0)
                    sc[i >> 2][r][i & 3] = -__builtin_inff();
        }
        float mx = kNone;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            mx = fmaxf(mx, sc[i >> 2][r][i & 3]);
        if (__any(mx - s.m[r] > kSlack)) { // a difference of floats is exact where their sum with 15 rounds to 16
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float m2 = fmaxf(mx - kBelow, s.m[r]), alpha = __builtin_amdgcn_exp2f(s.m[r] - m2);
            s.m[r] = m2;
            s.l[r] *= alpha;
#pragma unroll
            for (int e = 0; e < NV; ++e)
                s.o[r][e] *= alpha;
        }
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            p[i] = __builtin_amdgcn_exp2f(sc[i >> 2][r][i & 3] - s.m[r]);
        if (edge) { // the words of a hidden key may be anything
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool shown = (seen >> i & 1u) != 0;
                s.l[r] += shown ? p[i] * il[i] : 0.f;
                p[i] = shown ? p[i] * f[i] : 0.f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s.l[r] = __builtin_fmaf(p[i], il[i], s.l[r]);
                p[i] *= f[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) // rounded to 11 bits, as the output is: errors of either sign that average over the keys
            pp[r][i] = (_Float16)p[i];
    }
    // -(1024 + z) and -(64 + z) of pairs of keys
    const unsigned low = in_register(kLow), up = in_register(kHigh);
    half2          below[4], above[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned z = __builtin_amdgcn_perm(t.vw[i >> 1][2 * (i & 1) + 1], t.vw[i >> 1][2 * (i & 1)], 0x05040100u) & kLow;
        below[i] = __builtin_bit_cast(half2, z | 0xe400e400u);
        above[i] = __builtin_bit_cast(half2, z << 4 | 0xd400d400u);
    }
#pragma unroll
    for (int g = 0; g < (NV + 3) / 4; ++g) { // four elements of every key: one half of a dword
        uintx4 a0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            a0[i] = __builtin_amdgcn_perm(t.v[2 * i + 1][g >> 1], t.v[2 * i][g >> 1], (g & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uintx4 raw;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned w = e >= 2 ? a0[i] >> 8 : a0[i];
                const half2    v = (e & 1) ? __builtin_bit_cast(half2, (w & up) | 0x54005400u) + above[i]
                                           : __builtin_bit_cast(half2, (w & low) | 0x64006400u) + below[i];
                raw[i] = __builtin_bit_cast(unsigned, v);
            }
            const half8 va = __builtin_bit_cast(half8, raw);
#pragma unroll
            for (int r = 0; r < RT; ++r)
                s.o[r][4 * g + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pp[r], s.o[r][4 * g + e], 0, 0, 0);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    load_v();
    __builtin_amdgcn_sched_barrier(0);
}

// Rows of a block of 16 RT: the heads that share a key/value head for one token, then for the next.  Where sequences have
// different numbers of rows, a sequence's blocks begin at floor(first token * share / rows of a block) + its number, which leaves room for all of every sequence's.
__device__ __forceinline__ int block_base(const AttentionArgs& a, int b, int rows)
{
    if (a.cu == nullptr)
        return b * ((a.share + rows - 1) / rows);
    return (int)((int64_t)a.cu[b] * a.share / rows) + b;
}

// Where a block of rows stands: its sequence b, the sequence's first row, the place of that row's token (below 0 where it has
// none), the block's first row among the sequence's and how many it has (0: there is no such block).
struct Place {
    int b, first, place0, row0, rows, share;

    // Keys that some of rows `from` .. `from + count - 1` of the block see, lo .. hi, and those that all see, lo_all .. hi_all.
    __device__ __forceinline__ int top(int row) const { return place0 + (row0 + row) / share; }
    __device__ __forceinline__ int lo(const AttentionArgs& a, int from, int) const
    {
        return a.window > 0 ? max(0, top(from) - a.window + 1) : 0;
    }
    __device__ __forceinline__ int hi(const AttentionArgs&, int cap, int from, int count) const
    {
        return min(top(from + count - 1), cap - 1);
    }
    __device__ __forceinline__ int lo_all(const AttentionArgs& a, int from, int count) const
    {
        return a.window > 0 ? max(0, top(from + count - 1) - a.window + 1) : 0;
    }
    __device__ __forceinline__ int hi_all(int cap, int from, int count) const
    {
        return top(from) < 0 || top(from + count - 1) >= cap ? -1 : top(from);
    }
};

__device__ __forceinline__ Place place_of(const AttentionArgs& a, int block, int rows)
{
    Place p;
    p.b = 0, p.share = a.share, p.rows = 0;
    if (a.cu == nullptr) {
        p.b = block / ((a.share + rows - 1) / rows);
    } else {
        for (int top = a.batch; top - p.b > 1;) {
            const int mid = (p.b + top) >> 1;
            if (block_base(a, mid, rows) <= block)
                p.b = mid;
            else
                top = mid;
        }
    }
    const int behind = a.cu ? uniform_load(a.cu + p.b + 1) : p.b + 1;
    p.first          = a.cu ? uniform_load(a.cu + p.b) : p.b;
    p.place0         = uniform_load(a.lens + p.b) - (behind - p.first);
    p.row0           = (block - block_base(a, p.b, rows)) * rows;
    const int64_t left = (int64_t)(min(behind, a.tokens) - p.first) * a.share - p.row0;
    if (p.first >= 0 && p.row0 >= 0)
        p.rows = (int)min<int64_t>(rows, max<int64_t>(left, 0));
    return p;
}

// Rows of no sequence are 0 (with splits kv4_attention_join writes them): dealt to the blocks.
template <int D>
__device__ __forceinline__ void zero_idle(const AttentionArgs& a, int head, int block, int blocks)
{
    if (a.cu == nullptr || a.splits != 1)
        return;
    const int before = min(max(uniform_load(a.cu), 0), a.tokens), behind = min(max(uniform_load(a.cu + a.batch), 0), a.tokens);
    const int idle = before + a.tokens - behind;
    for (int i = block; i < idle; i += blocks) {
        const int64_t at = (int64_t)(i < before ? i : behind + i - before) * a.q_heads + head * a.share;
        for (int e = threadIdx.x; e < a.share * (D / 8); e += kWave * kWaves)
            *reinterpret_cast<uintx4*>(a.out + at * D + e * 8) = uintx4{0, 0, 0, 0};
        if (a.lse != nullptr)
            for (int e = threadIdx.x; e < a.share; e += kWave * kWaves)
                a.lse[at + e] = -__builtin_inff();
    }
}

template <int D, int RT, bool ONCE>
__global__ __launch_bounds__(kWave* kWaves, Shape<D>::waves(RT)) void kv4_attention(AttentionArgs a)
{
    constexpr int NV = Shape<D>::kVal, kRows = 16 * RT;
    __shared__ float join[kWaves][16][D + 4];
    __shared__ float join_m[kWaves][kRows], join_l[kWaves][kRows];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, h = lane >> 4;
    // heads are dealt first: workgroups go to the eight dies in turn, and so do a sequence's heads, whatever its length, while
    // all of a head's blocks of rows find its keys in one L2 wherever the number of heads is a multiple of eight
    const int head = blockIdx.x % a.kv_heads, block = blockIdx.x / a.kv_heads, split = blockIdx.y;

    zero_idle<D>(a, head, block, (int)(gridDim.x / a.kv_heads));

    const Place p = place_of(a, block, kRows);
    if (p.rows <= 0)
        return;
    const int  first = p.first, row0 = p.row0, rows = p.rows, place0 = p.place0;
    const int  cap   = a.width << a.page_log2;
    const int* table = a.table + (int64_t)p.b * a.stride;
    const int  lo = p.lo(a, 0, rows), hi = p.hi(a, cap, 0, rows), lo_all = p.lo_all(a, 0, rows), hi_all = p.hi_all(cap, 0, rows);
    // the workgroup's share of them in tiles of 32; wave w takes every fourth
    const int  t_lo = lo / kTile, t_all = hi < lo ? 0 : hi / kTile + 1 - t_lo, per = (t_all + a.splits - 1) / a.splits;
    const int  t0 = t_lo + split * per, t1 = min(t_lo + t_all, t0 + per);
    int        t = t0 + wave;
    const bool any = t < t1;

    // the first tile's loads go ahead of the queries'
    Keys<D> keys;
    int     p0 = -1, p1 = -1, n0 = -1, n1 = -1, tn = t;
    if (any) {
        p0 = page_of(a, entry_at(a, table, t * kTile), t * kTile);
        p1 = page_of(a, entry_at(a, table, t * kTile + 16), t * kTile + 16);
        tn = min(t + kWaves, t1 - 1); // the wave's last tile is loaded once more and not used
        n0 = entry_at(a, table, tn * kTile), n1 = entry_at(a, table, tn * kTile + 16);
        load_keys<D, ONCE>(keys, a, head, t * kTile, p0, p1, c, h);
        load_key_words<D>(keys, a, head, t * kTile, p0, p1, h);
        load_values<D, ONCE>(keys, a, head, t * kTile, p0, p1, c, h);
    }
    __builtin_amdgcn_sched_barrier(0);

    // the block's queries, each row scaled by a power of two that brings its largest element to 2^13: fp16 then holds them
    // exactly down to 2^-27 of that, with a factor 1/16 on those that meet the second nibble of a half
    Rows<D, RT> s;
    bool        large = false;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int  row  = r * 16 + c;
        const bool live = row < rows;
        const int  tok = (row0 + (live ? row : 0)) / a.share, sub = (row0 + (live ? row : 0)) % a.share;
        const uint16_t* q = a.q + (int64_t)(first + tok) * a.q_token + (int64_t)(head * a.share + sub) * a.q_head + h * (D / 4);
        uintx4 raw[Shape<D>::kSteps];
#pragma unroll
        for (int j = 0; j < Shape<D>::kSteps; ++j)
            raw[j] = *reinterpret_cast<const uintx4*>(q + 8 * j);
        float qmax = 0.f;
#pragma unroll
        for (int j = 0; j < Shape<D>::kSteps; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                qmax = fmaxf(qmax, fabsf(from16((uint16_t)(raw[j][i >> 1] >> (16 * (i & 1))), a.bf16)));
        qmax = fmaxf(qmax, __shfl_xor(qmax, 16));
        qmax = fmaxf(qmax, __shfl_xor(qmax, 32));
        // an infinity spoils the row whatever the scale; frexp: qmax < 2^exp
        const int qexp = qmax > 0.f && qmax < 3.4e38f ? min(13 - (int)__builtin_amdgcn_frexp_expf(qmax), 110) : 0;
        float     sum  = 0.f;
#pragma unroll
        for (int j = 0; j < Shape<D>::kSteps; ++j) {
            half8         v;
            constexpr int kOrder[8] = {0, 4, 1, 5, 2, 6, 3, 7}; // element of each half of the unpacked dword
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int   e    = kOrder[i];
                const float full = ldexpf(from16((uint16_t)(raw[j][e >> 1] >> (16 * (e & 1))), a.bf16), qexp);
                v[i]             = (_Float16)((i >> 1) & 1 ? full * 0.0625f : full);
                sum += (float)(_Float16)full;
            }
            s.q[r][j] = v;
        }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        s.qsum[r] = sum * 0x1p-24f;
        s.unit[r] = ldexpf(a.scale_log2, min(24 - qexp, 60));
        s.more[r] = ldexpf(1.f, max(24 - qexp, 60) - 60);
        large     = large || s.more[r] != 1.f;
        const int place = place0 + tok;
        s.first[r] = live && a.window > 0 ? max(0, place - a.window + 1) : 0;
        s.last[r]  = live && place < cap ? place : -1;
        s.m[r] = kNone;
        s.l[r] = 0.f;
#pragma unroll
        for (int e = 0; e < NV; ++e)
            s.o[r][e] = floatx4{0.f, 0.f, 0.f, 0.f};
    }

    large = __any(large);
    if (any) {
        for (; t < t1; t += kWaves) {
            const int  tile = t * kTile, next = tn * kTile;
            const int  q0 = page_of(a, n0, next), q1 = page_of(a, n1, next + 16);
            const bool whole = p0 >= 0 && p1 >= 0 && tile >= lo_all && tile + kTile - 1 <= hi_all;
            tn = min(tn + kWaves, t1 - 1);
            n0 = entry_at(a, table, tn * kTile), n1 = entry_at(a, table, tn * kTile + 16);
            step<D, RT>(
                s, keys, tile, !whole || large, large, (h < 2 ? p0 : p1) < 0, h,
                [&] { load_keys<D, ONCE>(keys, a, head, next, q0, q1, c, h); },
                [&] { load_key_words<D>(keys, a, head, next, q0, q1, h); },
                [&] { load_values<D, ONCE>(keys, a, head, next, q0, q1, c, h); });
            p0 = q0, p1 = q1;
        }
    }

    // join the waves
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        s.l[r] += __shfl_xor(s.l[r], 16);
        s.l[r] += __shfl_xor(s.l[r], 32);
        if (h == 0) {
            join_m[wave][r * 16 + c] = s.m[r];
            join_l[wave][r * 16 + c] = s.l[r];
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        float m = kNone;
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
            m = fmaxf(m, join_m[w][r * 16 + c]);
        const float alpha = __builtin_amdgcn_exp2f(s.m[r] - m);
        if (r > 0)
            __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < NV; ++e) {
                const int d = NV * (4 * h + i) + e;
                if (D != 96 || d < D) {
                    join[wave][c][d] = s.o[r][e][i] * alpha * 2.f; // f is half of the mantissa
                }
            }
        __syncthreads();
        for (int at = threadIdx.x; at < 16 * (D / 8); at += kWave * kWaves) {
            const int row = at / (D / 8), d0 = at % (D / 8) * 8;
            if (r * 16 + row >= rows)
                break;
            float mm = kNone, l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            for (int w = 0; w < kWaves; ++w)
                mm = fmaxf(mm, join_m[w][r * 16 + row]);
            for (int w = 0; w < kWaves; ++w) {
                l += join_l[w][r * 16 + row] * __builtin_amdgcn_exp2f(join_m[w][r * 16 + row] - mm);
                for (int i = 0; i < 8; ++i)
                    o[i] += join[w][row][d0 + i];
            }
            const int     g   = row0 + r * 16 + row;
            const int64_t idx = (int64_t)(first + g / a.share) * a.q_heads + head * a.share + g % a.share;
            if (a.splits > 1) {
                float* dst = a.part_o + ((int64_t)split * a.tokens * a.q_heads + idx) * D + d0;
                *reinterpret_cast<floatx4*>(dst)     = floatx4{o[0], o[1], o[2], o[3]};
                *reinterpret_cast<floatx4*>(dst + 4) = floatx4{o[4], o[5], o[6], o[7]};
                if (d0 == 0) {
                    float* ml = a.part_ml + ((int64_t)split * a.tokens * a.q_heads + idx) * 2;
                    ml[0] = mm, ml[1] = l;
                }
                continue;
            }
            const bool  none = l == 0.f; // no key seen (a sum of probabilities is never 0 otherwise)
            const float inv  = none ? 0.f : 1.f / l;
            uint16_t    e[8];
            for (int i = 0; i < 8; ++i)
                e[i] = to16(none ? 0.f : o[i] * inv, a.bf16);
            uintx4 v;
            __builtin_memcpy(&v, e, 16);
            *reinterpret_cast<uintx4*>(a.out + idx * D + d0) = v;
            if (a.lse != nullptr && d0 == 0) // l is twice the sum relative to m
                a.lse[idx] = none ? -__builtin_inff() : (__log2f(l) + (mm - 1.f)) * 0.69314718055994531f;
        }
    }
}

// Many rows per sequence (prompts and chunks of them): the waves of a workgroup, two row tiles each, share the keys, which go
// unpacked through LDS, 16 for every wave at a time: half of the waves unpack the codes of 32 keys each, the others those of
// values, as operands of the products, and the words as what a score is multiplied by (u), what is added to it (ev) and what
// its probability counts in the sum (il).  Bound by the issue of vector and matrix instructions, whose times were found to add
// up: 2 x 1024 rows over 8192 keys, 32 heads over 8 of 128 take 287 us, 715 TFLOP/s (a large product of the library reaches 1546);
// kv4_attention, which unpacks a key for every 32 rows, took 431 before this kernel was there.  Here z is taken off the keys' codes too, all rows of the block share the queries'
// scale, and a value's whole scale goes into the exponent, p'_t = 2^(log2 p_t + log2 s_t - m), with il = 2^-6 / s_t:
// logarithm and reciprocal are taken once for all rows of the block, and save a product for each probability.
template <int D>
struct Slab { // of 64 keys
    uintx4 k[4][D / 32][kWave];
    uintx4 v[2][Shape<D>::kVal][kWave];
    float  u[64], ev[64], il[64];
};

// What a wave loads of a slab: 32 keys' codes or values.
struct Raw {
    unsigned d[8];
    uintx4   w[2];
    unsigned own;
};

// The 32 keys from `base` on; p0 and p1 are the pages of the two halves.
template <int D>
__device__ __forceinline__ void load_raw(Raw& t, const AttentionArgs& a, int head, int base, int p0, int p1, bool values,
                                         int lane)
{
    // entries of the cache at the halves' beginnings, the same for the whole wave
    const int     c = lane & 15, h = lane >> 4, mask = (1 << a.page_log2) - 1;
    const int64_t half0 = (((int64_t)max(p0, 0) * a.kv_heads + head) << a.page_log2) + (base & mask);
    const int64_t half1 = (((int64_t)max(p1, 0) * a.kv_heads + head) << a.page_log2) + ((base + 16) & mask);
    const int64_t own   = ((lane & 31) < 16 ? half0 : half1) + (lane & 15);
    if (values) {
        const int64_t  vat = (h < 2 ? half0 : half1) + 8 * (h & 1);
        const uint8_t* vb  = a.v_codes + vat * (D / 2) + (D == 96 && c >= 12 ? 0 : c) * Shape<D>::kValBytes;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (Shape<D>::kValBytes == 2)
                t.d[j] = *reinterpret_cast<const uint16_t*>(vb + j * (D / 2));
            else
                t.d[j] = *reinterpret_cast<const unsigned*>(vb + j * (D / 2));
        }
        const uintx4* vw = reinterpret_cast<const uintx4*>(a.v_words + vat);
        t.w[0] = vw[0], t.w[1] = vw[1];
        t.own  = (unsigned)a.v_words[own];
    } else {
        constexpr int  N   = D / 32;
        const int64_t  kat = (c < 8 ? half0 : half1) + 8 * ((c >> 2) & 1) + (c & 3);
        const uint8_t* kc  = a.k_codes + kat * (D / 2) + h * (D / 8);
        unsigned       x[2][N];
        load_dwords<false>(x[0], kc);
        load_dwords<false>(x[1], kc + 4 * (D / 2));
#pragma unroll
        for (int j = 0; j < N; ++j)
            t.d[j] = x[0][j], t.d[N + j] = x[1][j];
        t.w[0][0] = (unsigned)a.k_words[kat], t.w[0][1] = (unsigned)a.k_words[kat + 4];
        t.own     = (unsigned)a.k_words[own];
    }
}

template <int D>
__device__ __forceinline__ void unpack(Slab<D>& slab, Raw& t, int g, bool values, float unit, int lane)
{
    const unsigned low = in_register(0x000f000fu), up = in_register(0x00f000f0u);
    auto code = [&](unsigned w, bool high, unsigned below, unsigned above) {
        const half2 v = high ? __builtin_bit_cast(half2, (w & up) | 0x54005400u) + __builtin_bit_cast(half2, above)
                             : __builtin_bit_cast(half2, (w & low) | 0x64006400u) + __builtin_bit_cast(half2, below);
        return __builtin_bit_cast(unsigned, v);
    };
    if (values) {
        const unsigned small = (unsigned)__ballot(t.own < kLeastWord); // bit i: key i of the 32; as zero_small
        if (__builtin_expect(small != 0, 0)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool mine = (small >> (8 * (lane >> 4) + j) & 1u) != 0;
                t.d[j] = mine ? 0u : t.d[j];
                t.w[j >> 2][j & 3] = mine ? kOneWord : t.w[j >> 2][j & 3];
            }
            t.own = t.own < kLeastWord ? kOneWord : t.own;
        }
        unsigned below[4], above[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned z = __builtin_amdgcn_perm(t.w[i >> 1][2 * (i & 1) + 1], t.w[i >> 1][2 * (i & 1)], 0x05040100u) & low;
            below[i] = z | 0xe400e400u;
            above[i] = z << 4 | 0xd400d400u;
        }
#pragma unroll
        for (int q = 0; q < Shape<D>::kVal / 4; ++q) {
            uintx4 a0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                a0[i] = __builtin_amdgcn_perm(t.d[2 * i + 1], t.d[2 * i], (q & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uintx4 out;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    out[i] = code(e >= 2 ? a0[i] >> 8 : a0[i], (e & 1) != 0, below[i], above[i]);
                slab.v[g][4 * q + e][lane] = out;
            }
        }
        if (lane < 32) { // a scale that is no positive number: NaN where it is seen, 0 where it is hidden
            const float w    = __uint_as_float(t.own);
            const bool  fine = w > 0.f && w < __builtin_inff();
            slab.ev[32 * g + lane] = fine ? __log2f(w) : __uint_as_float(0x7fc00000u);
            slab.il[32 * g + lane] = fine ? 0x1p-6f / w : 0.f;
        }
    } else {
#pragma unroll
        for (int T = 0; T < 2; ++T) {
            const unsigned z = (t.w[0][T] & 15u) * 0x00010001u, below = z | 0xe400e400u, above = z << 4 | 0xd400d400u;
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                const unsigned w = t.d[T * (D / 32) + j], w8 = w >> 8;
                slab.k[2 * g + T][j][lane] = uintx4{code(w, false, below, above), code(w, true, below, above),
                                                    code(w8, false, below, above), code(w8, true, below, above)};
            }
        }
        if (lane < 32)
            slab.u[32 * g + lane] = __uint_as_float(t.own) * unit;
    }
}

template <int D, int W>
__global__ __launch_bounds__(kWave* W, 2) void kv4_attention_rows(AttentionArgs a)
{
    constexpr int NV = Shape<D>::kVal, kSteps = Shape<D>::kSteps, RT = 2, kRows = 16 * RT * W, kStep = 16 * W;
    __shared__ Slab<D> slab[2][W / 4];
    __shared__ float   tops[W];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, h = lane >> 4;
    // the last blocks of rows, which see the most keys, go first
    const int head = blockIdx.x % a.kv_heads, blocks = gridDim.x / a.kv_heads, block = blocks - 1 - (int)blockIdx.x / a.kv_heads;
    const int split = blockIdx.y;
    zero_idle<D>(a, head, block, blocks);

    const Place p = place_of(a, block, kRows);
    if (p.rows <= 0)
        return;
    const int  cap = a.width << a.page_log2;
    const int* table = a.table + (int64_t)p.b * a.stride;
    const int  lo = p.lo(a, 0, p.rows), hi = p.hi(a, cap, 0, p.rows);
    const int  t_lo = lo / kStep, t_all = hi < lo ? 0 : hi / kStep + 1 - t_lo, per = (t_all + a.splits - 1) / a.splits;
    const int  t0 = t_lo + split * per, t1 = min(t_lo + t_all, t0 + per);
    // this wave's rows, and the keys that some, and that all of them see
    const int  w0 = wave * 16 * RT, w_rows = max(0, min(16 * RT, p.rows - w0));
    const int  w_lo = w_rows > 0 ? p.lo(a, w0, w_rows) : 0, w_hi = w_rows > 0 ? p.hi(a, cap, w0, w_rows) : -1;
    const int  all_lo = w_rows > 0 ? p.lo_all(a, w0, w_rows) : 0, all_hi = w_rows > 0 ? p.hi_all(cap, w0, w_rows) : -1;

    const int  group = wave % (W / 2); // the 32 keys that this wave unpacks
    const bool values = wave >= W / 2;
    Raw        raw;
    // Loads this wave's keys of step t, and for lane i the table's entry for keys 16 i .. of the step: which of them lie in no
    // page of the cache is asked for a step later.
    int  entry = 0;
    auto load = [&](int t) {
        const int pos = t * kStep + 32 * group, mine = t * kStep + 16 * (lane & (W - 1));
        const int p0 = page_of(a, entry_at(a, table, pos), pos), p1 = page_of(a, entry_at(a, table, pos + 16), pos + 16);
        entry = table[min(mine >> a.page_log2, a.width - 1)];
        load_raw<D>(raw, a, head, t * kStep + 32 * group, p0, p1, values, lane);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto absent = [&](int t) { // bit i: keys 16 i .. of step t, the one that was loaded last
        return (unsigned)__ballot(page_of(a, entry, t * kStep + 16 * (lane & (W - 1))) < 0) & ((1u << W) - 1);
    };
    if (t0 < t1)
        load(t0);

    // queries
    half8 q[RT][kSteps];
    int   first[RT], last[RT];
    float m[RT], l[RT];
    floatx4 o[RT][NV];
    uintx4  qraw[RT][kSteps];
    float   top = 0.f, row_top[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int  row  = w0 + r * 16 + c;
        const bool live = row < p.rows;
        const int  at = p.row0 + (live ? row : 0), tok = at / a.share, sub = at % a.share;
        const uint16_t* src = a.q + (int64_t)(p.first + tok) * a.q_token + (int64_t)(head * a.share + sub) * a.q_head + h * (D / 4);
        const int place = p.place0 + tok;
        first[r] = live && a.window > 0 ? max(0, place - a.window + 1) : 0;
        last[r]  = live && place < cap ? place : -1;
        m[r] = kNone, l[r] = 0.f;
#pragma unroll
        for (int d = 0; d < NV; ++d)
            o[r][d] = floatx4{0.f, 0.f, 0.f, 0.f};
        row_top[r] = 0.f;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            qraw[r][j] = *reinterpret_cast<const uintx4*>(src + 8 * j);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float mag = fabsf(from16((uint16_t)(qraw[r][j][i >> 1] >> (16 * (i & 1))), a.bf16));
                if (last[r] >= 0 && mag < 3.4e38f) // rows that see nothing and infinities do not count
                    row_top[r] = fmaxf(row_top[r], mag);
            }
        }
        row_top[r] = fmaxf(row_top[r], __shfl_xor(row_top[r], 16));
        row_top[r] = fmaxf(row_top[r], __shfl_xor(row_top[r], 32));
        top        = fmaxf(top, row_top[r]);
    }
#pragma unroll
    for (int x = 1; x < 16; x <<= 1)
        top = fmaxf(top, __shfl_xor(top, x));
    if (lane == 0)
        tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w)
        top = fmaxf(top, tops[w]);
    auto exponent = [](float x) { return x > 0.f ? min(13 - (int)__builtin_amdgcn_frexp_expf(x), 110) : 0; };
    // not below -20, elements of 2^33: with the exponent of a row near the type's end the scores of its neighbours, scaled by their
    // own, would not fit float32 before they are corrected
    const int   qexp = max(__builtin_amdgcn_readfirstlane(exponent(top)), -20);
    const float unit = ldexpf(a.scale_log2, -qexp);
    // A wave with a row 2^16 below the block's largest (fp16 would lose its bits) or above that exponent's range scales its rows one
    // by one and corrects the scores where it also hides keys, so that calls without such rows pay nothing for it.
    float row_unit[RT];
    int   row_exp[RT];
    bool  far = false;
#pragma unroll
    for (int r = 0; r < RT; ++r)
        far = far || (row_top[r] > 0.f && (exponent(row_top[r]) > qexp + 16 || exponent(row_top[r]) < qexp));
    const bool apart = __ballot(far) != 0;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        row_exp[r]  = apart && row_top[r] > 0.f ? exponent(row_top[r]) : qexp;
        row_unit[r] = ldexpf(1.f, qexp - row_exp[r]);
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            constexpr int kOrder[8] = {0, 4, 1, 5, 2, 6, 3, 7}; // element of each half of the unpacked dword
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int x = kOrder[i];
                q[r][j][i]  = (_Float16)ldexpf(from16((uint16_t)(qraw[r][j][x >> 1] >> (16 * (x & 1))), a.bf16), row_exp[r]);
            }
        }

    // 64 keys; bit i of `gone`: the i-th sixteen of them lie in no page
    auto work = [&](const Slab<D>& b, int tile, unsigned gone) {
        if (tile > w_hi || tile + 63 < w_lo)
            return;
        const bool edge = (gone & 15u) != 0 || tile < all_lo || tile + 63 > all_hi || apart;
        floatx4    sc[4][RT];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int r = 0; r < RT; ++r)
                sc[k][r] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const half8 kk = __builtin_bit_cast(half8, b.k[k][j][lane]);
#pragma unroll
                for (int r = 0; r < RT; ++r)
                    sc[k][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, q[r][j], sc[k][r], 0, 0, 0);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) { // keys 32 (k / 2) + 8 h + 4 (k % 2) + i
            const int     at = 32 * (k >> 1) + 8 * h + 4 * (k & 1);
            const floatx4 u = *reinterpret_cast<const floatx4*>(&b.u[at]), ev = *reinterpret_cast<const floatx4*>(&b.ev[at]);
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sc[k][r][i] = __builtin_fmaf(sc[k][r][i], u[i], ev[i]);
        }
        if (edge) {
            if (apart) { // (S u + ev - ev) row_unit + ev
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const floatx4 ev = *reinterpret_cast<const floatx4*>(&b.ev[32 * (k >> 1) + 8 * h + 4 * (k & 1)]);
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            sc[k][r][i] = __builtin_fmaf(sc[k][r][i] - ev[i], row_unit[r], ev[i]);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int  none = -(int)((gone >> (2 * (k >> 1) + (h >> 1))) & 1u);
                const int  at   = tile + 32 * (k >> 1) + 8 * h + 4 * (k & 1);
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int hidden = (at + i - first[r]) | (last[r] - at - i) | none; // below 0 where it is
                        sc[k][r][i] = hidden < 0 ? -__builtin_inff() : sc[k][r][i];
                    }
            }
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            float mx = kNone;
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    mx = fmaxf(mx, sc[k][r][i]);
            if (__any(mx - m[r] > kSlack)) { // exact, as in kv4_attention
                mx = fmaxf(mx, __shfl_xor(mx, 16));
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                const float m2 = fmaxf(mx - kBelow, m[r]), alpha = __builtin_amdgcn_exp2f(m[r] - m2);
                m[r] = m2;
                l[r] *= alpha;
#pragma unroll
                for (int d = 0; d < NV; ++d)
                    o[r][d] *= alpha;
            }
        }
        half8 pp[2][RT];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const floatx4 il = *reinterpret_cast<const floatx4*>(&b.il[32 * (k >> 1) + 8 * h + 4 * (k & 1)]);
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float ex = __builtin_amdgcn_exp2f(sc[k][r][i] - m[r]);
                    l[r] = __builtin_fmaf(ex, il[i], l[r]);
                    pp[k >> 1][r][4 * (k & 1) + i] = (_Float16)ex; // rounded to 11 bits, as in kv4_attention
                }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int d = 0; d < NV; ++d) {
                const half8 va = __builtin_bit_cast(half8, b.v[k][d][lane]);
#pragma unroll
                for (int r = 0; r < RT; ++r)
                    o[r][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pp[k][r], o[r][d], 0, 0, 0);
            }
    };

    if (t0 < t1) {
        unpack<D>(slab[0][group >> 1], raw, group & 1, values, unit, lane);
        unsigned gone = absent(t0);
        load(min(t0 + 1, t1 - 1));
        __syncthreads();
        for (int t = t0; t < t1; ++t) {
#pragma unroll
            for (int x = 0; x < W / 4; ++x)
                work(slab[(t - t0) & 1][x], t * kStep + 64 * x, gone >> (4 * x));
            if (t + 1 < t1) { // the other slab was last read before the barrier
                unpack<D>(slab[(t + 1 - t0) & 1][group >> 1], raw, group & 1, values, unit, lane);
                gone = absent(t + 1);
                load(min(t + 2, t1 - 1));
            }
            __syncthreads();
        }
    }

    // a lane holds 4 NV elements in a row of its row
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        l[r] += __shfl_xor(l[r], 16);
        l[r] += __shfl_xor(l[r], 32);
        const int row = w0 + r * 16 + c;
        if (row >= p.rows || 4 * NV * h >= D)
            continue;
        const int     at  = p.row0 + row;
        const int64_t idx = (int64_t)(p.first + at / a.share) * a.q_heads + head * a.share + at % a.share;
        if (a.splits > 1) {
            float* dst = a.part_o + ((int64_t)split * a.tokens * a.q_heads + idx) * D + 4 * NV * h;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int d = 0; d < NV; d += 4)
                    *reinterpret_cast<floatx4*>(dst + NV * i + d) = floatx4{o[r][d][i] * 0x1p-6f, o[r][d + 1][i] * 0x1p-6f,
                                                                           o[r][d + 2][i] * 0x1p-6f, o[r][d + 3][i] * 0x1p-6f};
            if (h == 0) {
                float* ml = a.part_ml + ((int64_t)split * a.tokens * a.q_heads + idx) * 2;
                ml[0] = m[r] + 7.f, ml[1] = l[r]; // as kv4_attention counts, whose sums are twice theirs, these 2^-6 of them
            }
            continue;
        }
        const bool  none = l[r] == 0.f;
        const float inv  = none ? 0.f : 0x1p-6f / l[r]; // as il is
        uint16_t    out[4 * NV];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < NV; ++d)
                out[NV * i + d] = to16(none ? 0.f : o[r][d][i] * inv, a.bf16);
        uint16_t* dst = a.out + idx * D + 4 * NV * h;
#pragma unroll
        for (int i = 0; i < 4 * NV; i += 8) {
            uintx4 v;
            __builtin_memcpy(&v, out + i, 16);
            *reinterpret_cast<uintx4*>(dst + i) = v;
        }
        if (a.lse != nullptr && h == 0)
            a.lse[idx] = none ? -__builtin_inff() : (__log2f(l[r]) + (m[r] + 6.f)) * 0.69314718055994531f;
    }
}

// Joins the splits of a row: threads of one row take 8 elements each, in `lanes` groups that deal the splits among them and
// meet in LDS.  Latency decides: 32 rows of 64 splits 5.5 us, 1280 rows of a few 3.4.
template <int D>
__global__ __launch_bounds__(256) void kv4_attention_join(AttentionArgs a, int lanes)
{
    constexpr int kChunks = D / 8;
    __shared__ float part[256][11];
    const int     width = kChunks * lanes, rows = 256 / width; // threads of a row, rows of a workgroup
    const int     in = threadIdx.x % width, chunk = in % kChunks, lane = in / kChunks;
    const int64_t all = (int64_t)a.tokens * a.q_heads, idx = (int64_t)blockIdx.x * rows + threadIdx.x / width;
    const bool    live = (int)threadIdx.x < rows * width && idx < all;
    float         mm = kNone, l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    // a token of no sequence has no partial results: its row is 0
    const int token = (int)(idx / a.q_heads);
    if (live && (a.cu == nullptr || (token >= a.cu[0] && token < a.cu[a.batch]))) {
        for (int s = lane; s < a.splits; s += lanes)
            mm = fmaxf(mm, a.part_ml[(s * all + idx) * 2]);
        for (int s = lane; s < a.splits; s += lanes) {
            const float  w   = __builtin_amdgcn_exp2f(a.part_ml[(s * all + idx) * 2] - mm);
            const float* src = a.part_o + (s * all + idx) * D + chunk * 8;
            const floatx4 u = *reinterpret_cast<const floatx4*>(src), v = *reinterpret_cast<const floatx4*>(src + 4);
            l += w * a.part_ml[(s * all + idx) * 2 + 1];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                o[i] += w * u[i];
                o[4 + i] += w * v[i];
            }
        }
    }
    if (lanes > 1) {
        float* mine = part[threadIdx.x];
        mine[8] = mm, mine[9] = l;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            mine[i] = o[i];
        __syncthreads();
        if (!live || lane != 0)
            return;
        for (int g = 1; g < lanes; ++g)
            mm = fmaxf(mm, part[threadIdx.x + g * kChunks][8]);
        l = 0.f;
        for (int i = 0; i < 8; ++i)
            o[i] = 0.f;
        for (int g = 0; g < lanes; ++g) {
            const float* p = part[threadIdx.x + g * kChunks];
            const float  w = __builtin_amdgcn_exp2f(p[8] - mm);
            l += w * p[9];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                o[i] += w * p[i];
        }
    } else if (!live) {
        return;
    }
    const bool  none = l == 0.f;
    const float inv  = none ? 0.f : 1.f / l;
    uint16_t    e[8];
    for (int i = 0; i < 8; ++i)
        e[i] = to16(none ? 0.f : o[i] * inv, a.bf16);
    uintx4 v;
    __builtin_memcpy(&v, e, 16);
    *reinterpret_cast<uintx4*>(a.out + idx * D + chunk * 8) = v;
    if (a.lse != nullptr && chunk == 0)
        a.lse[idx] = none ? -__builtin_inff() : (__log2f(l) + (mm - 1.f)) * 0.69314718055994531f;
}

namespace {

struct Plan {
    int     row_tiles, splits; // row tiles of a block; 8: kv4_attention_rows
    bool    once; // the average sequence has one block of rows
    int64_t blocks;
};

constexpr int kManyRows = 64; // average rows of a sequence from which its keys go through LDS

// Row tiles: as many as the average sequence fills.  Splits of the keys: two workgroups for every CU (three quarters of that
// is as good where they are long), none of less than 16 tiles of 32 keys (4 where all waves share them), and none at all
// below 32 tiles: the second launch costs 3 us.  Measured in us with 1 / 2 / 4 / 8 / 16 splits: one sequence of 2048 keys,
// 40 heads 19.5 / 16.4 / 13.5 / 13.9 / 13.9 (4 here); 131071 keys, 8 key/value heads 1020 / 518 / 265 / 139 / 76, then 46 / 39 /
// 44 with 32 / 64 / 128 (64 here); 4 sequences of 1000 keys, 8 heads 11.9 / 12.8 / 12.9 / 12.7 / 12.8 (1 here); 30 new tokens of
// 2 sequences of 1000 keys, 16 heads over 4 34.7 / 26.2 / 20.5 / 18.9 / 20.1 (8 here); 1024 new tokens over 8192 keys, 456
// workgroups 313 / 328 / 317 / 367 / 498 (1 here); 256 new tokens of 4 sequences over 8192, 288 workgroups 332 / 195 / 210 / 248 /
// 317 (2 here).
Plan plan_of(const KV4_Cache& c, const KV4_Batch& b, int q_heads, int window, int max_len)
{
    Plan          p;
    const int     share = q_heads / c.kv_heads;
    const int64_t rows  = (int64_t)b.total_tokens * share, each = (rows + b.batch - 1) / b.batch;
    p.row_tiles = each <= 16 || c.head_dim == 256 ? 1 : (each <= kManyRows ? 2 : 8);
    const int64_t per = 16 * p.row_tiles;
    p.once            = each <= per;
    p.blocks          = (b.cu_tokens == nullptr ? b.batch * ((share + per - 1) / per) : rows / per + b.batch);
    const int64_t capacity = (int64_t)b.table_width * c.page_size;
    int64_t       len      = max_len > 0 ? std::min<int64_t>(max_len, capacity) : capacity;
    if (window > 0) // what a block's rows see of it
        len = std::min<int64_t>(len, (int64_t)window + (per + share - 1) / share + kTile);
    const int64_t tiles = (len + kTile - 1) / kTile, groups = (int64_t)p.blocks * c.kv_heads;
    int64_t       want  = p.row_tiles == 8 && groups >= 384 ? 1 : (512 + groups - 1) / groups;
    const int64_t least = p.row_tiles == 8 ? 4 : 16;
    want                = tiles <= 32 && p.row_tiles < 8 ? 1 : std::min<int64_t>(want, (tiles + least - 1) / least);
    p.splits            = (int)std::max<int64_t>(1, std::min<int64_t>(want, 128));
    return p;
}

size_t workspace_of(const KV4_Cache& c, const KV4_Batch& b, int q_heads, const Plan& p)
{
    if (p.splits <= 1)
        return 0;
    const size_t rows = (size_t)p.splits * b.total_tokens * q_heads;
    return rows * (c.head_dim + 2) * sizeof(float);
}

int check_heads(const KV4_Cache* c, int q_heads)
{
    if (q_heads < 1 || q_heads % c->kv_heads != 0)
        return refuse("%d query heads over %d key/value heads", q_heads, c->kv_heads);
    return 0;
}

template <int D>
int run(hipStream_t stream, const Plan& p, const AttentionArgs& a)
{
    const dim3 grid((unsigned)p.blocks * a.kv_heads, (unsigned)p.splits, 1), block(kWave * kWaves, 1, 1);
    int        err;
    if (p.row_tiles == 1)
        err = launch(p.once ? kv4_attention<D, 1, true> : kv4_attention<D, 1, false>, grid, block, stream, a);
    else if constexpr (D < 256)
        err = launch(p.row_tiles == 8 ? kv4_attention_rows<D, 4> : (p.once ? kv4_attention<D, 2, true> : kv4_attention<D, 2, false>),
                     grid, block, stream, a);
    else
        return (int)hipErrorInvalidValue; // plan_of gives heads of 256 one row tile: two would not fit the registers
    if (err != 0 || p.splits == 1)
        return err;
    int lanes = 1;
    while (lanes < a.splits && 2 * lanes * (D / 8) <= 256)
        lanes *= 2;
    const int64_t per = 256 / (lanes * (D / 8)), all = (int64_t)a.tokens * a.q_heads;
    return launch(kv4_attention_join<D>, dim3((unsigned)((all + per - 1) / per), 1, 1), dim3(256, 1, 1), stream, a, lanes);
}

} // namespace
} // namespace decode

using namespace decode;

extern "C" size_t KV4_AttentionWorkspaceBytes(const KV4_Cache* cache, const KV4_Batch* batch, int q_heads, int window,
                                              int max_len)
{
    if (cache == nullptr || batch == nullptr || cache->kv_heads < 1 || q_heads < 1 || q_heads % cache->kv_heads != 0 ||
        batch->batch < 1 || batch->total_tokens < 1)
        return 0;
    return workspace_of(*cache, *batch, q_heads, plan_of(*cache, *batch, q_heads, window, max_len));
}

extern "C" int KV4_Attention(hipStream_t stream, const KV4_Cache* cache, const KV4_Batch* batch, KV4_Rows q, int q_heads,
                             void* out, float* lse, float scale, int window, int max_len, void* workspace,
                             size_t workspace_bytes, int dtype)
{
    if (int e = check_cache(cache))
        return e;
    if (int e = check_batch(batch, cache))
        return e;
    if (int e = check_heads(cache, q_heads))
        return e;
    if (dtype != DECODE_FP16 && dtype != DECODE_BF16)
        return refuse("unknown element type %d", dtype);
    if (window < 0 || max_len < 0 || !(scale == scale))
        return refuse("window %d, max_len %d, scale %f", window, max_len, (double)scale);
    if (batch->total_tokens == 0)
        return 0;
    // one that holds the whole table hides nothing; with the others a token before its sequence's start keeps place - window + 1 within
    // 32 bits
    const bool whole = window >= (int64_t)batch->table_width * cache->page_size;
    if (!whole && window > 0x7fffffff - batch->total_tokens)
        return refuse("a window of %d with %d tokens", window, batch->total_tokens);
    if (bad_pointer(q.data, 16) || bad_pointer(out, 16) || (lse != nullptr && bad_pointer(lse, 4)) ||
        (batch->total_tokens > 1 && q.token_stride % 8 != 0) || (q_heads > 1 && q.head_stride % 8 != 0))
        return refuse("a null or misaligned q, out or lse (16 bytes, strides multiples of 8 elements)");
    const Plan p = plan_of(*cache, *batch, q_heads, window, max_len);
    if (p.blocks * cache->kv_heads > 0x7fffffff || (int64_t)batch->total_tokens * q_heads > 0x7fffffff)
        return refuse("%d tokens of %d heads: the grid is too large", batch->total_tokens, q_heads);
    const size_t need = workspace_of(*cache, *batch, q_heads, p);
    if (need > 0 && (bad_pointer(workspace, 16) || workspace_bytes < need))
        return refuse("workspace of %zu bytes (16-byte aligned), %zu needed", workspace == nullptr ? (size_t)0 : workspace_bytes, need);
    AttentionArgs a{};
    a.k_codes = static_cast<const uint8_t*>(cache->k_codes), a.v_codes = static_cast<const uint8_t*>(cache->v_codes);
    a.k_words = cache->k_words, a.v_words = cache->v_words;
    a.table = batch->block_table, a.lens = batch->seq_lens, a.cu = batch->cu_tokens;
    a.q = static_cast<const uint16_t*>(q.data), a.q_token = q.token_stride, a.q_head = q.head_stride;
    a.out = static_cast<uint16_t*>(out), a.lse = lse;
    a.part_o     = static_cast<float*>(workspace);
    a.part_ml    = a.part_o + (size_t)p.splits * batch->total_tokens * q_heads * cache->head_dim;
    a.scale_log2 = scale * 1.44269504088896341f;
    a.num_pages = cache->num_pages, a.page_log2 = __builtin_ctz((unsigned)cache->page_size);
    a.kv_heads = cache->kv_heads, a.q_heads = q_heads, a.share = q_heads / cache->kv_heads;
    a.batch = batch->batch, a.width = batch->table_width, a.stride = batch->table_stride, a.tokens = batch->total_tokens;
    a.window = whole ? 0 : window, a.splits = p.splits, a.bf16 = dtype == DECODE_BF16;
    switch (cache->head_dim) {
    case 64: return run<64>(stream, p, a);
    case 96: return run<96>(stream, p, a);
    case 128: return run<128>(stream, p, a);
    default: return run<256>(stream, p, a);
    }
}
