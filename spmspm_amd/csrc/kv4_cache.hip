// Writing and reading the paged 4-bit key/value cache: KV4_Append, KV4_Gather (decode_api.h holds the format).
#include "decode_common.hiph"

#include <algorithm>

// Every product, sum and quotient below is rounded by itself: the codes are then the same wherever they are computed.
#pragma clang fp contract(off)

namespace decode {

struct CacheView {
    uint8_t* codes[2]; // keys, values
    int32_t* words[2];
    int      num_pages, page_log2, kv_heads, head_dim;
};

struct BatchView {
    const int *table, *lens, *cu;
    int        batch, width, stride, tokens;
};

// The largest of L lanes' values (at least 0), in all of them.
template <int PATTERN>
__device__ __forceinline__ float across(float v)
{
    return __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), PATTERN, 0xf, 0xf, true));
}
template <int L>
__device__ __forceinline__ float group_max(float v)
{
    v = fmaxf(v, across<0xb1>(v));  // neighbours
    v = fmaxf(v, across<0x4e>(v));  // pairs of a quad
    v = fmaxf(v, across<0x141>(v)); // quads of eight, mirrored
    if constexpr (L >= 16)
        v = fmaxf(v, across<0x140>(v)); // eights of sixteen, mirrored
    if constexpr (L == 32)
        v = fmaxf(v, __shfl_xor(v, 16, 32));
    return v;
}

struct AppendArgs {
    CacheView       cache;
    BatchView       batch;
    const uint16_t* src[3]; // k, v, q
    int64_t         token_stride[3], head_stride[3];
    uint16_t*       q_out;
    const float*    rot;
    const int*      positions;
    int             q_heads, rot_rows, rot_dims, interleaved, bf16;
    int             rot_quads; // the rotation's rows can be read 16 bytes at a time
    int             wide; // bit s: src[s] can be read 16 bytes at a time
};

// Place of row t in its sequence: page (or -1) and slot; `place` is the position, negative where there is none.
__device__ __forceinline__ int locate(const CacheView& c, const BatchView& b, int t, int& slot, int& place)
{
    int       first, count;
    const int s = sequence_of(t, b.cu, b.batch, first, count);
    place       = -1;
    slot        = 0;
    if (s < 0)
        return -1;
    const int pos = b.lens[s] - count + (t - first);
    if (pos < 0)
        return -1;
    place         = pos;
    const int idx = pos >> c.page_log2;
    if (idx >= b.width)
        return -1;
    const int page = b.table[(int64_t)s * b.stride + idx];
    if (page < 0 || page >= c.num_pages)
        return -1;
    slot = pos & ((1 << c.page_log2) - 1);
    return page;
}

// Eight 16-bit elements, one by one where they are not aligned.
__device__ __forceinline__ uintx4 load8(const uint16_t* p, bool wide)
{
    if (wide)
        return *reinterpret_cast<const uintx4*>(p);
    uint16_t raw[8];
    for (int i = 0; i < 8; ++i)
        raw[i] = p[i];
    uintx4 v;
    __builtin_memcpy(&v, raw, 16);
    return v;
}

__device__ __forceinline__ float element(const uintx4& v, int i, bool bf16)
{
    return from16((uint16_t)(v[i >> 1] >> (16 * (i & 1))), bf16);
}

// A group of L lanes (8 elements each; L = 8, 16 or 32) works for one token, the groups of a workgroup for tokens in a row,
// and takes `per` of its vectors one after the other: keys, values, then queries.  A vector is read once, rotated and encoded
// in registers (its extremes pass between the group's lanes) and written as one dword of codes per lane.  Tokens in a row lie
// side by side in a page, so that a workgroup writes whole lines of codes and words; with a workgroup for each token, codes
// and above all single words went to memory as parts of lines (14247 tokens, 8 key/value and 32 query heads of 128, 307 MB:
// 105 us; 80 now, 3.8 TB/s of reads and writes mixed).  The lane's part of the rotation's row is read once for all of the token's vectors.
template <int L>
__global__ __launch_bounds__(256) void kv4_append(AppendArgs a, int heads, int per)
{
    constexpr int kGroups = 256 / L;
    const int     lane = threadIdx.x & (L - 1), d0 = lane * 8, D = a.cache.head_dim;
    const int     t    = blockIdx.x * kGroups + threadIdx.x / L;
    const bool    live = d0 < D; // heads of 96 leave four lanes of sixteen idle: they exchange zeros below
    const int     first = blockIdx.y * per, last = min(heads, first + per);
    const int     kvh = a.cache.kv_heads, half = a.rot_dims >> 1;
    const bool    together = (half & 7) == 0; // the partners of eight elements are eight elements in a row
    if (t >= a.batch.tokens)
        return; // whole groups

    // a vector's elements, and those `half` away that they are rotated with
    auto source = [&](int unit) {
        const int side = unit < kvh ? 0 : (unit < 2 * kvh ? 1 : 2);
        return a.src[side] + t * a.token_stride[side] + (unit - side * kvh) * a.head_stride[side];
    };
    auto is_wide = [&](int unit) { return ((a.wide >> (unit < kvh ? 0 : (unit < 2 * kvh ? 1 : 2))) & 1) != 0; };
    auto partner = [&](int unit) {
        return together && !a.interleaved && d0 < a.rot_dims ? load8(source(unit) + (d0 < half ? d0 + half : d0 - half), is_wide(unit))
                                                             : uintx4{0, 0, 0, 0};
    };
    uintx4 raw{0, 0, 0, 0}, beside{0, 0, 0, 0};
    if (live && first < last) { // on their way before the token's place is known
        raw    = load8(source(first) + d0, is_wide(first));
        beside = partner(first);
    }
    int       slot, place;
    const int page = locate(a.cache, a.batch, t, slot, place);

    // what an element is multiplied by, and what its partner is before it is added
    const int  row  = a.positions != nullptr ? a.positions[t] : place;
    const bool turn = live && d0 < a.rot_dims && (a.positions != nullptr || place >= 0);
    float      own[8], other[8];
    if (turn) {
        const bool   inside = row >= 0 && row < a.rot_rows;
        const float* tab    = a.rot + (int64_t)(inside ? row : 0) * a.rot_dims;
        if (a.rot_quads) {
            if (a.interleaved) {
                const floatx4 c = *reinterpret_cast<const floatx4*>(tab + (d0 >> 1)), s = *reinterpret_cast<const floatx4*>(tab + half + (d0 >> 1));
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    own[i] = c[i >> 1], other[i] = (i & 1) ? s[i >> 1] : -s[i >> 1];
            } else {
                const bool   low = d0 < half;
                const float* at  = tab + (low ? d0 : d0 - half);
                floatx4      c[2], s[2];
                c[0] = *reinterpret_cast<const floatx4*>(at), c[1] = *reinterpret_cast<const floatx4*>(at + 4);
                s[0] = *reinterpret_cast<const floatx4*>(at + half), s[1] = *reinterpret_cast<const floatx4*>(at + half + 4);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    own[i] = c[i >> 2][i & 3], other[i] = low ? -s[i >> 2][i & 3] : s[i >> 2][i & 3]; // a + (-b) is a - b
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int  d = min(d0 + i, a.rot_dims - 1);
                const bool low = a.interleaved ? (i & 1) == 0 : d < half;
                const int  j = a.interleaved ? d >> 1 : (low ? d : d - half);
                own[i]   = tab[j];
                other[i] = low ? -tab[half + j] : tab[half + j];
            }
        }
        if (!inside) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                own[i] = other[i] = __uint_as_float(0x7fc00000u);
        }
    }
    for (int unit = first; unit < last; ++unit) {
        const int    side = unit < kvh ? 0 : (unit < 2 * kvh ? 1 : 2), head = unit - side * kvh;
        const uintx4 mine = raw, theirs = beside;
        if (live && unit + 1 < last) {
            raw    = load8(source(unit + 1) + d0, is_wide(unit + 1));
            beside = partner(unit + 1);
        }
        if (side < 2 && page < 0)
            continue; // the whole group
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = element(mine, i, a.bf16);
        if (turn && side != 1) {
            float y[8];
            if (a.interleaved) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    y[i] = x[i ^ 1];
            } else if (together) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    y[i] = element(theirs, i, a.bf16);
            } else {
                const uint16_t* src = source(unit);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int d = min(d0 + i, a.rot_dims - 1);
                    y[i]        = from16(src[d < half ? d + half : d - half], a.bf16);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[i] = d0 + i < a.rot_dims ? x[i] * own[i] + y[i] * other[i] : x[i];
        }
        if (side == 2) {
            uint16_t out[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                out[i] = to16(x[i], a.bf16);
            uintx4 v;
            __builtin_memcpy(&v, out, 16);
            if (live)
                *reinterpret_cast<uintx4*>(a.q_out + ((int64_t)t * a.q_heads + head) * D + d0) = v;
            continue;
        }
        float hi = 0.f, lo = 0.f, none = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            hi = __builtin_fmaxf(hi, x[i]);
            lo = __builtin_fminf(lo, x[i]);
            none = __builtin_fmaf(x[i], 0.f, none); // NaN with an infinity or a NaN
        }
        hi = none == 0.f ? hi : __builtin_inff();
        hi = group_max<L>(hi);
        lo = -group_max<L>(-lo);
        const bool  bad       = !(hi < __builtin_inff());
        const float fifteenth = 1.0f / 15.0f;
        const float s         = hi * fifteenth - lo * fifteenth;
        unsigned    word      = (__float_as_uint(s) + 8u) & ~15u;
        if (s < 0x1p-100f)
            word = 0x3f800000u;
        const float z = fminf(fmaxf(rintf(-lo * (1.0f / __uint_as_float(word))), 0.f), 15.f);
        word |= (unsigned)z;
        const float inv   = 1.0f / __uint_as_float(word);
        unsigned    codes = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float q = __builtin_amdgcn_fmed3f(rintf(x[i] * inv) + z, 0.f, 15.f);
            codes |= (unsigned)q << (4 * i);
        }
        if (bad) {
            word  = 0x7fc00000u;
            codes = 0;
        }
        const int64_t at = ((((int64_t)page * kvh + head)) << a.cache.page_log2) + slot;
        if (live)
            *reinterpret_cast<unsigned*>(a.cache.codes[side] + at * (D / 2) + lane * 4) = codes;
        if (lane == 0)
            a.cache.words[side][at] = (int)word;
    }
}

struct GatherArgs {
    CacheView cache;
    BatchView batch;
    uint16_t* dst[2];
    int       bf16;
};

// As kv4_append deals tokens: a lane reads one dword of codes and writes the 8 elements that it holds.  Bound by its writes:
// 14247 tokens, 8 key/value heads of 128, 74 MB in 20 us, 3.7 TB/s; a few tokens take 2.7 us, a launch.
template <int L>
__global__ __launch_bounds__(256) void kv4_gather(GatherArgs a, int per)
{
    constexpr int kGroups = 256 / L;
    const int     lane = threadIdx.x & (L - 1), d0 = lane * 8, D = a.cache.head_dim, kvh = a.cache.kv_heads;
    const int     t    = blockIdx.x * kGroups + threadIdx.x / L;
    const int     first = blockIdx.y * per, last = min(2 * kvh, first + per);
    if (t >= a.batch.tokens || d0 >= D)
        return;
    int       slot, place;
    const int page = locate(a.cache, a.batch, t, slot, place);
    for (int unit = first; unit < last; ++unit) {
        const int side = unit < kvh ? 0 : 1, head = unit - side * kvh;
        if (a.dst[side] == nullptr)
            continue;
        uint16_t out[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (page >= 0) {
            const int64_t  at    = (((int64_t)page * kvh + head) << a.cache.page_log2) + slot;
            const unsigned codes = *reinterpret_cast<const unsigned*>(a.cache.codes[side] + at * (D / 2) + lane * 4);
            const unsigned word  = (unsigned)a.cache.words[side][at];
            const int      z     = word & 15;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                out[i] = to16(__uint_as_float(word) * (float)((int)((codes >> (4 * i)) & 15) - z), a.bf16);
        }
        uintx4 v;
        __builtin_memcpy(&v, out, 16);
        *reinterpret_cast<uintx4*>(a.dst[side] + ((int64_t)t * kvh + head) * D + d0) = v;
    }
}

namespace {

CacheView view(const KV4_Cache& c)
{
    return {{static_cast<uint8_t*>(c.k_codes), static_cast<uint8_t*>(c.v_codes)},
            {c.k_words, c.v_words},
            c.num_pages,
            __builtin_ctz((unsigned)c.page_size),
            c.kv_heads,
            c.head_dim};
}

BatchView view(const KV4_Batch& b)
{
    return {b.block_table, b.seq_lens, b.cu_tokens, b.batch, b.table_width, b.table_stride, b.total_tokens};
}

int lanes_of(int head_dim)
{
    return head_dim == 64 ? 8 : (head_dim == 256 ? 32 : 16);
}

// Head vectors a group of lanes takes one after the other: more than one, so that a token's place and its row of the rotation
// are looked up less often, once that leaves 2048 workgroups.
int vectors_per_group(int heads, int64_t blocks)
{
    return (int)std::max<int64_t>(1, std::min<int64_t>(heads, heads * blocks / 2048));
}

int check_dtype(int dtype)
{
    return dtype == DECODE_FP16 || dtype == DECODE_BF16 ? 0 : refuse("unknown element type %d", dtype);
}

} // namespace
} // namespace decode

using namespace decode;

extern "C" int KV4_Append(hipStream_t stream, const KV4_Cache* cache, const KV4_Batch* batch, KV4_Rows k, KV4_Rows v,
                          KV4_Rows q, int q_heads, void* q_out, const KV4_Rotary* rotary, int dtype)
{
    if (int e = check_cache(cache))
        return e;
    if (int e = check_batch(batch, cache))
        return e;
    if (int e = check_dtype(dtype))
        return e;
    AppendArgs a{};
    a.cache = view(*cache);
    a.batch = view(*batch);
    if (rotary != nullptr) {
        if (rotary->dims < 0 || rotary->dims > cache->head_dim || (rotary->dims & 1))
            return refuse("%d rotated elements of a head of %d", rotary->dims, cache->head_dim);
        if (rotary->dims > 0 && (bad_pointer(rotary->table, 4) || rotary->table_rows < 1 ||
                                 (rotary->positions != nullptr && bad_pointer(rotary->positions, 4))))
            return refuse("a null, misaligned or empty rotation table");
        a.rot         = rotary->table;
        a.positions   = rotary->positions;
        a.rot_rows    = rotary->table_rows;
        a.rot_dims    = rotary->dims;
        a.interleaved = rotary->interleaved != 0;
        a.rot_quads   = rotary->dims % 16 == 0 && !bad_pointer(rotary->table, 16);
    }
    if (q.data != nullptr && rotary == nullptr)
        return refuse("queries are given and no rotation");
    if (q.data != nullptr && (q_heads < 1 || q_heads > 32768 || bad_pointer(q_out, 16)))
        return refuse("%d query heads, or a null or misaligned q_out (16 bytes)", q_heads);
    if (batch->total_tokens == 0)
        return 0;
    const KV4_Rows* src[3] = {&k, &v, &q};
    for (int s = 0; s < 3; ++s) {
        if (s == 2 && q.data == nullptr)
            break;
        if (bad_pointer(src[s]->data, 2))
            return refuse("a null or misaligned k, v or q");
        a.src[s]          = static_cast<const uint16_t*>(src[s]->data);
        a.token_stride[s] = src[s]->token_stride;
        a.head_stride[s]  = src[s]->head_stride;
        if (!bad_pointer(src[s]->data, 16) && src[s]->token_stride % 8 == 0 && src[s]->head_stride % 8 == 0)
            a.wide |= 1 << s;
    }
    a.q_out         = static_cast<uint16_t*>(q_out);
    a.q_heads       = q_heads;
    a.bf16          = dtype == DECODE_BF16;
    const int heads = 2 * cache->kv_heads + (q.data != nullptr ? q_heads : 0);
    const int L     = lanes_of(cache->head_dim), per = 256 / L;
    const unsigned blocks = (unsigned)((batch->total_tokens + per - 1) / per);
    const int      each   = vectors_per_group(heads, blocks);
    dim3      grid(blocks, (unsigned)((heads + each - 1) / each), 1);
    auto      kernel = L == 8 ? kv4_append<8> : (L == 16 ? kv4_append<16> : kv4_append<32>);
    return launch(kernel, grid, dim3(256, 1, 1), stream, a, heads, each);
}

extern "C" int KV4_Gather(hipStream_t stream, const KV4_Cache* cache, const KV4_Batch* batch, void* k, void* v, int dtype)
{
    if (int e = check_cache(cache))
        return e;
    if (int e = check_batch(batch, cache))
        return e;
    if (int e = check_dtype(dtype))
        return e;
    if ((k != nullptr && bad_pointer(k, 16)) || (v != nullptr && bad_pointer(v, 16)))
        return refuse("a misaligned output (16 bytes)");
    if (batch->total_tokens == 0 || (k == nullptr && v == nullptr))
        return 0;
    GatherArgs a{view(*cache), view(*batch), {static_cast<uint16_t*>(k), static_cast<uint16_t*>(v)}, dtype == DECODE_BF16};
    const int  L = lanes_of(cache->head_dim), per = 256 / L;
    const unsigned blocks = (unsigned)((batch->total_tokens + per - 1) / per);
    const int      each   = vectors_per_group(2 * cache->kv_heads, blocks);
    dim3       grid(blocks, (unsigned)((2 * cache->kv_heads + each - 1) / each), 1);
    auto       kernel = L == 8 ? kv4_gather<8> : (L == 16 ? kv4_gather<16> : kv4_gather<32>);
    return launch(kernel, grid, dim3(256, 1, 1), stream, a, each);
}
