// Writing and reading the paged 4-bit key/value cache: KV4_Append, KV4_Gather (decode_api.h holds the format).
#include "decode_common.hiph"

// Every product, sum and quotient below is rounded by itself: the codes are then the same wherever they are computed.
#pragma clang fp contract(off)

namespace decode {

struct CacheView {
    uint8_t* codes[2]; // keys, values
    int32_t* words[2];
    int      num_pages, page_size, kv_heads, head_dim;
};

struct BatchView {
    const int *table, *lens, *cu;
    int        batch, width, stride, tokens;
};

struct AppendArgs {
    CacheView       cache;
    BatchView       batch;
    const uint16_t* src[3]; // k, v, q
    int64_t         token_stride[3], head_stride[3];
    uint16_t*       q_out;
    const float*    rot;
    const int*      positions;
    int             q_heads, rot_rows, rot_dims, interleaved, bf16;
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
    const int idx = pos / c.page_size; // a power of two, but a division once per vector costs nothing here
    if (idx >= b.width)
        return -1;
    const int page = b.table[(int64_t)s * b.stride + idx];
    if (page < 0 || page >= c.num_pages)
        return -1;
    slot = pos & (c.page_size - 1);
    return page;
}

__device__ __forceinline__ void load8(const uint16_t* p, bool wide, bool bf16, float (&x)[8])
{
    uint16_t raw[8];
    if (wide) {
        const uintx4 v = *reinterpret_cast<const uintx4*>(p);
        __builtin_memcpy(raw, &v, 16);
    } else {
        for (int i = 0; i < 8; ++i)
            raw[i] = p[i];
    }
    for (int i = 0; i < 8; ++i)
        x[i] = from16(raw[i], bf16);
}

// Rotates elements d0 .. d0+7 (in x) of the head at `row`.
__device__ __forceinline__ void rotate8(const AppendArgs& a, const uint16_t* row, bool wide, int d0, int pos, float (&x)[8])
{
    const int half = a.rot_dims >> 1;
    if (d0 >= a.rot_dims)
        return;
    const bool   inside = pos >= 0 && pos < a.rot_rows;
    const float* tab    = a.rot + (int64_t)(inside ? pos : 0) * a.rot_dims;
    const float  nan    = __uint_as_float(0x7fc00000u);
    if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            if (d0 + i < a.rot_dims) {
                const float c = inside ? tab[(d0 + i) >> 1] : nan, s = inside ? tab[half + ((d0 + i) >> 1)] : nan;
                const float u = x[i], v = x[i + 1];
                x[i]     = u * c - v * s;
                x[i + 1] = v * c + u * s;
            }
        }
        return;
    }
    float other[8];
    if ((half & 7) == 0) { // all eight on one side: the partners are eight neighbours too
        load8(row + (d0 < half ? d0 + half : d0 - half), wide, a.bf16, other);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = d0 + i, p = d < half ? d + half : d - half;
            other[i]    = d < a.rot_dims ? from16(row[p], a.bf16) : 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = d0 + i;
        if (d < a.rot_dims) {
            const bool  low = d < half;
            const int   j   = low ? d : d - half;
            const float c = inside ? tab[j] : nan, s = inside ? tab[half + j] : nan;
            x[i] = low ? x[i] * c - other[i] * s : x[i] * c + other[i] * s;
        }
    }
}

// One group of L lanes (8 elements each; L = 8, 16 or 32) per head vector: keys, values, then queries of a token.  A key or
// value is read once, rotated and encoded in registers (the extremes pass between the group's lanes) and written as one
// dword of codes per lane.
template <int L>
__global__ __launch_bounds__(256) void kv4_append(AppendArgs a, int heads)
{
    const int lane = threadIdx.x & (L - 1), d0 = lane * 8;
    const int unit = blockIdx.y * (256 / L) + threadIdx.x / L;
    const int t    = blockIdx.x;
    if (unit >= heads)
        return; // whole groups
    const bool live = d0 < a.cache.head_dim; // heads of 96 leave four lanes of sixteen idle: they exchange zeros below
    const int side = unit < a.cache.kv_heads ? 0 : (unit < 2 * a.cache.kv_heads ? 1 : 2);
    const int head = unit - side * a.cache.kv_heads;
    int       slot, place;
    const int page = locate(a.cache, a.batch, t, slot, place);
    if (side < 2 && page < 0)
        return;
    const uint16_t* row  = a.src[side] + t * a.token_stride[side] + head * a.head_stride[side];
    const bool      wide = (a.wide >> side) & 1;
    float           x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live)
        load8(row + d0, wide, a.bf16, x);
    if (live && side != 1 && a.rot_dims > 0) {
        if (a.positions != nullptr)
            rotate8(a, row, wide, d0, a.positions[t], x);
        else if (place >= 0)
            rotate8(a, row, wide, d0, place, x);
    }
    if (side == 2) {
        if (!live)
            return;
        uint16_t out[8];
        for (int i = 0; i < 8; ++i)
            out[i] = to16(x[i], a.bf16);
        uintx4 v;
        __builtin_memcpy(&v, out, 16);
        *reinterpret_cast<uintx4*>(a.q_out + ((int64_t)t * a.q_heads + head) * a.cache.head_dim + d0) = v;
        return;
    }
    float hi = 0.f, lo = 0.f;
    int   bad = 0;
    for (int i = 0; i < 8; ++i) {
        hi = fmaxf(hi, x[i]);
        lo = fminf(lo, x[i]);
        bad |= (__float_as_uint(x[i]) & 0x7f800000u) == 0x7f800000u;
    }
#pragma unroll
    for (int m = 1; m < L; m <<= 1) {
        hi = fmaxf(hi, __shfl_xor(hi, m, L));
        lo = fminf(lo, __shfl_xor(lo, m, L));
        bad |= __shfl_xor(bad, m, L);
    }
    const float fifteenth = 1.0f / 15.0f;
    const float s         = hi * fifteenth - lo * fifteenth;
    unsigned    word      = (__float_as_uint(s) + 8u) & ~15u;
    if (s < 0x1p-100f)
        word = 0x3f800000u;
    const float z    = fminf(fmaxf(rintf(-lo * (1.0f / __uint_as_float(word))), 0.f), 15.f);
    word |= (unsigned)z;
    const float inv   = 1.0f / __uint_as_float(word);
    unsigned    codes = 0;
    for (int i = 0; i < 8; ++i) {
        const float q = fminf(fmaxf(rintf(x[i] * inv) + z, 0.f), 15.f);
        codes |= (unsigned)q << (4 * i);
    }
    if (bad) {
        word  = 0x7fc00000u;
        codes = 0;
    }
    if (!live)
        return;
    const int64_t at = ((int64_t)page * a.cache.kv_heads + head) * a.cache.page_size + slot;
    *reinterpret_cast<unsigned*>(a.cache.codes[side] + at * (a.cache.head_dim / 2) + lane * 4) = codes;
    if (lane == 0)
        a.cache.words[side][at] = (int)word;
}

struct GatherArgs {
    CacheView cache;
    BatchView batch;
    uint16_t* dst[2];
    int       bf16;
};

template <int L>
__global__ __launch_bounds__(256) void kv4_gather(GatherArgs a)
{
    const int lane = threadIdx.x & (L - 1), d0 = lane * 8;
    const int unit = blockIdx.y * (256 / L) + threadIdx.x / L;
    const int t    = blockIdx.x;
    if (unit >= 2 * a.cache.kv_heads || d0 >= a.cache.head_dim)
        return;
    const int side = unit < a.cache.kv_heads ? 0 : 1, head = unit - side * a.cache.kv_heads;
    if (a.dst[side] == nullptr)
        return;
    int       slot, place;
    const int page = locate(a.cache, a.batch, t, slot, place);
    uint16_t  out[8];
    for (int i = 0; i < 8; ++i)
        out[i] = 0;
    if (page >= 0) {
        const int64_t  at    = ((int64_t)page * a.cache.kv_heads + head) * a.cache.page_size + slot;
        const unsigned codes = *reinterpret_cast<const unsigned*>(a.cache.codes[side] + at * (a.cache.head_dim / 2) + lane * 4);
        const unsigned word  = (unsigned)a.cache.words[side][at];
        const int      z     = word & 15;
        for (int i = 0; i < 8; ++i)
            out[i] = to16(__uint_as_float(word) * (float)((int)((codes >> (4 * i)) & 15) - z), a.bf16);
    }
    uintx4 v;
    __builtin_memcpy(&v, out, 16);
    *reinterpret_cast<uintx4*>(a.dst[side] + ((int64_t)t * a.cache.kv_heads + head) * a.cache.head_dim + d0) = v;
}

namespace {

CacheView view(const KV4_Cache& c)
{
    return {{static_cast<uint8_t*>(c.k_codes), static_cast<uint8_t*>(c.v_codes)},
            {c.k_words, c.v_words},
            c.num_pages,
            c.page_size,
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
    }
    if (q.data != nullptr && rotary == nullptr)
        return refuse("queries are given and no rotation");
    if (q.data != nullptr && (q_heads < 1 || q_heads > 65536 || bad_pointer(q_out, 16)))
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
    dim3      grid((unsigned)batch->total_tokens, (unsigned)((heads + per - 1) / per), 1);
    auto      kernel = L == 8 ? kv4_append<8> : (L == 16 ? kv4_append<16> : kv4_append<32>);
    return launch(kernel, grid, dim3(256, 1, 1), stream, a, heads);
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
    dim3       grid((unsigned)batch->total_tokens, (unsigned)((2 * cache->kv_heads + per - 1) / per), 1);
    auto       kernel = L == 8 ? kv4_gather<8> : (L == 16 ? kv4_gather<16> : kv4_gather<32>);
    return launch(kernel, grid, dim3(256, 1, 1), stream, a);
}
