// Quantisation into 4 bits and back: keys and values as they enter the pages of a cache, weights once when they are loaded (format and layout:
// int4.cuh).
//
// Eight lanes take 64 neighbouring channels of a token's head, 8 a lane (a word of a key's codes): a group's extremes are found with shuffles.  A
// weight's quantisation gives a lane 4 columns.  Bound by the launch and by four loads that wait for one another (position, request, its slot, its
// page) for single tokens (2.7 us of the GPU's time), by the instructions - some 60 a value by the
// counters - for whole prompts (2,048 tokens of 8 heads of 128: written in 8.2 us, read back in 4.6).
#include "int4.cuh"

namespace {

struct CacheArgs {
    const void *k, *v;             // rows as given: [T, nkv, d], strides below (kv_read writes them)
    unsigned char* pages;          // [num_pages, nkv, page_size / 16, tile]
    const int *positions, *seq_of_token, *seq_slot, *block_table;
    int* status;
    long long k_token, k_head, v_token, v_head;      // strides in elements
    int T, nkv, d, group, page_size, max_pages, num_pages, vec;
};

template <typename T>
__device__ __forceinline__ void load4(const T* p, bool vec, float (&x)[4]) {
    if (vec) {
        const float4 v = ce_load4(p);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = CeType<T>::load(p + i);
    }
}
__device__ __forceinline__ void store4(float* p, bool vec, const float (&x)[4]) {
    if (vec) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    else
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = x[i];
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, bool vec, const float (&x)[4]) {
    __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
    if (vec) *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
    else { p[0] = a.x; p[1] = a.y; p[2] = b.x; p[3] = b.y; }
}

__device__ __forceinline__ void load8(const float* p, bool vec, float (&x)[8]) {
    float a[4], b[4];
    load4(p, vec, a);
    load4(p + 4, vec, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[i + 4] = b[i]; }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, bool vec, float (&x)[8]) {
    uint32_t w[4];
    if (vec) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else {
        const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = q[2 * i] | (uint32_t)q[2 * i + 1] << 16;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void store8(float* p, bool vec, const float (&x)[8]) {
    const float a[4] = {x[0], x[1], x[2], x[3]}, b[4] = {x[4], x[5], x[6], x[7]};
    store4(p, vec, a);
    store4(p + 4, vec, b);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, bool vec, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    if (vec) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else {
        unsigned short* q = reinterpret_cast<unsigned short*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = (unsigned short)(w[i >> 1] >> (i & 1 ? 16 : 0));
    }
}

// (s, z) of this lane's group and its four codes as 16 bits; ``lanes``: lanes of a group (8, 16 or 32)
__device__ __forceinline__ unsigned quantise4(const float (&x)[4], int lanes, __half2& sz) {
    float lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    bool ok = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) ok = ok && fabsf(x[i]) <= I4_LIMIT;
    for (int o = lanes >> 1; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        ok = __shfl_xor_sync(0xffffffffu, (int)ok, o) && ok;
    }
    sz = i4_step(lo, hi, ok);
    const float s = __low2float(sz), z = __high2float(sz), inv = ok ? i4_inverse(s) : 0.0f;
    unsigned q = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) q |= (inv > 0.0f ? i4_code(x[i], s, z, inv) : 0u) << (4 * i);
    return q;
}

// The tile of a token's position; null (and a status) where its request holds no such page.
__device__ __forceinline__ unsigned char* tile_of(const CacheArgs& a, int t, int h, int& slot_in_tile, int code) {
    const int pos = a.positions[t], pi = pos >= 0 ? pos / a.page_size : -1;
    const int page = pi >= 0 && pi < a.max_pages ? a.block_table[(size_t)a.seq_slot[a.seq_of_token[t]] * a.max_pages + pi] : -1;
    if (page < 0 || page >= a.num_pages) { atomicExch(a.status, code); return nullptr; }
    const int in = pos - pi * a.page_size;
    slot_in_tile = in & 15;
    return a.pages + (((size_t)page * a.nkv + h) * (a.page_size >> 4) + (in >> 4)) * (size_t)i4_cache_tile_bytes(a.d, a.group);
}

// the same for 8 channels a lane; ``lanes`` of a group: 4 or 8
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], int lanes, __half2& sz) {
    float lo = x[0], hi = x[0];
    bool ok = fabsf(x[0]) <= I4_LIMIT;
#pragma unroll
    for (int i = 1; i < 8; ++i) { lo = fminf(lo, x[i]); hi = fmaxf(hi, x[i]); ok = ok && fabsf(x[i]) <= I4_LIMIT; }
    for (int o = lanes >> 1; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        ok = __shfl_xor_sync(0xffffffffu, (int)ok, o) && ok;
    }
    sz = i4_step(lo, hi, ok);
    const float s = __low2float(sz), z = __high2float(sz), inv = ok ? i4_inverse(s) : 0.0f;
    if (!(inv > 0.0f)) return 0u;
    uint32_t q = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) q |= i4_code(x[i], s, z, inv) << (4 * i);
    return q;
}

// A thread's place: token t, head h, block b of 64 channels, i: its 8 of them.  It takes the key's and the value's (one search for the page).
struct Place {
    int t, h, b, i, channel;
    bool live;
};
__device__ __forceinline__ Place place(const CacheArgs& a) {
    const unsigned blocks = (unsigned)a.d >> 6, u = blockIdx.x * 32 + (threadIdx.x >> 3), t = u / blocks;
    Place p;
    p.live = t < (unsigned)a.T;
    p.t = p.live ? (int)t : a.T - 1;
    p.b = (int)(u - t * blocks);
    p.h = blockIdx.y;
    p.i = threadIdx.x & 7;
    p.channel = 64 * p.b + 8 * p.i;
    return p;
}

template <typename T>
__global__ void __launch_bounds__(256) int4_kv_write_kernel(CacheArgs a) {
    ce_pdl_begin();
    const Place p = place(a);
    float k[8], v[8];
    load8((const T*)a.k + p.t * a.k_token + p.h * a.k_head + p.channel, a.vec, k);
    load8((const T*)a.v + p.t * a.v_token + p.h * a.v_head + p.channel, a.vec, v);
    int at = 0;
    unsigned char* tile = tile_of(a, p.t, p.h, at, 2);
    __half2 k_step, v_step;
    const uint32_t kq = quantise8(k, a.group >> 3, k_step), vq = quantise8(v, a.group >> 3, v_step);
    // a word of values: channels 4 r .. 4 r + 3 of a block and those 32 further on, which lane i ^ 4 has
    const bool low = p.i < 4;
    const uint32_t got = __shfl_xor_sync(0xffffffffu, low ? vq >> 16 : vq & 0xffffu, 4);
    if (!p.live || !tile) return;
    const int groups = a.d / a.group, g = p.channel / a.group;
    *reinterpret_cast<uint32_t*>(tile + i4_k_word(at, p.channel)) = kq;
    *reinterpret_cast<uint32_t*>(tile + i4_v_word(a.d, at, p.b, 2 * (p.i & 3) + (low ? 0 : 1))) = low ? (vq & 0xffffu) | got << 16 : got | (vq >> 16) << 16;
    if (p.channel % a.group == 0) {
        *reinterpret_cast<__half2*>(tile + i4_k_step(a.d, groups, at, g)) = k_step;
        *reinterpret_cast<__half2*>(tile + i4_v_step(a.d, groups, at, g)) = v_step;
    }
}

__device__ __forceinline__ void values_of(uint32_t w, __half2 sz, float (&x)[8]) {
    const float s = __low2float(sz), z = __high2float(sz);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaf((float)((w >> (4 * i)) & 15u), s, z);
}

template <typename T>
__global__ void __launch_bounds__(256) int4_kv_read_kernel(CacheArgs a) {
    ce_pdl_begin();
    const Place p = place(a);
    int at = 0;
    const unsigned char* tile = p.live ? tile_of(a, p.t, p.h, at, 4) : nullptr;
    if (!tile) return;
    const int groups = a.d / a.group, g = p.channel / a.group;
    const uint32_t kq = *reinterpret_cast<const uint32_t*>(tile + i4_k_word(at, p.channel));
    const uint32_t first = *reinterpret_cast<const uint32_t*>(tile + i4_v_word(a.d, at, p.b, 2 * (p.i & 3)));
    const uint32_t second = *reinterpret_cast<const uint32_t*>(tile + i4_v_word(a.d, at, p.b, 2 * (p.i & 3) + 1));
    const __half2 k_step = *reinterpret_cast<const __half2*>(tile + i4_k_step(a.d, groups, at, g));
    const __half2 v_step = *reinterpret_cast<const __half2*>(tile + i4_v_step(a.d, groups, at, g));
    float x[8];
    values_of(kq, k_step, x);
    store8((T*)a.k + p.t * a.k_token + p.h * a.k_head + p.channel, a.vec, x);
    values_of(__byte_perm(first, second, p.i < 4 ? 0x5410u : 0x7632u), v_step, x);
    store8((T*)a.v + p.t * a.v_token + p.h * a.v_head + p.channel, a.vec, x);
}

struct WeightArgs {
    const void* w;                 // [rows, width], row stride ld (quantise reads it, dequantise writes it)
    unsigned char* tiles;          // [row tiles, ceil(width / 64), tile]
    long long ld;
    int rows, gated, width, kblocks, group, vec;
};
// a warp takes 128 neighbouring columns of one row of a tile: rows of padding, and columns beyond the width, hold zeros
template <typename T>
__global__ void __launch_bounds__(256) int4_quantise_weight_kernel(WeightArgs a) {
    ce_pdl_begin();
    const int lane = threadIdx.x & 31, pairs = (a.kblocks + 1) >> 1, kept = min(a.group, 64);
    const long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int padded = (int)(u / pairs), col = (int)(u - (long long)padded * pairs) * 128 + 4 * lane, tile_no = padded >> 4, in = padded & 15;
    const int part = a.gated ? a.rows >> 1 : a.rows, n = a.gated ? tile_no * 8 + (in & 7) : padded;
    if (tile_no * (a.gated ? 8 : 16) >= part) return;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (n < part && col < a.width) load4((const T*)a.w + (n + (a.gated && in >= 8 ? (long long)part : 0)) * a.ld + col, a.vec, x);
    __half2 sz;
    const unsigned q = quantise4(x, a.group >> 2, sz);
    const unsigned near = __shfl_xor_sync(0xffffffffu, q, 1);
    const int kb = col >> 6;
    if (kb >= a.kblocks) return;
    unsigned char* tile = a.tiles + ((size_t)tile_no * a.kblocks + kb) * i4_weight_tile_bytes(kept);
    if (!(lane & 1)) *reinterpret_cast<uint32_t*>(tile + i4_k_word(in, col & 63)) = q | near << 16;
    if ((4 * lane) % kept == 0) *reinterpret_cast<__half2*>(tile + 512 + (in * (64 / kept) + (col & 63) / kept) * 4) = sz;
}

// Runs behind a kernel that writes a weight, launched the ordinary way, and so begins when that has ended: from here on, no kernel that starts
// early beside the one before it can meet a weight that is still being written.
__global__ void int4_weight_done_kernel() {}

// a warp takes a tile: a lane the words of two rows, 8 columns of either half each
template <typename T>
__global__ void __launch_bounds__(256) int4_dequantise_weight_kernel(WeightArgs a) {
    ce_pdl_begin();
    const int lane = threadIdx.x & 31, r = lane >> 2, l = lane & 3, kept = min(a.group, 64), gb = 64 / kept;
    const int kb = blockIdx.y * 8 + (threadIdx.x >> 5), tile_no = blockIdx.x, half_rows = a.rows >> 1;
    if (kb >= a.kblocks) return;
    const unsigned char* tile = a.tiles + ((size_t)tile_no * a.kblocks + kb) * i4_weight_tile_bytes(kept);
    const uint4 w = *reinterpret_cast<const uint4*>(tile + lane * 16);
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {                     // rows r and r + 8, first and second 32 columns
        const int in = r + 8 * (e & 1), col = kb * 64 + 32 * (e >> 1) + 8 * l;
        const int n = a.gated ? tile_no * 8 + r : tile_no * 16 + in, row = a.gated && (e & 1) ? n + half_rows : n;
        if (n >= (a.gated ? half_rows : a.rows) || col >= a.width) continue;
        const __half2 sz = *reinterpret_cast<const __half2*>(tile + 512 + (in * gb + (gb == 2 ? e >> 1 : 0)) * 4);
        float x[8];
        values_of(words[e], sz, x);
        store8((T*)a.w + (long long)row * a.ld + col, a.vec, x);
    }
}

int check_cache(const CacheArgs& a, int dtype, const char* who) {
    if (!a.k || !a.v || !a.pages || !a.positions || !a.seq_of_token || !a.seq_slot || !a.block_table || !a.status)
        return ce_fail(CE_ERR_ARG, "%s: null pointer", who);
    if (dtype != CE_F32 && dtype != CE_BF16) return ce_fail(CE_ERR_ARG, "%s: unknown dtype %d", who, dtype);
    if (a.T < 0 || a.nkv < 1 || a.num_pages < 1 || a.max_pages < 1) return ce_fail(CE_ERR_SIZE, "%s: bad sizes", who);
    if (a.d < 64 || a.d > 256 || a.d % 64) return ce_fail(CE_ERR_SIZE, "%s: head size %d (64, 128, 192 or 256)", who, a.d);
    if (a.group != 32 && a.group != 64) return ce_fail(CE_ERR_SIZE, "%s: group %d (32 or 64)", who, a.group);
    if (a.page_size < 16 || a.page_size % 16) return ce_fail(CE_ERR_SIZE, "%s: page size %d is not a multiple of 16", who, a.page_size);
    return CE_OK;
}

bool aligned4(const void* p, long long s0, long long s1, int dtype) {
    return ((uintptr_t)p % (dtype == CE_F32 ? 16 : 8)) == 0 && s0 % 4 == 0 && s1 % 4 == 0;
}

template <typename F32, typename BF16>
int run_cache(CacheArgs& a, int dtype, F32 f32, BF16 bf16, const char* name, cudaStream_t stream) {
    if (a.T == 0) return CE_OK;
    const int wide = dtype == CE_F32 ? 4 : 8;             // values in 16 bytes
    a.vec = (((uintptr_t)a.k | (uintptr_t)a.v) & 15) == 0 && a.k_token % wide == 0 && a.k_head % wide == 0 && a.v_token % wide == 0 && a.v_head % wide == 0;
    const long long units = (long long)a.T * (a.d >> 6);
    const dim3 grid((unsigned)((units + 31) / 32), (unsigned)a.nkv);
    if (units > 0x7fffffffll || a.nkv > 65535) return ce_fail(CE_ERR_SIZE, "%s: too many rows", name);
    ce_note(name);
    const cudaError_t e = dtype == CE_F32 ? ce_launch(f32, grid, dim3(256), 0, stream, a) : ce_launch(bf16, grid, dim3(256), 0, stream, a);
    if (e != cudaSuccess) { (void)cudaGetLastError(); return ce_fail(CE_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e)); }
    return ce_check_launch(name);
}

int check_weight(const WeightArgs& a, int dtype, const char* who) {
    if (!a.w || !a.tiles) return ce_fail(CE_ERR_ARG, "%s: null pointer", who);
    if (dtype != CE_F32 && dtype != CE_BF16) return ce_fail(CE_ERR_ARG, "%s: unknown dtype %d", who, dtype);
    if (a.group != 32 && a.group != 64 && a.group != 128) return ce_fail(CE_ERR_SIZE, "%s: group %d (32, 64 or 128)", who, a.group);
    if (a.rows < 1 || a.width < 1 || (a.gated && a.rows % 2) || a.width % a.group || a.ld < a.width)
        return ce_fail(CE_ERR_SIZE, "%s: %d rows of %d do not fit (the width is a multiple of the group)", who, a.rows, a.width);
    return CE_OK;
}

}  // namespace

// A call's arguments, 8 bytes each in this order: one pointer to pass takes the host a fifth of the time of twenty arguments.
struct Int4KvCall {
    long long dtype;
    void *k, *v;
    long long k_token, k_head, v_token, v_head;
    void *pages;
    const int *positions, *seq_of_token, *seq_slot, *block_table;
    int* status;
    long long T, nkv, d, group, page_size, max_pages, num_pages;
    void* stream;
};
static int check_sizes(const Int4KvCall& c, const char* who) {
    const long long sizes[] = {c.T, c.nkv, c.d, c.group, c.page_size, c.max_pages, c.num_pages};
    for (long long size : sizes)
        if (size < 0 || size > 0x7fffffffll) return ce_fail(CE_ERR_SIZE, "%s: a size of %lld", who, size);
    return CE_OK;
}
static CacheArgs cache_args(const Int4KvCall& c) {
    return CacheArgs{c.k, c.v, (unsigned char*)c.pages, c.positions, c.seq_of_token, c.seq_slot, c.block_table, c.status, c.k_token, c.k_head,
                     c.v_token, c.v_head, (int)c.T, (int)c.nkv, (int)c.d, (int)c.group, (int)c.page_size, (int)c.max_pages, (int)c.num_pages, 0};
}

extern "C" int ce_int4_kv_write(const Int4KvCall* c) {
    CacheArgs a = cache_args(*c);
    if (int e = check_sizes(*c, "int4_kv_write")) return e;
    if (int e = check_cache(a, (int)c->dtype, "int4_kv_write")) return e;
    return run_cache(a, (int)c->dtype, int4_kv_write_kernel<float>, int4_kv_write_kernel<__nv_bfloat16>, "int4_kv_write_kernel", (cudaStream_t)c->stream);
}

// (writes k and v)
extern "C" int ce_int4_kv_read(const Int4KvCall* c) {
    CacheArgs a = cache_args(*c);
    if (int e = check_sizes(*c, "int4_kv_read")) return e;
    if (int e = check_cache(a, (int)c->dtype, "int4_kv_read")) return e;
    return run_cache(a, (int)c->dtype, int4_kv_read_kernel<float>, int4_kv_read_kernel<__nv_bfloat16>, "int4_kv_read_kernel", (cudaStream_t)c->stream);
}

// dtype, w, ld, tiles, rows, gated, width, group, stream
extern "C" int ce_int4_quantise_weight(int dtype, const void* w, long long ld, void* tiles, int rows, int gated, int width, int group, void* stream) {
    WeightArgs a{w, (unsigned char*)tiles, ld, rows, gated, width, (width + 63) / 64, group, 0};
    if (int e = check_weight(a, dtype, "int4_quantise_weight")) return e;
    a.vec = aligned4(w, ld, 0, dtype);
    const long long tiles_n = gated ? (rows / 2 + 7) / 8 : (rows + 15) / 16, warps = tiles_n * 16 * ((a.kblocks + 1) / 2), grid = (warps + 7) / 8;
    if (grid > 0x7fffffffll) return ce_fail(CE_ERR_SIZE, "int4_quantise_weight: too large");
    ce_note("int4_quantise_weight_kernel");
    const cudaError_t e = dtype == CE_F32 ? ce_launch(int4_quantise_weight_kernel<float>, dim3((unsigned)grid), dim3(256), 0, (cudaStream_t)stream, a)
                                          : ce_launch(int4_quantise_weight_kernel<__nv_bfloat16>, dim3((unsigned)grid), dim3(256), 0, (cudaStream_t)stream, a);
    if (e != cudaSuccess) { (void)cudaGetLastError(); return ce_fail(CE_ERR_CUDA, "int4_quantise_weight: %s", cudaGetErrorString(e)); }
    int4_weight_done_kernel<<<1, 32, 0, (cudaStream_t)stream>>>();
    return ce_check_launch("int4_quantise_weight");
}

extern "C" int ce_int4_dequantise_weight(int dtype, void* w, long long ld, const void* tiles, int rows, int gated, int width, int group, void* stream) {
    WeightArgs a{w, (unsigned char*)tiles, ld, rows, gated, width, (width + 63) / 64, group, 0};
    if (int e = check_weight(a, dtype, "int4_dequantise_weight")) return e;
    a.vec = ((uintptr_t)w & 15) == 0 && ld % (dtype == CE_F32 ? 4 : 8) == 0;
    const dim3 grid((unsigned)(gated ? (rows / 2 + 7) / 8 : (rows + 15) / 16), (unsigned)((a.kblocks + 7) / 8));
    if (grid.y > 65535) return ce_fail(CE_ERR_SIZE, "int4_dequantise_weight: too large");
    ce_note("int4_dequantise_weight_kernel");
    const cudaError_t e = dtype == CE_F32 ? ce_launch(int4_dequantise_weight_kernel<float>, grid, dim3(256), 0, (cudaStream_t)stream, a)
                                          : ce_launch(int4_dequantise_weight_kernel<__nv_bfloat16>, grid, dim3(256), 0, (cudaStream_t)stream, a);
    if (e != cudaSuccess) { (void)cudaGetLastError(); return ce_fail(CE_ERR_CUDA, "int4_dequantise_weight: %s", cudaGetErrorString(e)); }
    int4_weight_done_kernel<<<1, 32, 0, (cudaStream_t)stream>>>();           // (a product may read its weight ahead of the kernels in front)
    return ce_check_launch("int4_dequantise_weight");
}
