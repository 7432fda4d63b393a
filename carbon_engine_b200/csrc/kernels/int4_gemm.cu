// Products of a few tokens with a weight held in 4 bits (int4.cuh): out[t, n] = sum_k x[t, k] W[n, k], W[n, k] = s_ng c_nk + z_ng for the
// group g of k, so
//   out[t, n] = sum_g (s_ng (x_tg . c_ng) + z_ng sum x_tg).
// The codes are the first operand of mma.sync m16n8k16 (16 rows of the weight), 8 tokens the second; a step scales a group's partial sum in
// float32, a minimum meets the group's sum of x.  No value of W is ever rounded.
//
// int4_prepare_kernel lays the tokens out as that second operand once for all blocks: each token is brought into [2^14, 2^15) by a power of
// two and rounded to float16 (exact for bfloat16 down to 2^-30 of the token's largest; float32 as two pieces, 22 bits), with the groups' sums of
// what was rounded.
#include "int4.cuh"

namespace {

constexpr int WARPS = 8;

struct Operand {                   // what int4_prepare_kernel writes: see operand_floats
    uint32_t* frag;                // [kblocks][token tiles][pieces][2 halves][32 lanes][4 words]
    float* sums;                   // [kblocks * groups of a block][token tiles * 8]
    float* back;                   // [token tiles * 8]: what a token's sums are multiplied by at the end
};

struct PrepareArgs {
    const void* x;
    long long ld;
    Operand to;
    int M, K, kblocks, group, vec;      // group: 32 or 64
};

// one block a token of the padded tiles
template <typename T, int P>
__global__ void __launch_bounds__(256) int4_prepare_kernel(PrepareArgs a) {
    ce_pdl_begin();
    __shared__ float scratch[32];
    const int t = blockIdx.x, tiles = gridDim.x >> 3, nt = t >> 3, r = t & 7;
    const bool real = t < a.M;
    const T* src = (const T*)a.x + (size_t)(real ? t : 0) * a.ld;
    float largest = 0.f;
    bool finite = true;
    if (real)
        for (int c = threadIdx.x * 8; c < a.K; c += 256 * 8)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = fabsf(CeType<T>::load(src + c + i));
                largest = fmaxf(largest, v);
                finite = finite && v <= 3.402823466e38f;
            }
    largest = ce_block_max(finite ? largest : INFINITY, scratch);
    const float up = i4_row_scale(largest);
    if (threadIdx.x == 0) a.to.back[t] = i4_unit<P == 2> / up;
    // a thread takes 8 neighbouring columns: the four words of lane (r, l) for a half of a block; four threads hold a run of 32
    const int groups = 64 / a.group;
    for (int c = threadIdx.x * 8; c < a.kblocks * 64; c += 256 * 8) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = 0.f;
        if (real && c < a.K) {                        // (K is a multiple of 32)
            if (a.vec) {
                const float4 u = ce_load4(src + c), v = ce_load4(src + c + 4);
                y[0] = u.x; y[1] = u.y; y[2] = u.z; y[3] = u.w; y[4] = v.x; y[5] = v.y; y[6] = v.z; y[7] = v.w;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = CeType<T>::load(src + c + i);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] *= up;
        }
        const int kb = c >> 6, half = (c >> 5) & 1, l = (c >> 3) & 3;
        float sum = 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f = i & 1 ? 0.0625f : 1.0f, b = i & 1 ? 16.0f : 1.0f;      // odd codes come 16 times too large
                w[i] = i4_pack(y[i] * f, y[i + 4] * f);
                const float2 got = i4_unpack(w[i]);
                sum += (got.x + got.y) * b;
                y[i] -= got.x * b; y[i + 4] -= got.y * b;
            }
            *reinterpret_cast<uint4*>(a.to.frag + ((((size_t)kb * tiles + nt) * P + p) * 2 + half) * 128 + (4 * r + l) * 4) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        const unsigned here = 0xffu << (threadIdx.x & 24);      // the 8 threads of a block of 64 columns: all of them or none are here
        sum += __shfl_xor_sync(here, sum, 1);
        sum += __shfl_xor_sync(here, sum, 2);
        if (a.group == 64) sum += __shfl_xor_sync(here, sum, 4);
        if (c % a.group == 0) a.to.sums[(size_t)(kb * groups + (c & 63) / a.group) * (tiles * 8) + t] = sum * (1.0f / i4_unit<P == 2>);
    }
}

struct GemmArgs {
    const unsigned char* w;        // [row tiles][kblocks][tile]
    Operand x;
    void* out;
    int M, N, kblocks, tiles, ldo, mode, up_tile;        // up_tile: row tiles between a gate row and its up row
};

enum { STORE = 0, STORE_F32 = 1, ACCUM_F32 = 2, SWIGLU = 3, RELUGLU = 4, RELU2 = 5 };

// one block a tile of 16 rows (and the up rows that belong to it): its warps share K
template <typename T, int G, int NT, int HALVES>
__global__ void __launch_bounds__(WARPS * 32) int4_gemm_kernel(GemmArgs a) {
    constexpr int P = sizeof(T) == 4 ? 2 : 1, TILE = i4_weight_tile_bytes(G), GB = 64 / G;
    __shared__ float part[WARPS][16][NT * 8 + 1];
    __shared__ float total[HALVES][16][NT * 8 + 1];
    ce_pdl_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, l = lane & 3;
    const int tokens = a.tiles * 8;
    for (int h = 0; h < HALVES; ++h) {
        float y[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) y[nt][0] = y[nt][1] = y[nt][2] = y[nt][3] = 0.f;
        const unsigned char* rows = a.w + (size_t)(blockIdx.x + h * a.up_tile) * a.kblocks * TILE;
        for (int kb = warp; kb < a.kblocks; kb += WARPS) {
            const unsigned char* tile = rows + (size_t)kb * TILE;
            const uint4 w = *reinterpret_cast<const uint4*>(tile + lane * 16);
            float acc[NT][P][4];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t wa = half ? w.z : w.x, wb = half ? w.w : w.y;
                if ((half * 32) % G == 0)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int p = 0; p < P; ++p) acc[nt][p][0] = acc[nt][p][1] = acc[nt][p][2] = acc[nt][p][3] = 0.f;
                uint32_t e0, e1, e2, e3, o0, o1, o2, o3;
                i4_pairs<P == 2, 0>(wa, e0, e2); i4_pairs<P == 2, 0>(wb, e1, e3);
                i4_pairs<P == 2, 8>(wa, o0, o2); i4_pairs<P == 2, 8>(wb, o1, o3);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        if (nt < a.tiles) {
                            const uint4 x = *reinterpret_cast<const uint4*>(a.x.frag + ((((size_t)kb * a.tiles + nt) * P + p) * 2 + half) * 128 + lane * 4);
                            i4_mma(acc[nt][p], e0, e1, e2, e3, x.x, x.y);
                            i4_mma(acc[nt][p], o0, o1, o2, o3, x.z, x.w);
                        }
                    }
                if ((half * 32 + 32) % G == 0) {
                    const int g = half * 32 / G;
                    const float2 fa = i4_step_of<P == 2>(*reinterpret_cast<const uint32_t*>(tile + 512 + (r * GB + g) * 4));
                    const float2 fb = i4_step_of<P == 2>(*reinterpret_cast<const uint32_t*>(tile + 512 + ((r + 8) * GB + g) * 4));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if (nt >= a.tiles) continue;
                        const float2 s = *reinterpret_cast<const float2*>(a.x.sums + (size_t)(kb * GB + g) * tokens + nt * 8 + 2 * l);
                        float c[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            c[e] = acc[nt][0][e];
                            if constexpr (P == 2) c[e] += acc[nt][1][e];
                        }
                        y[nt][0] = fmaf(fa.x, c[0], fmaf(fa.y, s.x, y[nt][0]));
                        y[nt][1] = fmaf(fa.x, c[1], fmaf(fa.y, s.y, y[nt][1]));
                        y[nt][2] = fmaf(fb.x, c[2], fmaf(fb.y, s.x, y[nt][2]));
                        y[nt][3] = fmaf(fb.x, c[3], fmaf(fb.y, s.y, y[nt][3]));
                    }
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[warp][r + (e >> 1) * 8][nt * 8 + 2 * l + (e & 1)] = y[nt][e];
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * NT * 8; i += WARPS * 32) {
            const int row = i / (NT * 8), t = i - row * (NT * 8);
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) v += part[w][row][t];
            total[h][row][t] = v;
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < 16 * NT * 8; i += WARPS * 32) {
        const int t = i >> 4, row = i & 15, n = blockIdx.x * 16 + row;
        if (t >= a.M || n >= a.N) continue;
        const float back = a.x.back[t];
        float v = total[0][row][t] * back;
        const float u = HALVES == 2 ? total[HALVES - 1][row][t] * back : 0.f;
        const size_t at = (size_t)t * a.ldo + n;
        switch (a.mode) {
            case STORE_F32: ((float*)a.out)[at] = v; break;
            case ACCUM_F32: ((float*)a.out)[at] += v; break;
            case SWIGLU: CeType<T>::store((T*)a.out + at, ce_silu_glu(v, u)); break;
            case RELUGLU: CeType<T>::store((T*)a.out + at, fmaxf(v, 0.f) * u); break;
            case RELU2: v = fmaxf(v, 0.f); CeType<T>::store((T*)a.out + at, v * v); break;
            default: CeType<T>::store((T*)a.out + at, v);
        }
    }
}

int pieces(int dtype) { return dtype == CE_F32 ? 2 : 1; }

template <typename T, int G, int NT>
cudaError_t launch(const GemmArgs& a, int row_tiles, bool gated, cudaStream_t stream) {
    ce_note("int4_gemm_kernel");
    if (gated) return ce_launch(int4_gemm_kernel<T, G, NT, 2>, dim3(row_tiles), dim3(WARPS * 32), 0, stream, a);
    return ce_launch(int4_gemm_kernel<T, G, NT, 1>, dim3(row_tiles), dim3(WARPS * 32), 0, stream, a);
}
template <typename T, int G>
cudaError_t launch_tiles(const GemmArgs& a, int row_tiles, bool gated, cudaStream_t stream) {
    if (a.tiles == 1) return launch<T, G, 1>(a, row_tiles, gated, stream);
    if (a.tiles == 2) return launch<T, G, 2>(a, row_tiles, gated, stream);
    if (a.tiles <= 4) return launch<T, G, 4>(a, row_tiles, gated, stream);
    return launch<T, G, 8>(a, row_tiles, gated, stream);
}

}  // namespace

// float32 words of scratch memory for a product of M tokens and K columns
extern "C" long long ce_int4_gemm_scratch(int dtype, int M, int K, int group) {
    const long long tiles = (M + 7) / 8, kblocks = (K + 63) / 64;
    return kblocks * tiles * pieces(dtype) * 256 + kblocks * (64 / (group < 64 ? group : 64)) * tiles * 8 + tiles * 8;
}

// dtype, x, ldx, w, out, ldo, M, N, K, group, mode, scratch, stream.  N: columns of the result (a gated weight has N gate rows and N up rows).
extern "C" int ce_int4_gemm(int dtype, const void* x, long long ldx, const void* w, void* out, int ldo, int M, int N, int K, int group, int mode,
                            float* scratch, void* stream) {
    if (!x || !w || !out || !scratch) return ce_fail(CE_ERR_ARG, "int4_gemm: null pointer");
    if (dtype != CE_F32 && dtype != CE_BF16) return ce_fail(CE_ERR_ARG, "int4_gemm: unknown dtype %d", dtype);
    if (group != 32 && group != 64 && group != 128) return ce_fail(CE_ERR_SIZE, "int4_gemm: group %d (32, 64 or 128)", group);
    if (mode < STORE || mode > RELU2) return ce_fail(CE_ERR_SIZE, "int4_gemm: epilogue %d is not one of this product's", mode);
    if (M < 0 || M > 64 || N < 1 || K < 1 || K % group || ldx < K || ldo < N)
        return ce_fail(CE_ERR_SIZE, "int4_gemm: %d tokens (at most 64), %d rows of %d (a multiple of the group)", M, N, K);
    if (((uintptr_t)w & 15) || ((uintptr_t)scratch & 15)) return ce_fail(CE_ERR_ARG, "int4_gemm: the weight or the scratch memory is not aligned to 16 bytes");
    if (M == 0) return CE_OK;
    const int kept = group < 64 ? group : 64, tiles = (M + 7) / 8, kblocks = (K + 63) / 64;
    const bool gated = mode == SWIGLU || mode == RELUGLU;
    Operand op;
    op.frag = (uint32_t*)scratch;
    op.sums = scratch + (size_t)kblocks * tiles * pieces(dtype) * 256;
    op.back = op.sums + (size_t)kblocks * (64 / kept) * tiles * 8;
    const int el = dtype == CE_F32 ? 4 : 2;
    PrepareArgs p{x, ldx, op, M, K, kblocks, kept, ((uintptr_t)x % (4 * el)) == 0 && ldx % 4 == 0};
    ce_note("int4_prepare_kernel");
    cudaError_t e = dtype == CE_F32 ? ce_launch(int4_prepare_kernel<float, 2>, dim3(tiles * 8), dim3(256), 0, (cudaStream_t)stream, p)
                                    : ce_launch(int4_prepare_kernel<__nv_bfloat16, 1>, dim3(tiles * 8), dim3(256), 0, (cudaStream_t)stream, p);
    if (e == cudaSuccess) {
        const int row_tiles = (N + 15) / 16;
        GemmArgs a{(const unsigned char*)w, op, out, M, N, kblocks, tiles, ldo, mode, row_tiles};
        if (dtype == CE_F32)
            e = kept == 32 ? launch_tiles<float, 32>(a, row_tiles, gated, (cudaStream_t)stream) : launch_tiles<float, 64>(a, row_tiles, gated, (cudaStream_t)stream);
        else
            e = kept == 32 ? launch_tiles<__nv_bfloat16, 32>(a, row_tiles, gated, (cudaStream_t)stream)
                           : launch_tiles<__nv_bfloat16, 64>(a, row_tiles, gated, (cudaStream_t)stream);
    }
    if (e != cudaSuccess) { (void)cudaGetLastError(); return ce_fail(CE_ERR_CUDA, "int4_gemm: %s", cudaGetErrorString(e)); }
    return ce_check_launch("int4_gemm");
}
