// Products of a few tokens with a weight held in 4 bits (int4.cuh): out[t, n] = sum_k x[t, k] W[n, k], W[n, k] = s_ng c_nk + z_ng for the
// group g of k, so
//   out[t, n] = sum_g (s_ng (x_tg . c_ng) + z_ng sum x_tg).
// The codes are the first operand of mma.sync m16n8k16 (16 rows of the weight), 8 tokens the second; a step scales a group's partial sum in
// float32, a minimum meets the group's sum of x.  No value of W is ever rounded.
//
// Up to 16 tokens run int4_stream_kernel, more bfloat16 ones (or wider) int4_gemm_tc.cu, more float32 ones (or wider) int4_gemm_kernel, for which
// int4_prepare_kernel lays the tokens out as that second operand: each token is brought into [2^14, 2^15) by a power of two and rounded to two
// float16 pieces (22 bits), with the groups' sums of what was rounded (4,096 x 4,096: 27 us for 17 tokens, 53 for 64).
//
// The stream is bound by the instructions that take codes apart and by the latencies between them, not by memory: 6,144 x 4,096 for one token
// 6.4 us (2.2 TB/s), 12,288 + 12,288 rows of 4,096 for 8 tokens 17.3 us (3.3 TB/s), 75,776 x 4,096 for one token 40 us (4.4 TB/s).  Up to 8 tokens it
// is the faster one everywhere; for 9 to 16 it is as long as rows are few (4,096 x 12,288, 16 tokens: 19.6 us, on tcgen05 24; 12,288 + 12,288 x 4,096:
// 33, 51), and 10 % slower for 75,776 rows of 4,096 (112, 99).  Warm weights; past cold ones 12,288 + 12,288 x 4,096 take 21 us for 8 tokens, 40 for 16.
#include "int4.cuh"

namespace {

constexpr int WARPS = 8;

constexpr int PIECES = 2;          // float16 numbers of a float32 token's value

struct Operand {                   // what int4_prepare_kernel writes: ce_int4_gemm_scratch counts it
    uint32_t* frag;                // [kblocks][token tiles][PIECES][2 halves][32 lanes][4 words]
    float* sums;                   // [kblocks * groups of a block][token tiles * 8]
    float* back;                   // [token tiles * 8]: what a token's sums are multiplied by at the end
};

struct PrepareArgs {
    const float* x;
    long long ld;
    Operand to;
    int M, K, kblocks, group, vec;      // group: 32 or 64
};

// one block a token of the padded tiles
__global__ void __launch_bounds__(256) int4_prepare_kernel(PrepareArgs a) {
    ce_pdl_begin();
    __shared__ float scratch[32];
    const int t = blockIdx.x, tiles = gridDim.x >> 3, nt = t >> 3, r = t & 7;
    const bool real = t < a.M;
    const float* src = a.x + (size_t)(real ? t : 0) * a.ld;
    float largest = 0.f;
    bool finite = true;
    if (real)
        for (int c = threadIdx.x * 8; c < a.K; c += 256 * 8)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = fabsf(src[c + i]);
                largest = fmaxf(largest, v);
                finite = finite && v <= 3.402823466e38f;
            }
    largest = ce_block_max(finite ? largest : INFINITY, scratch);
    const float up = i4_row_scale(largest);
    if (threadIdx.x == 0) a.to.back[t] = 1.0f / up;
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
                for (int i = 0; i < 8; ++i) y[i] = src[c + i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] *= up;
        }
        const int kb = c >> 6, half = (c >> 5) & 1, l = (c >> 3) & 3;
        float sum = 0.f;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f = i & 1 ? 0.0625f : 1.0f, b = i & 1 ? 16.0f : 1.0f;      // odd codes come 16 times too large
                w[i] = i4_pack(y[i] * f, y[i + 4] * f);
                const float2 got = i4_unpack(w[i]);
                sum += (got.x + got.y) * b;
                y[i] -= got.x * b; y[i + 4] -= got.y * b;
            }
            *reinterpret_cast<uint4*>(a.to.frag + ((((size_t)kb * tiles + nt) * PIECES + p) * 2 + half) * 128 + (4 * r + l) * 4) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        const unsigned here = 0xffu << (threadIdx.x & 24);      // the 8 threads of a block of 64 columns: all of them or none are here
        sum += __shfl_xor_sync(here, sum, 1);
        sum += __shfl_xor_sync(here, sum, 2);
        if (a.group == 64) sum += __shfl_xor_sync(here, sum, 4);
        if (c % a.group == 0) a.to.sums[(size_t)(kb * groups + (c & 63) / a.group) * (tiles * 8) + t] = sum;
    }
}

struct GemmArgs {
    const unsigned char* w;        // [row tiles][kblocks][tile]
    Operand x;
    void* out;
    long long ldo;
    int M, N, kblocks, tiles, mode, gated;
};

enum { STORE = 0, STORE_F32 = 1, ACCUM_F32 = 2, SWIGLU = 3, RELUGLU = 4, RELU2 = 5 };

template <typename T>
__device__ __forceinline__ void finish(void* out, size_t at, int mode, float v, float u) {
    switch (mode) {
        case STORE_F32: ((float*)out)[at] = v; break;
        case ACCUM_F32: ((float*)out)[at] += v; break;
        case SWIGLU: CeType<T>::store((T*)out + at, ce_silu_glu(v, u)); break;
        case RELUGLU: CeType<T>::store((T*)out + at, i4_relu(v) * u); break;
        case RELU2: v = i4_relu(v); CeType<T>::store((T*)out + at, v * v); break;
        default: CeType<T>::store((T*)out + at, v);
    }
}

// one block a tile of 16 rows: its warps share K
template <int G, int NT>
__global__ void __launch_bounds__(WARPS * 32) int4_gemm_kernel(GemmArgs a) {
    constexpr int P = PIECES, TILE = i4_weight_tile_bytes(G), GB = 64 / G;
    __shared__ float part[WARPS][16][NT * 8 + 1];
    __shared__ float total[16][NT * 8 + 1];
    ce_pdl_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, l = lane & 3;
    const int tokens = a.tiles * 8;
    {
        float y[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) y[nt][0] = y[nt][1] = y[nt][2] = y[nt][3] = 0.f;
        const unsigned char* rows = a.w + (size_t)blockIdx.x * a.kblocks * TILE;
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
                i4_pairs<true, 0>(wa, e0, e2); i4_pairs<true, 0>(wb, e1, e3);
                i4_pairs<true, 8>(wa, o0, o2); i4_pairs<true, 8>(wb, o1, o3);
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
                    const float2 fa = i4_step_of<true>(*reinterpret_cast<const uint32_t*>(tile + 512 + (r * GB + g) * 4));
                    const float2 fb = i4_step_of<true>(*reinterpret_cast<const uint32_t*>(tile + 512 + ((r + 8) * GB + g) * 4));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if (nt >= a.tiles) continue;
                        const float2 s = *reinterpret_cast<const float2*>(a.x.sums + (size_t)(kb * GB + g) * tokens + nt * 8 + 2 * l);
                        float c[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) c[e] = acc[nt][0][e] + acc[nt][1][e];
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
            total[row][t] = v;
        }
        __syncthreads();
    }
    const int rows_out = a.gated ? 8 : 16;
    for (int i = threadIdx.x; i < rows_out * NT * 8; i += WARPS * 32) {
        const int t = i / rows_out, row = i - t * rows_out, n = blockIdx.x * rows_out + row;
        if (t >= a.M || n >= a.N) continue;
        const float back = a.x.back[t];
        finish<float>(a.out, (size_t)t * a.ldo + n, a.mode, total[row][t] * back, a.gated ? total[row + 8][t] * back : 0.f);
    }
}

// ---------------------------------------------------------------------------------------------
// Up to 16 tokens: a stream of weights past tokens that stay in registers.
//
// A block takes some tiles of 16 rows and a slice of K; each of its 16 warps a run of up to KW blocks of 64
// columns of that slice.  A warp holds its run of all tokens as the second operand (laid out and scaled by itself: nothing to prepare, and one
// launch) and meets the rows' tiles one after another, each a run of bytes that one lane copies into the warp's ring ahead of time.  What the
// warps make of a tile is added up in their order, what the blocks of a cluster make of it (slices of K) in theirs, through shared memory.
// The copies begin before the kernels in front have ended: no kernel writes a weight (ops_int4.Int4Weight sees to that).
// ---------------------------------------------------------------------------------------------
constexpr int SW = 16;             // warps

struct StreamArgs {
    const void* x;
    const unsigned char* w;
    void* out;
    int* status;
    long long ldx, ldo;
    int M, N, K, kblocks, mode, gated, units, each, slices, overlap, vec;
};

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float load_cluster(uint32_t local, int rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(local), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

template <typename T, int G, int NT, int KW>
struct StreamShape {
    static constexpr int TILE = i4_weight_tile_bytes(G), STAGE = KW * TILE, STAGES = 16 / KW, RING = SW * STAGES * STAGE;
    static constexpr int LD = 20;                                             // floats of a token's 16 rows: no two lanes of a store meet in a bank
    static constexpr int SUMS = NT * 8 * LD;                                  // floats of a tile's sums of one warp
    static constexpr int BATCH = 4 / NT;                                      // tiles between two meetings of the warps
    static constexpr int PART = BATCH * SW * SUMS * 4;
    static constexpr int TOTAL = NT * 8 * 16 * 4;                             // bytes of a tile's sums of a slice, where others add theirs
    static constexpr int MOST = (227 * 1024 - 4096 - RING - PART) / TOTAL;    // tiles a block can take
    static constexpr size_t smem(int tiles, int slices) { return RING + PART + (slices > 1 ? (size_t)tiles * TOTAL : 0); }
};

// The groups' sums of the tokens, which meet the minima.  bfloat16: as two float16 pieces (22 bits) of sum / 2^7, the second operand of ONE product
// whose first holds the minima of the run's groups (2 l and 2 l + 1 at lane (r, l), twice: once for each piece) - instead of four fma, and
// two conversions, a group.  float32: float32, since its minimum is that of code 8 and no float16.
template <int P, int G, int NT, int KW> struct Sums { uint32_t b[NT][2]; };
template <int G, int NT, int KW> struct Sums<2, G, NT, KW> { float f[KW][64 / G][NT][2]; };

// A warp's run of one tile: its sums of 16 rows by the tokens, in float32.  ``at``: byte offsets of the run's blocks of 64 columns; a run with
// fewer than KW repeats its last, against tokens that are zeros there (``z_at``: of the minima of this lane's groups): no question a block, and the loads and products of all of them overlap
// (four chains of products side by side).
template <typename T, int G, int NT, int KW>
__device__ __forceinline__ void stream_run(const unsigned char* stage, const int (&at)[KW], const int (&z_at)[2], int lane, const uint32_t (&xf)[KW][NT][sizeof(T) == 4 ? 2 : 1][2][4],
                                           const Sums<sizeof(T) == 4 ? 2 : 1, G, NT, KW>& sums, float (&y)[NT][4]) {
    constexpr int P = sizeof(T) == 4 ? 2 : 1, GB = 64 / G;
    constexpr bool C8 = P == 2;
    const int r = lane >> 2;
    if constexpr (P == 1) {
        // minima of this lane's two groups for rows r and r + 8 (groups beyond the run: any of the row, their sums are 0)
        uint32_t za, zb;
        const unsigned char *p = stage + z_at[0], *q = stage + z_at[1];
        if constexpr (GB == 2) {
            const uint2 u = *reinterpret_cast<const uint2*>(p), v = *reinterpret_cast<const uint2*>(p + 64);
            za = __byte_perm(u.x, u.y, 0x7632); zb = __byte_perm(v.x, v.y, 0x7632);
        } else {
            za = __byte_perm(*reinterpret_cast<const uint32_t*>(p), *reinterpret_cast<const uint32_t*>(q), 0x7632);
            zb = __byte_perm(*reinterpret_cast<const uint32_t*>(p + 32), *reinterpret_cast<const uint32_t*>(q + 32), 0x7632);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) i4_mma_first(y[nt], za, zb, za, zb, sums.b[nt][0], sums.b[nt][1]);
    }
    uint4 w[KW];
    uint32_t sa[KW][GB], sb[KW][GB];
#pragma unroll
    for (int k = 0; k < KW; ++k) {
        const unsigned char* tile = stage + at[k];
        w[k] = *reinterpret_cast<const uint4*>(tile + lane * 16);
        if constexpr (GB == 2) {
            const uint2 u = *reinterpret_cast<const uint2*>(tile + 512 + r * 8), v = *reinterpret_cast<const uint2*>(tile + 512 + r * 8 + 64);
            sa[k][0] = u.x; sa[k][1] = u.y; sb[k][0] = v.x; sb[k][1] = v.y;
        } else {
            sa[k][0] = *reinterpret_cast<const uint32_t*>(tile + 512 + r * 4);
            sb[k][0] = *reinterpret_cast<const uint32_t*>(tile + 512 + r * 4 + 32);
        }
    }
    float acc[KW][GB][NT][P][4];
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
            for (int k = 0; k < KW; ++k) {
                const uint32_t wa = half ? w[k].z : w[k].x, wb = half ? w[k].w : w[k].y;
                uint32_t a0, a1, a2, a3;
                if (st) { i4_pairs<C8, 8>(wa, a0, a2); i4_pairs<C8, 8>(wb, a1, a3); }
                else { i4_pairs<C8, 0>(wa, a0, a2); i4_pairs<C8, 0>(wb, a1, a3); }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        float (&c)[4] = acc[k][half * 32 / G][nt][p];
                        if (st == 0 && half * 32 % G == 0) i4_mma_first(c, a0, a1, a2, a3, xf[k][nt][p][half][0], xf[k][nt][p][half][1]);
                        else i4_mma(c, a0, a1, a2, a3, xf[k][nt][p][half][2 * st], xf[k][nt][p][half][2 * st + 1]);
                    }
            }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[nt][e] = P == 1 ? y[nt][e] * (128.0f / i4_unit<false>) : 0.f;
#pragma unroll
    for (int k = 0; k < KW; ++k)
#pragma unroll
        for (int g = 0; g < GB; ++g) {
            const float2 fa = i4_step_of<C8>(sa[k][g]), fb = i4_step_of<C8>(sb[k][g]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float c[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    c[e] = acc[k][g][nt][0][e];
                    if constexpr (P == 2) c[e] += acc[k][g][nt][1][e];
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if constexpr (P == 2) {
                        y[nt][e] = fmaf(fa.y, sums.f[k][g][nt][e], y[nt][e]);
                        y[nt][2 + e] = fmaf(fb.y, sums.f[k][g][nt][e], y[nt][2 + e]);
                    }
                    y[nt][e] = fmaf(fa.x, c[e], y[nt][e]);
                    y[nt][2 + e] = fmaf(fb.x, c[2 + e], y[nt][2 + e]);
                }
            }
        }
}

template <typename T, int G, int NT, int KW>
__global__ void __launch_bounds__(SW * 32) int4_stream_kernel(StreamArgs a) {
    using Shape = StreamShape<T, G, NT, KW>;
    constexpr int P = sizeof(T) == 4 ? 2 : 1, TILE = Shape::TILE, STAGES = Shape::STAGES, GB = 64 / G;
    constexpr bool C8 = P == 2;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) uint64_t full[SW][STAGES];
    constexpr int BATCH = Shape::BATCH, SUMS = Shape::SUMS, LD = Shape::LD;
    float* part = reinterpret_cast<float*>(smem + Shape::RING);               // [BATCH][SW][tokens][LD]
    float* total = reinterpret_cast<float*>(smem + Shape::RING + Shape::PART);    // [tiles of the block][tokens][16], where K has slices
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, l = lane & 3;
    const int slice = blockIdx.x % a.slices, first = blockIdx.x / a.slices * a.each, its = min(a.each, a.units - first);
    const int kb_begin = (int)((long long)a.kblocks * slice / a.slices), kb_end = (int)((long long)a.kblocks * (slice + 1) / a.slices);
    const int run = (kb_end - kb_begin + SW - 1) / SW, kb0 = min(kb_begin + warp * run, kb_end), count = min(run, kb_end - kb0);
    unsigned char* ring = smem + warp * (STAGES * Shape::STAGE);
    if (a.overlap) ce_pdl_launch_dependents();
    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < STAGES; ++s) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(i4_smem(&full[warp][s])));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    const unsigned char* next = a.w + ((size_t)first * a.kblocks + kb0) * TILE;
    const size_t step = (size_t)a.kblocks * TILE;
    auto issue = [&](int it) {
        if (lane == 0 && count > 0) i4_copy(ring + it % STAGES * Shape::STAGE, next, count * TILE, &full[warp][it % STAGES]);
        next += step;
    };
    for (int it = 0; it < min(STAGES, its); ++it) issue(it);
    ce_pdl_wait();

    // ---- the warp's run of the tokens: lane (r, l) lays out token 8 nt + r, columns 8 l .. + 8 of every 32
    uint32_t xf[KW][NT][P][2][4];
    Sums<P, G, NT, KW> sums;
    float back[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int t = nt * 8 + r;
        const T* src = (const T*)a.x + (size_t)t * a.ldx + kb0 * 64 + 8 * l;
        float up;
        if constexpr (P == 1) {
            // in pairs, as they lie; the groups' sums as products with codes of 1 (as ordinary numbers): a third of the instructions, which a block runs
            // once and cold (6,144 x 4,096, one token: 4,500 cycles of 10,800 before)
            uint32_t x[KW][2][4];
#pragma unroll
            for (int k = 0; k < KW; ++k)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int c = k * 64 + half * 32;
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[k][half][i] = 0;
                    if (t < a.M && k < count && kb0 * 64 + c + 8 * l < a.K) {
                        if (a.vec) {
                            const uint2 u = *reinterpret_cast<const uint2*>(src + c), v = *reinterpret_cast<const uint2*>(src + c + 4);
                            x[k][half][0] = u.x; x[k][half][1] = u.y; x[k][half][2] = v.x; x[k][half][3] = v.y;
                        } else {
                            const unsigned short* p = reinterpret_cast<const unsigned short*>(src + c);
#pragma unroll
                            for (int i = 0; i < 4; ++i) x[k][half][i] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
                        }
                    }
                }
            __nv_bfloat162 most = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
            for (int k = 0; k < KW; ++k)
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int i = 0; i < 4; ++i) most = __hmax2_nan(most, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&x[k][half][i])));
            const float2 two = __bfloat1622float2(most);
            float largest = two.x <= 3.402823466e38f && two.y <= 3.402823466e38f ? fmaxf(two.x, two.y) : INFINITY;
            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
            up = i4_row_scale(largest);
            const float up16 = up * 0.0625f;                                  // odd codes come 16 times too large
            sums.b[nt][0] = sums.b[nt][1] = 0;
#pragma unroll
            for (int k = 0; k < KW; ++k) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t* v = x[k][half];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        xf[k][nt][0][half][2 * i] = i4_pack(__uint_as_float(v[i] << 16) * up, __uint_as_float(v[i + 2] << 16) * up);
                        xf[k][nt][0][half][2 * i + 1] = i4_pack(__uint_as_float(v[i] & 0xffff0000u) * up16, __uint_as_float(v[i + 2] & 0xffff0000u) * up16);
                    }
                }
#pragma unroll
                for (int g = 0; g < GB; ++g) {
                    float c[4];
#pragma unroll
                    for (int half = g * G / 32; half < (g + 1) * G / 32; ++half) {
                        const uint32_t* v = xf[k][nt][0][half];
                        if (half == g * G / 32) i4_mma_first(c, 0x3c003c00u, 0x3c003c00u, 0x4c004c00u, 0x4c004c00u, v[0], v[1]);
                        else i4_mma(c, 0x3c003c00u, 0x3c003c00u, 0x4c004c00u, 0x4c004c00u, v[0], v[1]);
                        i4_mma(c, 0x3c003c00u, 0x3c003c00u, 0x4c004c00u, 0x4c004c00u, v[2], v[3]);
                    }
                    // (sums of tokens 2 l and 2 l + 1 are here; of token r wanted)
                    const float even = __shfl_sync(0xffffffffu, c[0], r >> 1), odd = __shfl_sync(0xffffffffu, c[1], r >> 1);
                    const float part = (r & 1 ? odd : even) * (1.0f / 128.0f), high = __half2float(__float2half_rn(part));
                    const int at = k * GB + g;                                // of the run's groups
                    if (at >> 1 == l) {
                        sums.b[nt][0] |= i4_pack(at & 1 ? 0.f : part, at & 1 ? part : 0.f);
                        sums.b[nt][1] |= i4_pack(at & 1 ? 0.f : part - high, at & 1 ? part - high : 0.f);
                    }
                }
            }
        } else {
            float x[KW][2][8], largest = 0.f;
            bool finite = true;
#pragma unroll
            for (int k = 0; k < KW; ++k)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int c = k * 64 + half * 32;
                    if (t < a.M && k < count && kb0 * 64 + c + 8 * l < a.K) {
                        if (a.vec) {
                            const float4 u = ce_load4(src + c), v = ce_load4(src + c + 4);
                            x[k][half][0] = u.x; x[k][half][1] = u.y; x[k][half][2] = u.z; x[k][half][3] = u.w;
                            x[k][half][4] = v.x; x[k][half][5] = v.y; x[k][half][6] = v.z; x[k][half][7] = v.w;
                        } else {
#pragma unroll
                            for (int i = 0; i < 8; ++i) x[k][half][i] = CeType<T>::load(src + c + i);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[k][half][i] = 0.f;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) { largest = fmaxf(largest, fabsf(x[k][half][i])); finite = finite && fabsf(x[k][half][i]) <= 3.402823466e38f; }
                }
            if (!finite) largest = INFINITY;
            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
            up = i4_row_scale(largest);
#pragma unroll
            for (int k = 0; k < KW; ++k) {
                float sum[GB];
#pragma unroll
                for (int g = 0; g < GB; ++g) sum[g] = 0.f;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float y[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = x[k][half][i] * up;
#pragma unroll
                    for (int p = 0; p < P; ++p)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float f = i & 1 ? 0.0625f : 1.0f, b = i & 1 ? 16.0f : 1.0f;      // odd codes come 16 times too large
                            xf[k][nt][p][half][i] = i4_pack(y[i] * f, y[i + 4] * f);
                            const float2 got = i4_unpack(xf[k][nt][p][half][i]);
                            sum[half * 32 / G] += (got.x + got.y) * b;
                            y[i] -= got.x * b; y[i + 4] -= got.y * b;
                        }
                }
#pragma unroll
                for (int g = 0; g < GB; ++g) {
                    sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
                    sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
#pragma unroll
                    for (int e = 0; e < 2; ++e) sums.f[k][g][nt][e] = __shfl_sync(0xffffffffu, sum[g], 4 * (2 * l + e)) * (1.0f / i4_unit<C8>);
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) back[nt][e] = 1.0f / __shfl_sync(0xffffffffu, up, 4 * (2 * l + e));      // (not times the unit: of tokens of 2^117 that is no float32)
    }

    // a batch's sums, one a thread: of tile u of it, token t, row
    static_assert(BATCH * NT * 8 * 16 == SW * 32, "one result a thread");
    const int row = threadIdx.x & 15, u = (threadIdx.x >> 4) / a.M, t = (threadIdx.x >> 4) - u * a.M;
    const bool sums_here = u < BATCH;
    const float* from = part + u * SW * SUMS + t * LD + row;
    float* mine = part + warp * SUMS + 2 * l * LD + r;
    int at[KW];
#pragma unroll
    for (int k = 0; k < KW; ++k) at[k] = max(0, min(k, count - 1)) * TILE;
    // where this lane's two minima lie: see stream_run
    const int z_at[2] = {max(0, min(GB == 2 ? l : 2 * l, count - 1)) * TILE + 512 + r * (4 * GB), max(0, min(2 * l + 1, count - 1)) * TILE + 512 + r * 4};
    int gave_up = -1;                                 // the tile whose copy was not waited for to the end
    for (int it = 0; it < its; ++it) {
        float* to = mine + it % BATCH * (SW * SUMS);
        if (count > 0) {
            if (gave_up < 0 && !i4_warp_wait(&full[warp][it % STAGES], (it / STAGES) & 1)) {
                gave_up = it;
                atomicExch(a.status, 59);
            }
            float y[NT][4];
            stream_run<T, G, NT, KW>(ring + it % STAGES * Shape::STAGE, at, z_at, lane, xf, sums, y);
            __syncwarp();
            if (it + STAGES < its && gave_up < 0) issue(it + STAGES);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) to[(nt * 8 + (e & 1)) * LD + (e >> 1) * 8] = y[nt][e] * i4_unit<C8> * back[nt][e & 1];
        } else {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) to[(nt * 8 + (e & 1)) * LD + (e >> 1) * 8] = 0.f;
        }
        if ((it + 1) % BATCH && it + 1 < its) continue;
        // the warps' sums of this batch's tiles, in their order
        __syncthreads();
        const int base = it / BATCH * BATCH;
        const bool real = sums_here && base + u < its;
        float v = 0.f;
        if (real)
#pragma unroll
            for (int w = 0; w < SW; ++w) v += from[w * SUMS];
        if (a.slices > 1) {
            if (real) total[(base + u) * (NT * 128) + t * 16 + row] = v;
        } else {
            const float up = __shfl_down_sync(0xffffffffu, v, 8);             // (of a gate row)
            const int tile_no = first + base + u, n = a.gated ? tile_no * 8 + row : tile_no * 16 + row;
            if (real && n < a.N && (!a.gated || row < 8)) finish<T>(a.out, (size_t)t * a.ldo + n, a.mode, v, up);
        }
        if (it + 1 < its) __syncthreads();
    }
    // a wait that gave up leaves copies in flight: they are waited for, with a limit, before the block may end
    if (gave_up >= 0)
        for (int i = gave_up; i < min(gave_up + STAGES, its); ++i) i4_wait(&full[warp][i % STAGES], (i / STAGES) & 1);
    if (a.slices == 1) return;
    // the slices' sums, in their order: a block adds up every ``slices``-th run of 512 results of the cluster's
    cluster_sync();
    const int results = its * a.M * 16;
    for (int o = threadIdx.x + slice * (SW * 32); o < (results + 31) / 32 * 32; o += a.slices * (SW * 32)) {
        const int row = o & 15, rest = o >> 4, u = rest / a.M, t = rest - u * a.M;
        float v = 0.f;
        if (o < results)
            for (int s = 0; s < a.slices; ++s) v += load_cluster(i4_smem(total + u * (NT * 128) + t * 16 + row), s);
        const float up = __shfl_down_sync(0xffffffffu, v, 8);
        const int n = a.gated ? (first + u) * 8 + row : (first + u) * 16 + row;
        if (o < results && n < a.N && (!a.gated || row < 8)) finish<T>(a.out, (size_t)t * a.ldo + n, a.mode, v, up);
    }
    cluster_sync();                                   // nobody leaves while its sums are read
}

// Returns 1 where the sizes are not this kernel's.
template <typename T, int G, int NT>
int launch_stream(StreamArgs a, cudaStream_t stream) {
    constexpr int P = sizeof(T) == 4 ? 2 : 1, KW = 4 / (NT * P);
    using Shape = StreamShape<T, G, NT, KW>;
    auto kernel = int4_stream_kernel<T, G, NT, KW>;
    // slices of K: as few as the registers ask for; more where there are fewer tiles than SMs, down to 1,024 columns a slice
    const int sms = ce_sm_count();
    int slices = (a.kblocks + SW * KW - 1) / (SW * KW);
    while (slices < 8 && a.units * slices * 3 < sms * 2 && a.kblocks / (slices + 1) >= 16) ++slices;
    if (slices > 8) return 1;
    static std::atomic<unsigned long long> done{0};
    cudaError_t e = ce_allow_smem(done, kernel, Shape::smem(Shape::MOST, 2));
    if (e != cudaSuccess) { (void)cudaGetLastError(); return ce_fail(CE_ERR_CUDA, "int4_gemm: %s", cudaGetErrorString(e)); }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    cfg.blockDim = dim3(SW * 32);
    cfg.stream = stream;
    cfg.attrs = attr;
    int most = sms;
    if (slices > 1) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {(unsigned)slices, 1, 1};
        cfg.numAttrs = 1;
        cfg.gridDim = dim3(slices);
        cfg.dynamicSmemBytes = Shape::smem(Shape::MOST, 2);
        static CeRoom room[9];
        most = ce_clusters_at_once(room[slices], kernel, cfg);
        if (most < 1) return 1;
    }
    a.slices = slices;
    a.each = (a.units + most - 1) / most;             // tiles a block
    if (slices > 1) a.each = min(a.each, Shape::MOST);
    const int groups = (a.units + a.each - 1) / a.each;
    a.overlap = (slices == 1 || groups <= most) && ce_pdl_enabled();
    cfg.gridDim = dim3((unsigned)(groups * slices));
    cfg.dynamicSmemBytes = Shape::smem(a.each, slices);
    cfg.numAttrs = slices > 1 ? 1 : 0;
    if (a.overlap) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++cfg.numAttrs;
    }
    ce_note("int4_stream_kernel");
    e = cudaLaunchKernelEx(&cfg, kernel, a);
    if (e != cudaSuccess) { (void)cudaGetLastError(); return ce_fail(CE_ERR_CUDA, "int4_gemm: %s", cudaGetErrorString(e)); }
    return ce_check_launch("int4_gemm");
}
template <typename T, int G>
int launch_stream_tiles(const StreamArgs& a, int tiles, cudaStream_t stream) {
    return tiles == 1 ? launch_stream<T, G, 1>(a, stream) : launch_stream<T, G, 2>(a, stream);
}

template <int G, int NT>
cudaError_t launch(const GemmArgs& a, int row_tiles, cudaStream_t stream) {
    ce_note("int4_gemm_kernel");
    return ce_launch(int4_gemm_kernel<G, NT>, dim3(row_tiles), dim3(WARPS * 32), 0, stream, a);
}
template <int G>
cudaError_t launch_tiles(const GemmArgs& a, int row_tiles, cudaStream_t stream) {
    if (a.tiles == 1) return launch<G, 1>(a, row_tiles, stream);          // (K beyond the stream's registers)
    if (a.tiles == 2) return launch<G, 2>(a, row_tiles, stream);
    if (a.tiles <= 4) return launch<G, 4>(a, row_tiles, stream);
    return launch<G, 8>(a, row_tiles, stream);
}

}  // namespace

long long ce_int4_gemm_tc_scratch(int M, int K);
int ce_int4_gemm_tc(const void* x, long long ldx, const void* w, void* out, long long ldo, int M, int N, int K, int kept, int mode, float* scratch, int* status,
                    cudaStream_t stream);

namespace {

// Whether the stream of weights takes these sizes: up to 16 tokens, K within the registers of 8 blocks
bool streamed(int dtype, int M, int K) {
    const int tiles = (M + 7) / 8, nt_p = tiles * (dtype == CE_F32 ? PIECES : 1);
    return tiles <= 2 && (K + 63) / 64 <= 8 * SW * (4 / nt_p);
}

}  // namespace

// float32 words of scratch memory (0: none) for a product of M tokens and K columns
extern "C" long long ce_int4_gemm_scratch(int dtype, int M, int K, int group) {
    if (streamed(dtype, M, K)) return 0;
    if (dtype == CE_BF16) return ce_int4_gemm_tc_scratch(M, K);
    const long long tiles = (M + 7) / 8, kblocks = (K + 63) / 64;
    return kblocks * tiles * PIECES * 256 + kblocks * (64 / (group < 64 ? group : 64)) * tiles * 8 + tiles * 8;
}

// A call's arguments, 8 bytes each in this order.  N: columns of the result (a gated weight has N gate rows and N up rows).
struct Int4GemmCall {
    long long dtype;
    const void* x;
    long long ldx;
    const void* w;
    void* out;
    long long ldo, M, N, K, group, mode;
    float* scratch;
    int* status;
    void* stream;
};

extern "C" int ce_int4_gemm(const Int4GemmCall* c) {
    const void *x = c->x, *w = c->w;
    void *out = c->out, *stream = c->stream;
    float* scratch = c->scratch;
    const long long ldx = c->ldx, ldo = c->ldo;
    const int dtype = (int)c->dtype, M = (int)c->M, N = (int)c->N, K = (int)c->K, group = (int)c->group, mode = (int)c->mode;
    if (!x || !w || !out) return ce_fail(CE_ERR_ARG, "int4_gemm: null pointer");
    if (dtype != CE_F32 && dtype != CE_BF16) return ce_fail(CE_ERR_ARG, "int4_gemm: unknown dtype %d", dtype);
    if (group != 32 && group != 64 && group != 128) return ce_fail(CE_ERR_SIZE, "int4_gemm: group %d (32, 64 or 128)", group);
    if (mode < STORE || mode > RELU2) return ce_fail(CE_ERR_SIZE, "int4_gemm: epilogue %d is not one of this product's", mode);
    if (c->M < 0 || c->M > 64 || c->N < 1 || c->N > 0x3fffffff || c->K < 1 || c->K > 0x3fffffff || K % group || ldx < K || ldo < N)
        return ce_fail(CE_ERR_SIZE, "int4_gemm: %lld tokens (at most 64), %lld rows of %lld (a multiple of the group)", c->M, c->N, c->K);
    if (((uintptr_t)w & 15) || ((uintptr_t)scratch & 15)) return ce_fail(CE_ERR_ARG, "int4_gemm: the weight or the scratch memory is not aligned to 16 bytes");
    if (M == 0) return CE_OK;
    const int kept = group < 64 ? group : 64, tiles = (M + 7) / 8, kblocks = (K + 63) / 64;
    const bool gated = mode == SWIGLU || mode == RELUGLU;
    const int el = dtype == CE_F32 ? 4 : 2, row_tiles = gated ? (N + 7) / 8 : (N + 15) / 16;
    const bool vec = ((uintptr_t)x % (4 * el)) == 0 && ldx % 4 == 0;
    if (streamed(dtype, M, K)) {
        StreamArgs a{x, (const unsigned char*)w, out, c->status, ldx, ldo, M, N, K, kblocks, mode, gated, row_tiles, 0, 0, 0, vec};
        const int code = dtype == CE_F32 ? (kept == 32 ? launch_stream_tiles<float, 32>(a, tiles, (cudaStream_t)stream)
                                                       : launch_stream_tiles<float, 64>(a, tiles, (cudaStream_t)stream))
                                         : (kept == 32 ? launch_stream_tiles<__nv_bfloat16, 32>(a, tiles, (cudaStream_t)stream)
                                                       : launch_stream_tiles<__nv_bfloat16, 64>(a, tiles, (cudaStream_t)stream));
        return code == 1 ? ce_fail(CE_ERR_SIZE, "int4_gemm: no room for clusters on this device") : code;
    }
    if (!scratch) return ce_fail(CE_ERR_ARG, "int4_gemm: these sizes need scratch memory");
    if (dtype == CE_BF16) return ce_int4_gemm_tc(x, ldx, w, out, ldo, M, N, K, kept, mode, scratch, c->status, (cudaStream_t)stream);
    Operand op;
    op.frag = (uint32_t*)scratch;
    op.sums = scratch + (size_t)kblocks * tiles * PIECES * 256;
    op.back = op.sums + (size_t)kblocks * (64 / kept) * tiles * 8;
    PrepareArgs p{(const float*)x, ldx, op, M, K, kblocks, kept, vec};
    ce_note("int4_prepare_kernel");
    cudaError_t e = ce_launch(int4_prepare_kernel, dim3(tiles * 8), dim3(256), 0, (cudaStream_t)stream, p);
    if (e == cudaSuccess) {
        GemmArgs a{(const unsigned char*)w, op, out, ldo, M, N, kblocks, tiles, mode, gated};
        e = kept == 32 ? launch_tiles<32>(a, row_tiles, (cudaStream_t)stream) : launch_tiles<64>(a, row_tiles, (cudaStream_t)stream);
    }
    if (e != cudaSuccess) { (void)cudaGetLastError(); return ce_fail(CE_ERR_CUDA, "int4_gemm: %s", cudaGetErrorString(e)); }
    return ce_check_launch("int4_gemm");
}
