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

template <typename T>
__device__ __forceinline__ void finish(void* out, size_t at, int mode, float v, float u) {
    switch (mode) {
        case STORE_F32: ((float*)out)[at] = v; break;
        case ACCUM_F32: ((float*)out)[at] += v; break;
        case SWIGLU: CeType<T>::store((T*)out + at, ce_silu_glu(v, u)); break;
        case RELUGLU: CeType<T>::store((T*)out + at, fmaxf(v, 0.f) * u); break;
        case RELU2: v = fmaxf(v, 0.f); CeType<T>::store((T*)out + at, v * v); break;
        default: CeType<T>::store((T*)out + at, v);
    }
}

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
        finish<T>(a.out, at, a.mode, v, u);
    }
}

// ---------------------------------------------------------------------------------------------
// Up to 16 tokens: a stream of weights past tokens that stay in registers.
//
// A block takes ``upb`` tiles of 16 rows (with a gate: pairs of tiles) and a slice of K; each of its 16 warps a run of up to KW blocks of 64
// columns of that slice.  A warp holds its run of all tokens as the second operand (laid out and scaled by itself: nothing to prepare, and one
// launch) and meets the rows' tiles one after another, each a run of bytes that one lane copies into the warp's ring ahead of time.  What the
// warps make of a tile is added up in their order, what the blocks of a cluster make of it (slices of K) in theirs, through shared memory.
// The copies begin before the kernels in front have ended: no kernel writes a weight (ops_int4.Int4Weight sees to that).
// ---------------------------------------------------------------------------------------------
constexpr int SW = 16;             // warps
constexpr uint32_t SPIN = 1u << 20;

struct StreamArgs {
    const void* x;
    const unsigned char* w;
    void* out;
    int* status;
    long long ldx;
    int M, N, K, kblocks, ldo, mode, up_tile, units, upb, slices, overlap, vec;
};

__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ bool wait_full(uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < SPIN; ++i) {
        uint32_t ok;
        asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                     : "=r"(ok) : "r"(smem_of(bar)), "r"(parity) : "memory");
        if (ok) return true;
        if (i > 256) __nanosleep(64);
    }
    return false;
}
__device__ __forceinline__ void copy_in(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_of(bar)), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_of(dst)), "l"(src), "r"(bytes), "r"(smem_of(bar)) : "memory");
}
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
    static constexpr int PART = SW * NT * 128 * 4;                            // bytes of one tile's sums of all warps
    static constexpr int ROOM = 227 * 1024 - 4096 - RING - 2 * PART;          // for the tiles' totals
    static constexpr int MOST = ROOM / (NT * 128 * 4);                        // tiles a block can take
    static constexpr size_t smem(int tiles) { return RING + 2 * PART + (size_t)tiles * NT * 128 * 4; }
};

template <typename T, int G, int NT, int KW, int HALVES>
__global__ void __launch_bounds__(SW * 32) int4_stream_kernel(StreamArgs a) {
    using Shape = StreamShape<T, G, NT, KW>;
    constexpr int P = sizeof(T) == 4 ? 2 : 1, TILE = Shape::TILE, STAGES = Shape::STAGES, GB = 64 / G;
    constexpr bool C8 = P == 2;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) uint64_t full[SW][STAGES];
    float* part = reinterpret_cast<float*>(smem + Shape::RING);               // [2][SW][NT][32 lanes][4]
    float* total = part + 2 * SW * NT * 128;                                  // [tiles of the block][NT][32 lanes][4]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, l = lane & 3;
    const int slice = blockIdx.x % a.slices, first = blockIdx.x / a.slices * a.upb, units = min(a.upb, a.units - first), its = units * HALVES;
    const int kb_begin = (int)((long long)a.kblocks * slice / a.slices), kb_end = (int)((long long)a.kblocks * (slice + 1) / a.slices);
    const int run = (kb_end - kb_begin + SW - 1) / SW, kb0 = min(kb_begin + warp * run, kb_end), count = min(run, kb_end - kb0);
    unsigned char* ring = smem + warp * (STAGES * Shape::STAGE);
    if (a.overlap) ce_pdl_launch_dependents();
    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < STAGES; ++s) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_of(&full[warp][s])));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    auto issue = [&](int it) {
        const int unit = first + it / HALVES, h = it % HALVES;
        if (lane == 0 && count > 0)
            copy_in(ring + it % STAGES * Shape::STAGE, a.w + ((size_t)(unit + h * a.up_tile) * a.kblocks + kb0) * TILE, count * TILE, &full[warp][it % STAGES]);
    };
    for (int it = 0; it < min(STAGES, its); ++it) issue(it);
    ce_pdl_wait();

    // ---- the warp's run of the tokens: lane (r, l) lays out token 8 nt + r, columns 8 l .. + 8 of every 32
    uint32_t xf[KW][NT][P][2][4];
    float sums[KW][GB][NT][2], back[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int t = nt * 8 + r;
        const T* src = (const T*)a.x + (size_t)t * a.ldx + kb0 * 64 + 8 * l;
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
        const float up = i4_row_scale(largest);
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
                for (int e = 0; e < 2; ++e) sums[k][g][nt][e] = __shfl_sync(0xffffffffu, sum[g], 4 * (2 * l + e)) * (1.0f / i4_unit<C8>);
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) back[nt][e] = i4_unit<C8> / __shfl_sync(0xffffffffu, up, 4 * (2 * l + e));
    }

    bool ok = true;
    int gone = 0;                                     // tiles whose copies this warp has waited for
    for (int it = 0; it < its; ++it) {
        float y[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) y[nt][0] = y[nt][1] = y[nt][2] = y[nt][3] = 0.f;
        if (ok && count > 0) {
            ok = wait_full(&full[warp][it % STAGES], (it / STAGES) & 1);
            if (ok) ++gone;
            else if (lane == 0) atomicExch(a.status, 59);
        }
#pragma unroll
        for (int k = 0; k < KW; ++k) {
            if (k >= count) break;
            const unsigned char* tile = ring + it % STAGES * Shape::STAGE + k * TILE;
            const uint4 w = *reinterpret_cast<const uint4*>(tile + lane * 16);
            uint32_t sa[GB], sb[GB];
#pragma unroll
            for (int g = 0; g < GB; ++g) {
                sa[g] = *reinterpret_cast<const uint32_t*>(tile + 512 + (r * GB + g) * 4);
                sb[g] = *reinterpret_cast<const uint32_t*>(tile + 512 + ((r + 8) * GB + g) * 4);
            }
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
                i4_pairs<C8, 0>(wa, e0, e2); i4_pairs<C8, 0>(wb, e1, e3);
                i4_pairs<C8, 8>(wa, o0, o2); i4_pairs<C8, 8>(wb, o1, o3);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        i4_mma(acc[nt][p], e0, e1, e2, e3, xf[k][nt][p][half][0], xf[k][nt][p][half][1]);
                        i4_mma(acc[nt][p], o0, o1, o2, o3, xf[k][nt][p][half][2], xf[k][nt][p][half][3]);
                    }
                if ((half * 32 + 32) % G == 0) {
                    const int g = half * 32 / G;
                    const float2 fa = i4_step_of<C8>(sa[g]), fb = i4_step_of<C8>(sb[g]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float c[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            c[e] = acc[nt][0][e];
                            if constexpr (P == 2) c[e] += acc[nt][1][e];
                        }
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            y[nt][e] = fmaf(fa.x, c[e], fmaf(fa.y, sums[k][g][nt][e], y[nt][e]));
                            y[nt][2 + e] = fmaf(fb.x, c[2 + e], fmaf(fb.y, sums[k][g][nt][e], y[nt][2 + e]));
                        }
                    }
                }
            }
        }
        __syncwarp();
        if (ok && it + STAGES < its) issue(it + STAGES);
        float* mine = part + (it & 1) * (SW * NT * 128) + warp * (NT * 128);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            *reinterpret_cast<float4*>(mine + nt * 128 + lane * 4) =
                make_float4(y[nt][0] * back[nt][0], y[nt][1] * back[nt][1], y[nt][2] * back[nt][0], y[nt][3] * back[nt][1]);
        __syncthreads();
        // the warps' sums, in their order; four warps after another take the turn (the buffer is written again two tiles later, behind the
        // next tile's barrier)
        const int turn = (warp + SW - it * 4 * NT % SW) % SW;
        if (turn < 4 * NT) {
            const float* from = part + (it & 1) * (SW * NT * 128) + turn * 32 + lane;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < SW; ++w) v += from[w * (NT * 128)];
            total[it * (NT * 128) + turn * 32 + lane] = v;
        }
    }
    // a wait that gave up leaves copies in flight: they are waited for, with a limit, before the block may end
    if (!ok)
        for (int i = gone; i < min(gone + STAGES, its); ++i) wait_full(&full[warp][i % STAGES], (i / STAGES) & 1);
    if (a.slices > 1) cluster_sync();
    else __syncthreads();
    const int outs = units * a.M * 16;
    for (int o = threadIdx.x + slice * (SW * 32); o < outs; o += a.slices * (SW * 32)) {
        const int row = o & 15, rest = o >> 4, u = rest / a.M, t = rest - u * a.M, n = (first + u) * 16 + row;
        const int at = (t >> 3) * 128 + ((row & 7) * 4 + ((t & 7) >> 1)) * 4 + (row >> 3) * 2 + (t & 1);
        float v[2] = {0.f, 0.f};
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            const float* p = total + (u * HALVES + h) * (NT * 128) + at;
            if (a.slices == 1) v[h] = *p;
            else
                for (int s = 0; s < a.slices; ++s) v[h] += load_cluster(smem_of(p), s);
        }
        if (n < a.N) finish<T>(a.out, (size_t)t * a.ldo + n, a.mode, v[0], v[1]);
    }
    if (a.slices > 1) cluster_sync();                 // nobody leaves while its totals are read
}

// Returns 1 where the sizes are not this kernel's.
template <typename T, int G, int NT, int HALVES>
int launch_stream(StreamArgs a, cudaStream_t stream) {
    constexpr int P = sizeof(T) == 4 ? 2 : 1, KW = 4 / (NT * P);
    using Shape = StreamShape<T, G, NT, KW>;
    auto kernel = int4_stream_kernel<T, G, NT, KW, HALVES>;
    // slices of K: as few as the registers ask for; more where there are fewer tiles than SMs, down to 1,024 columns a slice
    const int sms = ce_sm_count();
    int slices = (a.kblocks + SW * KW - 1) / (SW * KW);
    while (slices < 8 && a.units * slices * 3 < sms * 2 && a.kblocks / (slices + 1) >= 16) ++slices;
    if (slices > 8) return 1;
    static std::atomic<unsigned long long> done{0};
    cudaError_t e = ce_allow_smem(done, kernel, Shape::smem(Shape::MOST));
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
        cfg.dynamicSmemBytes = Shape::smem(Shape::MOST);
        static CeRoom room[9];
        most = ce_clusters_at_once(room[slices], kernel, cfg);
        if (most < 1) return 1;
    }
    a.slices = slices;
    a.upb = min((a.units + most - 1) / most, Shape::MOST / HALVES);
    const int groups = (a.units + a.upb - 1) / a.upb;
    a.overlap = (slices == 1 || groups <= most) && ce_pdl_enabled();
    cfg.gridDim = dim3((unsigned)(groups * slices));
    cfg.dynamicSmemBytes = Shape::smem(a.upb * HALVES);
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
int launch_stream_tiles(const StreamArgs& a, int tiles, bool gated, cudaStream_t stream) {
    if (tiles == 1) return gated ? launch_stream<T, G, 1, 2>(a, stream) : launch_stream<T, G, 1, 1>(a, stream);
    return gated ? launch_stream<T, G, 2, 2>(a, stream) : launch_stream<T, G, 2, 1>(a, stream);
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

// Whether the stream of weights takes these sizes: up to 16 tokens, K within the registers of 8 blocks
bool streamed(int dtype, int M, int K) {
    const int tiles = (M + 7) / 8, nt_p = tiles * pieces(dtype);
    return tiles <= 2 && (K + 63) / 64 <= 8 * SW * (4 / nt_p);
}

}  // namespace

// float32 words of scratch memory (0: none) for a product of M tokens and K columns
extern "C" long long ce_int4_gemm_scratch(int dtype, int M, int K, int group) {
    if (streamed(dtype, M, K)) return 0;
    const long long tiles = (M + 7) / 8, kblocks = (K + 63) / 64;
    return kblocks * tiles * pieces(dtype) * 256 + kblocks * (64 / (group < 64 ? group : 64)) * tiles * 8 + tiles * 8;
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
    const long long ldx = c->ldx;
    const int dtype = (int)c->dtype, ldo = (int)c->ldo, M = (int)c->M, N = (int)c->N, K = (int)c->K, group = (int)c->group, mode = (int)c->mode;
    if (!x || !w || !out) return ce_fail(CE_ERR_ARG, "int4_gemm: null pointer");
    if (dtype != CE_F32 && dtype != CE_BF16) return ce_fail(CE_ERR_ARG, "int4_gemm: unknown dtype %d", dtype);
    if (group != 32 && group != 64 && group != 128) return ce_fail(CE_ERR_SIZE, "int4_gemm: group %d (32, 64 or 128)", group);
    if (mode < STORE || mode > RELU2) return ce_fail(CE_ERR_SIZE, "int4_gemm: epilogue %d is not one of this product's", mode);
    if (M < 0 || M > 64 || N < 1 || K < 1 || K % group || ldx < K || ldo < N)
        return ce_fail(CE_ERR_SIZE, "int4_gemm: %d tokens (at most 64), %d rows of %d (a multiple of the group)", M, N, K);
    if (((uintptr_t)w & 15) || ((uintptr_t)scratch & 15)) return ce_fail(CE_ERR_ARG, "int4_gemm: the weight or the scratch memory is not aligned to 16 bytes");
    if (M == 0) return CE_OK;
    const int kept = group < 64 ? group : 64, tiles = (M + 7) / 8, kblocks = (K + 63) / 64;
    const bool gated = mode == SWIGLU || mode == RELUGLU;
    const int el = dtype == CE_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)x % (4 * el)) == 0 && ldx % 4 == 0;
    if (!scratch) {
        if (!streamed(dtype, M, K)) return ce_fail(CE_ERR_ARG, "int4_gemm: these sizes need scratch memory");
        StreamArgs a{x, (const unsigned char*)w, out, c->status, ldx, M, N, K, kblocks, ldo, mode, (N + 15) / 16, (N + 15) / 16, 0, 0, 0, vec};
        const int code = dtype == CE_F32 ? (kept == 32 ? launch_stream_tiles<float, 32>(a, tiles, gated, (cudaStream_t)stream)
                                                       : launch_stream_tiles<float, 64>(a, tiles, gated, (cudaStream_t)stream))
                                         : (kept == 32 ? launch_stream_tiles<__nv_bfloat16, 32>(a, tiles, gated, (cudaStream_t)stream)
                                                       : launch_stream_tiles<__nv_bfloat16, 64>(a, tiles, gated, (cudaStream_t)stream));
        return code == 1 ? ce_fail(CE_ERR_SIZE, "int4_gemm: no room for clusters on this device") : code;
    }
    Operand op;
    op.frag = (uint32_t*)scratch;
    op.sums = scratch + (size_t)kblocks * tiles * pieces(dtype) * 256;
    op.back = op.sums + (size_t)kblocks * (64 / kept) * tiles * 8;
    PrepareArgs p{x, ldx, op, M, K, kblocks, kept, vec};
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
