// Products of up to 64 bfloat16 tokens - the stream of weights (int4_gemm.cu) takes up to 16 - with a weight held in 4 bits (int4.cuh) on the 5th-generation tensor cores.
//
//   out[t, n] = sum_g (s_ng (x_tg . (c_ng - 8)) + (z_ng + 8 s_ng) sum x_tg)
//
// A block takes 128 rows of the weight (8 tiles of 16) and a slice of K; blocks of a cluster share K.  For each group of columns, tcgen05.mma forms
// the codes' products with all tokens in a piece of tensor memory of its own; eight warps (a row and half of the tokens a lane) read it back and
// add it to their sums in float32, times the row's step: no value of W is ever rounded, and what is read back is as much work as the products are.
// The second term is a product too, of 4 columns a group, added up in tensor memory: (s, z, s, z) with the groups' sums in two float16 pieces
// (8 hi, hi, 8 lo, lo).  (Read from shared memory and added in registers it takes 256 of the 650 cycles of a group: a whole warp's load of the
// same 16 bytes occupies the pipe as long as one of 512.)  Eight warps turn codes into float16 integers (c - 8, the even ones, 16 (c - 8), the odd:
// the tokens are laid out to match), one issues the products, one the copies of codes - before the tokens are there - and one those of tokens.
// Slices' sums are added in their order through shared memory.  The parts hand each other 128 columns at a time.
//
// 64 tokens x 12,288 columns x 4,096 rows take 29 us in groups of 32, 25.5 in groups of 64 (9 tokens: 26 and 24): what bounds it is the chain of
// hand-overs - 1,300 cycles for 128 columns, of which the products take some 300 - and the 10 us before the first and behind the last of them
// (tokens prepared, slices joined), neither memory (5 us) nor the tensor cores.  The 16-bit product of these sizes takes no longer (gemm_tc.cu:
// past cold weights 24 to 30 us for 17 to 64 tokens, this one 27 to 34): a 4-bit weight of so many tokens saves memory, not time.
//
// The tokens come prepared (int4_tokens_kernel): each brought into [2^14, 2^15) by a power of two and rounded to float16 - exact for bfloat16 down
// to 2^-27 of the token's largest - as the second operands' images, swizzle included.
#include "int4.cuh"
#include "int4_ring.h"

namespace {

constexpr int ROWS = 128, MAKERS = 8, ADDERS = 8, FIRST = 3, THREADS = 32 * (FIRST + MAKERS + ADDERS);
constexpr int RUN = 4, RAW = 4, AS = 3, DS = 2;             // blocks of 64 columns a copy of codes; stages of codes, of operands (two blocks each), of sums (two groups each)
constexpr int SUM_AT = 64 * 2 * DS, A_AT = SUM_AT + 64;      // columns of tensor memory: products, the second term, operands
static_assert(A_AT + 64 * AS <= 512, "tensor memory");

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(i4_smem(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(i4_smem(bar)) : "memory");
}
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// one lane of a whole warp issues, always the same one
__device__ __forceinline__ void umma(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n.reg .pred p, q;\nelect.sync _|q, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d_tmem), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
// the same with the first operand in tensor memory: a row a lane, two values a column
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n.reg .pred p, q;\nelect.sync _|q, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
                 ::"r"(d_tmem), "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
// 16 rows of 32 columns: a lane's words of rows lane / 4 (even ones) and 8 on (odd ones), every fourth column
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&q)[16]) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 ::"r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3]), "r"(q[4]), "r"(q[5]), "r"(q[6]), "r"(q[7]),
                   "r"(q[8]), "r"(q[9]), "r"(q[10]), "r"(q[11]), "r"(q[12]), "r"(q[13]), "r"(q[14]), "r"(q[15]), "r"(taddr) : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\n@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}"
                 ::"r"(i4_smem(bar)) : "memory");
}
// N columns of this lane's row (16 or 32): under way until tmem_landed
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&q)[N]) {
    if constexpr (N == 16)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                     : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7]),
                       "=r"(q[8]), "=r"(q[9]), "=r"(q[10]), "=r"(q[11]), "=r"(q[12]), "=r"(q[13]), "=r"(q[14]), "=r"(q[15])
                     : "r"(taddr));
    else
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                     "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                     : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7]),
                       "=r"(q[8]), "=r"(q[9]), "=r"(q[10]), "=r"(q[11]), "=r"(q[12]), "=r"(q[13]), "=r"(q[14]), "=r"(q[15]),
                       "=r"(q[16]), "=r"(q[17]), "=r"(q[18]), "=r"(q[19]), "=r"(q[20]), "=r"(q[21]), "=r"(q[22]), "=r"(q[23]),
                       "=r"(q[24]), "=r"(q[25]), "=r"(q[26]), "=r"(q[27]), "=r"(q[28]), "=r"(q[29]), "=r"(q[30]), "=r"(q[31])
                     : "r"(taddr));
}
// (the registers pass through, so that nothing reads them before)
template <int N>
__device__ __forceinline__ void tmem_landed(uint32_t (&q)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(q[i]));
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 load_cluster(uint32_t local, int rank) {
    uint32_t at;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(local), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

enum { STORE = 0, STORE_F32 = 1, ACCUM_F32 = 2, SWIGLU = 3, RELUGLU = 4, RELU2 = 5 };

// A K-major operand without a swizzle: 8 rows of 16 bytes side by side, groups of 8 rows 128 bytes apart, the second 8 columns ``ahead`` bytes on
__device__ __forceinline__ uint64_t desc_plain(uint32_t addr, uint32_t ahead) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(ahead >> 4) << 16) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}
__device__ __forceinline__ void finish(void* out, size_t at, int mode, float v, float up) {
    __nv_bfloat16* half = (__nv_bfloat16*)out;
    switch (mode) {
        case STORE_F32: ((float*)out)[at] = v; break;
        case ACCUM_F32: ((float*)out)[at] += v; break;
        case SWIGLU: half[at] = __float2bfloat16_rn(ce_silu_glu(v, up)); break;
        case RELUGLU: half[at] = __float2bfloat16_rn(i4_relu(v) * up); break;
        case RELU2: v = i4_relu(v); half[at] = __float2bfloat16_rn(v * v); break;
        default: half[at] = __float2bfloat16_rn(v);
    }
}

// bytes of a block of 64 columns of the prepared tokens: the operand's image, then 16 bytes a token of the groups' sums (2^-9 of them, of 64
// values below 2^15 each, is what float16 holds eight times of)
__host__ __device__ constexpr int tokens_bytes(int tokens) { return tokens * 144; }
constexpr float SUMS = 512.0f;

struct TokensArgs {
    const __nv_bfloat16* x;
    unsigned char* to;             // [kblocks + 1][tokens_bytes], the last of zeros, then float32 [tokens]: what a token's sums are multiplied by at the end
    long long ld;
    int M, K, kblocks, tokens, group, vec;
};
// one block a token (of 32 or 64: those beyond M are zeros); up to 16,384 columns are read once and kept in registers
__global__ void __launch_bounds__(1024) int4_tokens_kernel(TokensArgs a) {
    ce_pdl_begin();
    __shared__ float scratch[32];
    const int t = blockIdx.x, per_block = tokens_bytes(a.tokens);
    const bool real = t < a.M;
    const __nv_bfloat16* src = a.x + (size_t)(real ? t : 0) * a.ld;
    auto load8 = [&](int c) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (!real || c >= a.K) return u;              // (K is a multiple of 32)
        if (a.vec) return *reinterpret_cast<const uint4*>(src + c);
        const unsigned short* p = reinterpret_cast<const unsigned short*>(src + c);
        u.x = p[0] | (uint32_t)p[1] << 16; u.y = p[2] | (uint32_t)p[3] << 16; u.z = p[4] | (uint32_t)p[5] << 16; u.w = p[6] | (uint32_t)p[7] << 16;
        return u;
    };
    constexpr int KEPT = 2, STEP = 1024 * 8;
    uint4 kept[KEPT];
    float largest = 0.f;
    bool finite = true;
    auto look = [&](uint4 u) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p = fabsf(__uint_as_float(w[i] << 16)), q = fabsf(__uint_as_float(w[i] & 0xffff0000u));
            largest = fmaxf(largest, fmaxf(p, q));
            finite = finite && p <= 3.402823466e38f && q <= 3.402823466e38f;
        }
    };
#pragma unroll
    for (int i = 0; i < KEPT; ++i) kept[i] = load8(threadIdx.x * 8 + i * STEP);
#pragma unroll
    for (int i = 0; i < KEPT; ++i) look(kept[i]);
    for (int c = threadIdx.x * 8 + KEPT * STEP; c < a.K; c += STEP) look(load8(c));
    largest = ce_block_max(finite ? largest : INFINITY, scratch);
    const float up = i4_row_scale(largest);
    if (threadIdx.x == 0) reinterpret_cast<float*>(a.to + (size_t)(a.kblocks + 1) * per_block)[t] = 1.0f / up;
    auto put = [&](int c, uint4 u) {
        if (c >= (a.kblocks + 1) * 64) return;              // (8 threads, a block of 64 columns, together)
        const uint32_t in[4] = {u.x, u.y, u.z, u.w};
        float y[8], sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) { y[2 * i] = __uint_as_float(in[i] << 16) * up; y[2 * i + 1] = __uint_as_float(in[i] & 0xffff0000u) * up; }
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float f = i & 1 ? 0.0625f : 1.0f, b = i & 1 ? 16.0f : 1.0f;          // odd codes come 16 times too large
            w[i] = i4_pack(y[i] * f, y[i + 4] * f);
            const float2 got = i4_unpack(w[i]);
            sum += (got.x + got.y) * b;
        }
        unsigned char* block = a.to + (size_t)(c >> 6) * per_block;
        // columns in the order in which tmem_st lays the codes out: these words are every fourth of 16
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint32_t*>(block + t * 128 + ((((c & 32) / 8 + i) ^ (t & 7)) << 4) + ((c >> 3) & 3) * 4) = w[i];
        const unsigned here = 0xffu << (threadIdx.x & 24);
        sum += __shfl_xor_sync(here, sum, 1);
        sum += __shfl_xor_sync(here, sum, 2);
        if (a.group == 64) sum += __shfl_xor_sync(here, sum, 4);
        if (c % a.group == 0) {
            sum *= 1.0f / SUMS;
            const float hi = __half2float(__float2half_rn(sum)), lo = sum - hi;
            const uint32_t first = i4_pack(8.0f * hi, hi), second = i4_pack(8.0f * lo, lo);
            unsigned char* sums = block + a.tokens * 128 + (t >> 3) * 128 + (t & 7) * 16;
            if (a.group == 64) *reinterpret_cast<uint4*>(sums) = make_uint4(first, second, 0, 0);
            else *reinterpret_cast<uint2*>(sums + (c & 32) / 4) = make_uint2(first, second);
        }
    };
#pragma unroll
    for (int i = 0; i < KEPT; ++i) put(threadIdx.x * 8 + i * STEP, kept[i]);
    for (int c = threadIdx.x * 8 + KEPT * STEP; c < (a.kblocks + 1) * 64; c += STEP) put(c, load8(c));
}

struct Args {
    const unsigned char *w, *x;    // x: as int4_tokens_kernel leaves it
    const float* back;
    void* out;
    int* status;
    long long ldo;
    int M, N, kblocks, units, slices, mode, gated, overlap;           // units: tiles of 16 rows
};

template <int G, int TOKENS>
struct Shape {
    static constexpr int TILE = i4_weight_tile_bytes(G), XB = tokens_bytes(TOKENS), XSTEP = (XB + 1023) / 1024 * 1024;     // XSTEP: of a block in shared memory
    static constexpr uint32_t X = 0, Z = AS * 2 * XSTEP, CODES = Z + AS * ROWS * 32, BARS = CODES + RAW * 8 * RUN * TILE;
    static constexpr uint32_t BYTES = BARS + 8 * (2 * RAW + 2 * AS + 2 * DS + 2);
    static_assert(TOKENS * ROWS * 4 <= BARS, "sums");                   // of the slices, token by token, in the place of the stages
};

template <int G, int TOKENS>
__global__ void __launch_bounds__(THREADS) int4_gemm_tc_kernel(Args a) {
    using S = Shape<G, TOKENS>;
    constexpr int TILE = S::TILE, GB = 64 / G;
    extern __shared__ __align__(1024) unsigned char sm[];
    const uint32_t base = i4_smem(sm);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + S::BARS);
    uint64_t *raw_full = bars, *raw_empty = bars + RAW, *full = raw_empty + RAW, *empty = full + AS;
    uint64_t *d_full = empty + AS, *d_empty = d_full + DS;
    uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(d_empty + DS);
    uint64_t* drained = d_empty + DS + 1;               // all products have ended
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int slice = blockIdx.x % a.slices, unit0 = blockIdx.x / a.slices * 8, tiles = min(8, a.units - unit0);
    const int kb_begin = (int)((long long)a.kblocks * slice / a.slices), kb_end = (int)((long long)a.kblocks * (slice + 1) / a.slices);
    const int n_kb = kb_end - kb_begin, runs = (n_kb + RUN - 1) / RUN, pairs = (n_kb + 1) / 2;
    if ((base & 1023u) != 0) {                          // cannot happen with dynamic shared memory alone; refuse rather than mis-swizzle
        if (threadIdx.x == 0) atomicCAS(a.status, 0, 58);
        if (a.slices > 1) { cluster_sync(); cluster_sync(); }
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < RAW; ++i) { mbar_init(&raw_full[i], 1); mbar_init(&raw_empty[i], MAKERS + ADDERS); }
        for (int i = 0; i < AS; ++i) { mbar_init(&full[i], MAKERS + 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < DS; ++i) { mbar_init(&d_full[i], 1); mbar_init(&d_empty[i], ADDERS); }
        mbar_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // codes of runs of columns, by one lane (a weight is never still being written here: int4_weight_done_kernel)
    auto copy_codes = [&](int run) {
        const int count = min(RUN, n_kb - run * RUN);
        uint64_t* bar = &raw_full[run % RAW];
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(i4_smem(bar)), "r"(tiles * count * TILE) : "memory");
        for (int u = 0; u < tiles; ++u)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                         ::"r"(base + S::CODES + (run % RAW * 8 + u) * RUN * TILE),
                         "l"(a.w + ((size_t)(unit0 + u) * a.kblocks + kb_begin + run * RUN) * TILE), "r"(count * TILE), "r"(i4_smem(bar)) : "memory");
    };
    if (warp == 1 && lane == 0)
        for (int run = 0; run < min(runs, RAW); ++run) copy_codes(run);
    __syncwarp();
    ce_pdl_wait();                                      // (before tensor memory is taken: a neighbour that this grid waits for may need it)
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(i4_smem(&tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (a.overlap) ce_pdl_launch_dependents();
    const uint32_t tmem = tmem_slot;
    constexpr int PART = TOKENS / 2;                    // tokens of a lane that adds
    float y[PART];
    bool ok = true;

    if (warp == 0) {
        // ---- the products: a group's of all tokens into the next piece of tensor memory
        const uint32_t idesc = (1u << 4) | ((uint32_t)(TOKENS >> 3) << 17) | (8u << 24);
        for (int i = 0; i < pairs && ok; ++i) {
            ok = i4_warp_wait(&full[i % AS], (i / AS) & 1);
            if (!ok) break;
            const uint32_t x_addr = base + S::X + i % AS * 2 * S::XSTEP, a_at = tmem + A_AT + i % AS * 64;
            const int groups = min(2, n_kb - 2 * i) * GB;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            umma(tmem + SUM_AT, desc_plain(base + S::Z + i % AS * ROWS * 32, ROWS * 16), desc_plain(x_addr + TOKENS * 128, S::XSTEP), idesc, i > 0 ? 1u : 0u);
#pragma unroll
            for (int u = 0; u < GB; ++u) {              // two groups at a time
                const int d = i * GB + u;
                if (2 * u >= groups) break;
                if (d >= DS) ok = ok && i4_warp_wait(&d_empty[d % DS], (d / DS - 1) & 1);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int g = 2 * u; g < 2 * u + 2; ++g) {
                    if (g >= groups) break;
#pragma unroll
                    for (int kk = 0; kk < G / 16; ++kk) {
                        const int k16 = g % GB * (G / 16) + kk;
                        umma_ts(tmem + d % DS * 128 + (g & 1) * 64, a_at + g / GB * 32 + k16 * 8, desc_kmajor(x_addr + g / GB * S::XSTEP + k16 * 32), idesc, kk > 0 ? 1u : 0u);
                    }
                }
                umma_commit(&d_full[d % DS]);
            }
            umma_commit(&empty[i % AS]);
        }
        if (!ok && lane == 0) atomicCAS(a.status, 0, 51);
        // (whoever gave up: no product is under way when tensor and shared memory become another's)
        umma_commit(drained);
        i4_warp_wait(drained, 0);
    } else if (warp == 1) {
        // ---- the copies of codes, RUN blocks of columns at a time
        if (lane == 0) {
            int run = min(runs, RAW);
            for (; run < runs && ok; ++run) {
                ok = i4_wait(&raw_empty[run % RAW], (run / RAW - 1) & 1);
                if (ok) copy_codes(run);
                else break;
            }
            if (!ok) atomicCAS(a.status, 0, 52);
            // (whoever gave up: what is on its way lands before the stages are others')
            i4_drain<RAW>(run, [&](int at, uint32_t parity) { i4_wait(&raw_full[at], parity); });
        }
        __syncwarp();
    } else if (warp == 2) {
        // ---- the copies of tokens, two blocks of columns at a time
        if (lane == 0) {
            int i = 0;
            for (; i < pairs && ok; ++i) {
                if (i >= AS) ok = i4_wait(&empty[i % AS], (i / AS - 1) & 1);
                if (!ok) break;
                uint64_t* bar = &full[i % AS];
                // (a last block alone: the one behind it comes along, for a product with zeros)
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(i4_smem(bar)), "r"(2 * S::XB) : "memory");
                for (int k = 0; k < 2; ++k)
                    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                                 ::"r"(base + S::X + (i % AS * 2 + k) * S::XSTEP), "l"(a.x + (size_t)(kb_begin + 2 * i + k) * S::XB), "r"(S::XB), "r"(i4_smem(bar))
                                 : "memory");
            }
            if (!ok) atomicCAS(a.status, 0, 52);
            // (a stage that its makers gave up is waited for as long as a wait may take: longer than a copy does)
            i4_drain<AS>(i, [&](int at, uint32_t parity) { i4_wait(&full[at], parity); });
        }
        __syncwarp();
    } else if (warp < FIRST + MAKERS) {
        // ---- codes into float16 integers: two tiles of 16 rows of a block of columns a warp
        const int maker = warp & 3, k = (warp - FIRST) >> 2;        // (whose lanes of tensor memory these are; which block of a pair)
        for (int i = 0; i < pairs && ok; ++i) {
            const int run = 2 * i / RUN;
            if (2 * i % RUN == 0) ok = i4_warp_wait(&raw_full[run % RAW], (run / RAW) & 1);
            if (!ok) break;
            // (an odd last block: the second of the pair is what lay there, for no product)
            uint4 w[2];
#pragma unroll
            for (int u = 0; u < 2; ++u)
                w[u] = *reinterpret_cast<const uint4*>(sm + S::CODES + ((run % RAW * 8 + maker * 2 + u) * RUN + 2 * i % RUN + k) * TILE + lane * 16);
            // of row 32 maker + lane: (s, z, s, z) a group
            const uint32_t* step = reinterpret_cast<const uint32_t*>(
                sm + S::CODES + ((run % RAW * 8 + maker * 2 + (lane >> 4)) * RUN + 2 * i % RUN + k) * TILE + 512 + (lane & 15) * GB * 4);
            uint4 z = make_uint4(0, 0, 0, 0);
            if (2 * i + k < n_kb) { z.x = z.y = step[0]; if (GB == 2) z.z = z.w = step[GB - 1]; }
            if (2 * i % RUN == RUN - 2 || i == pairs - 1) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&raw_empty[run % RAW]);
            }
            if (i >= AS) ok = i4_warp_wait(&empty[i % AS], (i / AS - 1) & 1);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            *reinterpret_cast<uint4*>(sm + S::Z + i % AS * ROWS * 32 + k * ROWS * 16 + (maker * 32 + lane) * 16) = z;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t v[16];
#pragma unroll
                for (int e = 0; e < 4; ++e) {           // words of rows r and r + 8, first and second 32 columns
                    const uint32_t word = e == 0 ? w[u].x : e == 1 ? w[u].y : e == 2 ? w[u].z : w[u].w;
                    uint32_t* at = v + (e >> 1) * 8 + (e & 1);
                    i4_pairs<true, 0>(word, at[0], at[2]);
                    i4_pairs<true, 8>(word, at[4], at[6]);
                }
                tmem_st(tmem + A_AT + i % AS * 64 + k * 32 + ((uint32_t)(maker * 32 + u * 16) << 16), v);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[i % AS]);
        }
        if (!ok && lane == 0) atomicCAS(a.status, 0, 53);
    } else {
        // ---- the sums: a row and half of the tokens a lane, two groups at a time
        const int quad = warp & 3, row = quad * 32 + lane, unit = row >> 4, first = (warp - FIRST - MAKERS) / 4 * PART;
        const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16) + first;
#pragma unroll
        for (int t = 0; t < PART; ++t) y[t] = 0.f;
        for (int i = 0; i < pairs && ok; ++i) {
            const int run = 2 * i / RUN, groups = min(2, n_kb - 2 * i) * GB;
            if (2 * i % RUN == 0) ok = i4_warp_wait(&raw_full[run % RAW], (run / RAW) & 1);
            if (!ok) break;
            uint32_t step[2 * GB];
#pragma unroll
            for (int g = 0; g < 2 * GB; ++g)
                step[g] = reinterpret_cast<const uint32_t*>(sm + S::CODES + ((run % RAW * 8 + unit) * RUN + 2 * i % RUN + g / GB) * TILE + 512 + (row & 15) * GB * 4)[g % GB];
            if (2 * i % RUN == RUN - 2 || i == pairs - 1) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&raw_empty[run % RAW]);
            }
#pragma unroll
            for (int u = 0; u < GB; ++u) {
                const int d = i * GB + u;
                if (2 * u >= groups) break;
                ok = ok && i4_warp_wait(&d_full[d % DS], (d / DS) & 1);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t got[2][PART];
#pragma unroll
                for (int g = 0; g < 2; ++g) tmem_ld<PART>(from + d % DS * 128 + g * 64, got[g]);     // (of a last group alone, the second is not used)
#pragma unroll
                for (int g = 0; g < 2; ++g) tmem_landed<PART>(got[g]);
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&d_empty[d % DS]);
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    if (2 * u + g >= groups) break;
                    const float f = i4_step_of<false>(step[2 * u + g]).x;
#pragma unroll
                    for (int t = 0; t < PART; t += 2) {
                        const float2 p = __ffma2_rn(make_float2(f, f), make_float2(__uint_as_float(got[g][t]), __uint_as_float(got[g][t + 1])), make_float2(y[t], y[t + 1]));
                        y[t] = p.x; y[t + 1] = p.y;
                    }
                }
            }
        }
        // the second term (its last product was issued before the last group's)
        uint32_t got[PART];
        tmem_ld<PART>(from + SUM_AT, got);
        tmem_landed<PART>(got);
#pragma unroll
        for (int t = 0; t < PART; ++t) y[t] = fmaf(SUMS, __uint_as_float(got[t]), y[t]);
        if (!ok && lane == 0) atomicCAS(a.status, 0, 54);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();                                    // the stages are free: the rows' sums take their place
    if (warp == 0) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
    float* total = reinterpret_cast<float*>(sm);
    if (warp >= FIRST + MAKERS) {
        const int row = (warp & 3) * 32 + lane, first = (warp - FIRST - MAKERS) / 4 * PART;
#pragma unroll
        for (int t = 0; t < PART; ++t) total[(first + t) * ROWS + row] = y[t];
    }
    if (a.slices > 1) cluster_sync();
    else __syncthreads();
    // four rows' results of a token: the slices' sums in their order (all of them asked for at once), what was scaled scaled back; a block takes
    // every ``slices``-th run of results
    const int fours = a.gated ? 16 : ROWS / 4;
    for (int o = slice * THREADS + threadIdx.x; o < fours * a.M; o += a.slices * THREADS) {
        const int t = a.gated ? o >> 4 : o >> 5, i = (o & (fours - 1)) * 4, row = a.gated ? (i >> 3) * 16 + (i & 7) : i;
        const int n = unit0 * (a.gated ? 8 : 16) + i;
        const float back = a.back[t];
        float* at = total + t * ROWS + row;
        float v[4] = {0.f, 0.f, 0.f, 0.f}, u[4] = {0.f, 0.f, 0.f, 0.f};
        auto add = [](float (&x)[4], float4 y) { x[0] += y.x; x[1] += y.y; x[2] += y.z; x[3] += y.w; };
        if (a.slices > 1) {
            float4 vs[8], us[8];
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                vs[s] = us[s] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (s < a.slices) {
                    vs[s] = load_cluster(i4_smem(at), s);
                    if (a.gated) us[s] = load_cluster(i4_smem(at + 8), s);
                }
            }
#pragma unroll
            for (int s = 0; s < 8; ++s) { add(v, vs[s]); add(u, us[s]); }
        } else {
            add(v, *reinterpret_cast<const float4*>(at));
            if (a.gated) add(u, *reinterpret_cast<const float4*>(at + 8));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (n + k < a.N) finish(a.out, (size_t)t * a.ldo + n + k, a.mode, v[k] * back, u[k] * back);
    }
    if (a.slices > 1) cluster_sync();                   // nobody leaves while its sums are read
}

template <int G, int TOKENS>
int run(TokensArgs p, Args a, cudaStream_t stream) {
    using S = Shape<G, TOKENS>;
    auto kernel = int4_gemm_tc_kernel<G, TOKENS>;
    // more than it uses: beside a block of another stream's kernel that holds tensor memory, one of this kernel would wait for it inside its
    // cluster, and that one's cluster, elsewhere, for a block that waits for this kernel's
    constexpr int SMEM = 220 * 1024;
    static_assert(S::BYTES <= SMEM, "shared memory");
    static std::atomic<unsigned long long> done{0};
    cudaError_t e = ce_allow_smem(done, kernel, SMEM);
    if (e == cudaSuccess) {
        ce_note("int4_tokens_kernel");
        e = ce_launch(int4_tokens_kernel, dim3(TOKENS), dim3(1024), 0, stream, p);
    }
    if (e == cudaSuccess) {
        // as many slices of K as fill the chip, of 8 blocks of 64 columns at least
        const int blocks = (a.units + 7) / 8, sms = ce_sm_count();
        int slices = 1;
        while (slices < 8 && blocks * (slices + 1) <= sms && a.kblocks / (slices + 1) >= 8) ++slices;
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[2];
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = SMEM;
        cfg.stream = stream;
        cfg.attrs = attr;
        a.overlap = ce_pdl_enabled();
        static CeRoom room[9];
        for (;; --slices) {
            cfg.numAttrs = 0;
            cfg.gridDim = dim3((unsigned)(blocks * slices));
            if (slices == 1) break;
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim = {(unsigned)slices, 1, 1};
            cfg.numAttrs = 1;
            if (blocks <= ce_clusters_at_once(room[slices], kernel, cfg)) break;       // (clusters that do not all run at once: fewer slices)
        }
        a.slices = slices;
        if (a.overlap) {
            attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
        }
        ce_note("int4_gemm_tc_kernel");
        e = cudaLaunchKernelEx(&cfg, kernel, a);
    }
    if (e != cudaSuccess) { (void)cudaGetLastError(); return ce_fail(CE_ERR_CUDA, "int4_gemm_tc: %s", cudaGetErrorString(e)); }
    return ce_check_launch("int4_gemm_tc");
}

}  // namespace

// float32 words of scratch memory for M tokens (at most 64) of K columns
long long ce_int4_gemm_tc_scratch(int M, int K) {
    const int tokens = M <= 32 ? 32 : 64;
    return (long long)((K + 63) / 64 + 1) * tokens_bytes(tokens) / 4 + tokens;
}

// The checks of ce_int4_gemm come first: it calls this.  scratch: on a 16-byte boundary; kept: columns of a group in the weight's tiles (32 or 64)
int ce_int4_gemm_tc(const void* x, long long ldx, const void* w, void* out, long long ldo, int M, int N, int K, int kept, int mode, float* scratch, int* status,
                    cudaStream_t stream) {
    const int tokens = M <= 32 ? 32 : 64, kblocks = (K + 63) / 64, gated = mode == SWIGLU || mode == RELUGLU;
    unsigned char* to = (unsigned char*)scratch;
    TokensArgs p{(const __nv_bfloat16*)x, to, ldx, M, K, kblocks, tokens, kept, ((uintptr_t)x & 15) == 0 && ldx % 8 == 0};
    Args a{(const unsigned char*)w, to, reinterpret_cast<const float*>(to + (size_t)(kblocks + 1) * tokens_bytes(tokens)), out, status, ldo, M, N, kblocks,
           gated ? (N + 7) / 8 : (N + 15) / 16, 1, mode, gated, 0};
    if (tokens == 32) return kept == 32 ? run<32, 32>(p, a, stream) : run<64, 32>(p, a, stream);
    return kept == 32 ? run<32, 64>(p, a, stream) : run<64, 64>(p, a, stream);
}
