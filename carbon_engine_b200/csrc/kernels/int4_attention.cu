// Attention over a paged cache held in 4 bits (int4.cuh): rows of queries against the tiles of 16 keys of one KV head.
//
// For a query row q and the keys j it sees, with group g of the channels:
//   S_j = scale sum_g (s_jg (q_g . c_jg) + z_jg sum q_g),   p_j = exp(S_j - max S),
//   out_g = sum_j (p_j s_jg c_jg + p_j z_jg) / sum_j p_j
// so the codes themselves are the operands of both products, and steps and minima never touch a value: a step scales a group's partial score
// (keys) or the probability (values), a minimum takes part in float32.  Keys (values' channels) are the 16 rows of mma.sync m16n8k16, query
// rows its 8 columns, which is how the heads of a group that share a KV head fill a tile.
//
// Roundings: a query row is brought into [2^14, 2^15) by a power of two and rounded to float16, which is exact for bfloat16 values down to 2^-27 of
// the row's largest (half of them divided by 16, for codes that come 16 times too large); float32 rows are two float16 pieces, 22 bits.  p_j s_jg is
// rounded to float16 (by 2^-11 of itself at most; two pieces for float32), scaled so that the largest probability times the largest step that the warp
// has met in any group lies near 2^10: sums of thousands of small weights keep their bits.  Below 2^-14 float16's steps are fixed, so that each key may
// err by 15 2^-34 of that largest step, in units of the largest probability: what a group with far smaller steps than its neighbours' loses.
// Everything else is float32.
//
// A block takes up to 8 or 16 rows (tokens by heads of the KV head) and a run of the keys; its 8 or 4 warps take tiles in turn, each with a
// ring of its own that one lane fills with bulk copies (a tile is one run of bytes in the page); warps, then blocks, are joined in a fixed order.
//
// 64 sequences of 8,192 keys of 8 KV heads of 128 take 135 us, 4.5 TB/s: bound by instructions (313 a tile a warp, the ALU pipe, which takes the codes
// apart, half busy, 2.2 instructions a cycle of an SM).  A block costs some 4 us to begin (place, queries, first tiles) and end (joins), which
// is what short and uneven requests are bound by (21 of 450 to 9,000 keys: 49 us of which 19.5 are the bytes').
#include "int4.cuh"

namespace {

constexpr int WARPS = 8;                       // of a block, at most
// tiles of a warp's ring: 4, or up to 6 where two blocks of an SM have room for it
constexpr int ring_tiles(int tile) { return 110592 / (WARPS * tile) < 4 ? 4 : 110592 / (WARPS * tile) > 6 ? 6 : 110592 / (WARPS * tile); }
constexpr int PAIR_UP_TO = 128;
constexpr float NOTHING = -3.402823466e38f;    // the maximum of no scores
constexpr float HEADROOM = 5.0f;               // scores may pass the running maximum by this many powers of two before it is moved
// From this magnitude of m on, float32's steps (0.5 and more) tell in what a weight comes out as: there, weights are cut to the HEADROOM that they
// may have (m is rounded down: none is lost).  Keys whose scores lie a few such steps below the largest may count for more than they should.
constexpr float COARSE = 0x1p22f;
constexpr float LOG2E = 1.4426950408889634f;

struct Args {
    const void* q;                 // [T, heads, d]: token stride q_stride, heads d apart
    void* out;                     // [T, heads, d] contiguous
    const unsigned char* pages;
    const int *seq_slot, *q_start, *ctx_len, *block_table, *tiles;
    int* status;
    float *part_o, *part_ml;       // splits > 1: [row block, split, rows, d], [row block, split, rows, 2]
    long long q_stride;
    int nh, nkv, page_size, max_pages, num_pages, window, splits, share, subs;    // share: tiles of a split; subs: row blocks of a sequence (or of a tile of 64 tokens)
    int vec, clustered, overlap;   // clustered: the splits of a row block are a cluster and join through shared memory
    float scale;
};

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// What a block works on: rows [row0, row0 + 8 NT) of the (token, head) pairs of tokens q0 .. of a sequence
struct Job {
    int b, slot, t0, token0, tokens, base, row0, kvh;        // base: position of token 0 of the tile
};
__device__ __forceinline__ Job job_of(const Args& a, int job, int rows) {
    Job j;
    const int sub = job % a.subs, rest = job / a.subs, i = rest / a.nkv;
    j.kvh = rest - i * a.nkv;
    int q0 = 0;
    if (a.tiles) { j.b = a.tiles[2 * i]; q0 = a.tiles[2 * i + 1]; }
    else j.b = i;
    const int start = a.q_start[j.b], n = a.q_start[j.b + 1] - start;
    j.slot = a.seq_slot[j.b];
    j.t0 = start + q0;
    j.tokens = min(a.tiles ? 64 : 1, n - q0);         // (none: a place of the batch that nobody took)
    j.base = a.ctx_len[j.b] - n + q0;
    j.row0 = sub * rows;
    return j;
}

template <typename T> struct Pieces;
template <> struct Pieces<__nv_bfloat16> { static constexpr int N = 1; };
template <> struct Pieces<float> { static constexpr int N = 2; };

// A lane's channels of a query row, 8 of every 32, as they were read
template <typename T, int CH> struct Raw;
template <int CH> struct Raw<__nv_bfloat16, CH> {
    uint2 w[CH][2];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int c = 0; c < CH; ++c) w[c][0] = w[c][1] = make_uint2(0, 0);
    }
    __device__ __forceinline__ void load(const __nv_bfloat16* src, bool vec) {
        const unsigned short* p = reinterpret_cast<const unsigned short*>(src);
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i, p += 4) {
                w[c][i] = vec ? *reinterpret_cast<const uint2*>(p) : make_uint2(p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16);
                if (i) p += 24;
            }
    }
    // the largest magnitude, infinity where one is not finite
    __device__ __forceinline__ float largest() const {
        __nv_bfloat162 most = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t v = (i & 1) ? w[c][i >> 1].y : w[c][i >> 1].x;
                most = __hmax2_nan(most, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&v)));
            }
        const float2 two = __bfloat1622float2(most);
        return two.x <= 3.402823466e38f && two.y <= 3.402823466e38f ? fmaxf(two.x, two.y) : INFINITY;
    }
    __device__ __forceinline__ float at(int c, int i) const {
        const uint32_t v = (i & 2) ? w[c][i >> 2].y : w[c][i >> 2].x;
        return __uint_as_float(i & 1 ? v & 0xffff0000u : v << 16);
    }
};
template <int CH> struct Raw<float, CH> {
    float4 w[CH][2];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int c = 0; c < CH; ++c) w[c][0] = w[c][1] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __device__ __forceinline__ void load(const float* p, bool vec) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i, p += 4) {
                w[c][i] = vec ? *reinterpret_cast<const float4*>(p) : make_float4(p[0], p[1], p[2], p[3]);
                if (i) p += 24;
            }
    }
    __device__ __forceinline__ float largest() const {
        float most = 0.f;
        bool finite = true;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) { const float x = fabsf(at(c, i)); most = fmaxf(most, x); finite = finite && x <= 3.402823466e38f; }
        return finite ? most : INFINITY;
    }
    __device__ __forceinline__ float at(int c, int i) const {
        const float4& v = w[c][i >> 2];
        return (i & 3) == 0 ? v.x : (i & 3) == 1 ? v.y : (i & 3) == 2 ? v.z : v.w;
    }
};

// (s, z) of one token's groups out of shared memory, as they lie: NG words
template <int NG>
__device__ __forceinline__ void load_steps(const unsigned char* p, uint32_t (&v)[NG]) {
    if constexpr (NG == 1) v[0] = *reinterpret_cast<const uint32_t*>(p);
    else if constexpr (NG == 2) { const uint2 x = *reinterpret_cast<const uint2*>(p); v[0] = x.x; v[1] = x.y; }
    else if constexpr (NG == 3 || NG == 6) {
#pragma unroll
        for (int i = 0; i < NG; ++i) v[i] = reinterpret_cast<const uint32_t*>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < NG / 4; ++i) {
            const uint4 x = reinterpret_cast<const uint4*>(p)[i];
            v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = x.z; v[4 * i + 3] = x.w;
        }
    }
}

// what a run of keys with maximum m and sum l counts for beside the largest maximum (a run that saw nothing: nothing; a sum of NaN stays one)
__device__ __forceinline__ float weight_of(float m, float l, float M) { return l == 0.f ? 0.f : exp2f(m - M); }

// four channels of a row, rounded once; a row that saw no key becomes zeros
template <typename T>
__device__ __forceinline__ void store_row(const Args& a, const Job& j, int row, int d, int ch, float4 v, float L) {
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    const int each = a.nh / a.nkv, rho = j.row0 + row, tok = a.tiles ? rho / each : 0;
    T* dst = (T*)a.out + ((size_t)(j.t0 + tok) * a.nh + j.kvh * each + rho - tok * each) * d + ch;
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(dst) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    } else {
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
    }
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_rank(uint32_t local, int rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(local), "r"(rank));
    return at;
}
__device__ __forceinline__ float load_cluster(uint32_t local, int rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at_rank(local, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float4 load_cluster4(uint32_t local, int rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at_rank(local, rank)) : "memory");
    return v;
}

template <typename T, int D, int G, int NT>
__global__ void __launch_bounds__(WARPS * 32, Pieces<T>::N * NT * D <= PAIR_UP_TO ? 2 : 1) int4_attention_kernel(Args a) {
    constexpr bool C8 = Pieces<T>::N == 2;            // codes less 8: see i4_pairs
    constexpr int NB = D / 64, NG = D / G, P = Pieces<T>::N, ROWS = 8 * NT, TILE = i4_cache_tile_bytes(D, G), CH = D / 32, STAGES = ring_tiles(TILE);
    // tiles a warp takes at a time: two chains of products and exponentials side by side (64 sequences of 8,192 keys 145 -> 140 us, 21 of 450 to
    // 9,000 58 -> 50), where the sums are few enough to leave two blocks of 8 warps their registers
    constexpr int PAIR = P * NT * D <= PAIR_UP_TO ? 2 : 1;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) uint64_t full[WARPS][STAGES];
    __shared__ float s_m[WARPS][ROWS], s_l[WARPS][ROWS], s_join[ROWS][2];
    if (a.overlap) ce_pdl_launch_dependents();
    ce_pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, l = lane & 3, warps = blockDim.x >> 5;
    const int split = blockIdx.x % a.splits, job_id = blockIdx.x / a.splits;
    const Job j = job_of(a, job_id, ROWS);
    const int each = a.nh / a.nkv, rows = min(ROWS, j.tokens * each - j.row0);
    if (rows <= 0) return;                            // a tile with fewer tokens than its row blocks take
    auto token_of = [&](int rho) { return a.tiles ? rho / each : 0; };        // (a single token's rows are its heads)
    const int first_pos = j.base + token_of(j.row0), last_pos = j.base + token_of(j.row0 + rows - 1);
    const int block_lo = a.window > 0 ? max(0, first_pos - a.window + 1) : 0;
    const int tile_lo = block_lo >> 4, tiles = last_pos < block_lo ? 0 : (last_pos >> 4) + 1 - tile_lo;
    // shares of the longest context's length (shorter sequences take fewer blocks), or as many keys as it takes
    const int share = max(a.share, (tiles + a.splits - 1) / a.splits), begin = min(split * share, tiles), end = min(begin + share, tiles);
    const int mine = end - begin > warp ? (end - begin - warp + warps - 1) / warps : 0;      // tiles begin + warp, + warps, ...
    const int* table = a.block_table + (size_t)j.slot * a.max_pages;
    unsigned char* ring = smem + warp * (STAGES * TILE);
    const int per_page = a.page_size >> 4;

    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < STAGES; ++s) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(i4_smem(&full[warp][s])));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    // where 32 of the warp's tiles lie, one a lane
    int looked = 0;
    const unsigned char* place = a.pages;
    auto look_up = [&](int from) {
        looked = from;
        const int i = from + lane, t = tile_lo + begin + warp + i * warps, pi = t / per_page;
        int page = i >= mine ? 0 : pi < a.max_pages ? table[pi] : -1;
        if (page < 0 || page >= a.num_pages) { atomicExch(a.status, 4); page = 0; }      // (the step's results are not used)
        place = a.pages + (((size_t)page * a.nkv + j.kvh) * per_page + (t - pi * per_page)) * TILE;
    };
    auto issue = [&](int i) {
        if (i >= looked + 32) look_up(i);
        const unsigned char* src = reinterpret_cast<const unsigned char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(place), i - looked));
        if (lane == 0) i4_copy(ring + (i % STAGES) * TILE, src, TILE, &full[warp][i % STAGES]);
    };
    Raw<T, CH> raw[NT];                               // asked for ahead of the pages: both take a trip
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = nt * 8 + r, rho = j.row0 + row, tok = token_of(rho);
        raw[nt].clear();
        if (row < rows) raw[nt].load((const T*)a.q + (size_t)(j.t0 + tok) * a.q_stride + (size_t)(j.kvh * each + rho - tok * each) * D + 8 * l, a.vec);
    }
    look_up(0);
    for (int i = 0; i < min(STAGES, mine); ++i) issue(i);

    // ---- queries: the second operand of K Q^T.  Lane (r, l) holds row 8 nt + r, channels 32 c + 8 l .. + 8; codes pair channels i and i + 4,
    // and odd codes come 16 times too large
    uint32_t qf[NT][P][CH][4];
    float qsum[NT][NG][2], row_scale[NT][2];          // of rows 8 nt + 2 l and + 1, as the scores lie
    int hi[NT][2], lo[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float largest = raw[nt].largest();
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        const float up = i4_row_scale(largest), up16 = up * 0.0625f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = raw[nt].at(c, i) * (i & 1 ? up16 : up), y = raw[nt].at(c, i + 4) * (i & 1 ? up16 : up);
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    qf[nt][p][c][i] = i4_pack(x, y);
                    if (p + 1 < P) {
                        const float2 got = i4_unpack(qf[nt][p][c][i]);
                        x -= got.x; y -= got.y;
                    }
                }
            }
        // the groups' sums, where the scores will lie: products with codes of 1, as ordinary numbers
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float acc[P][4];
#pragma unroll
            for (int c = g * G / 32; c < (g + 1) * G / 32; ++c)
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    if (c == g * G / 32) i4_mma_first(acc[p], 0x3c003c00u, 0x3c003c00u, 0x4c004c00u, 0x4c004c00u, qf[nt][p][c][0], qf[nt][p][c][1]);
                    else i4_mma(acc[p], 0x3c003c00u, 0x3c003c00u, 0x4c004c00u, 0x4c004c00u, qf[nt][p][c][0], qf[nt][p][c][1]);
                    i4_mma(acc[p], 0x3c003c00u, 0x3c003c00u, 0x4c004c00u, 0x4c004c00u, qf[nt][p][c][2], qf[nt][p][c][3]);
                }
#pragma unroll
            for (int e = 0; e < 2; ++e) qsum[nt][g][e] = (P == 2 ? acc[0][e] + acc[P - 1][e] : acc[0][e]) * (1.0f / i4_unit<C8>);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float u = __shfl_sync(0xffffffffu, up, 4 * (2 * l + e));
            row_scale[nt][e] = i4_normal(a.scale * LOG2E / u * i4_unit<C8>);        // (in this order nothing passes float32 on the way)
            const int rr = nt * 8 + 2 * l + e, pos = j.base + token_of(j.row0 + rr);
            hi[nt][e] = rr < rows ? pos : -1;
            lo[nt][e] = a.window > 0 ? pos - a.window + 1 : 0;
        }
    }

    float o[NT][NB * 4][4], oz[NT][NG][2], m[NT][2], sum[NT][2];
    // Weights are kept as 2^(S - m): m follows the scores (within HEADROOM) and, in the same number, the steps: a weight times a step is to lie
    // near 2^10, so m holds log2(top / 2^10) too, top a power of two that no step of V seen so far passes in magnitude.  Sums, parts of minima and products
    // all carry the factor, which falls out at the end.
    float top = 0x1p-24f, high[NT][2];                // high: what a score (before its row's scale) may reach before m is moved
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < NB * 4; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) oz[nt][g][0] = oz[nt][g][1] = 0.f;
        m[nt][0] = m[nt][1] = NOTHING;
        high[nt][0] = high[nt][1] = NOTHING;
        sum[nt][0] = sum[nt][1] = 0.f;
    }
    // tiles in [whole_lo, whole_hi] hold only keys that every row sees
    const int inner_lo = a.window > 0 ? max(0, last_pos - a.window + 1) : 0;

    bool ok = true;
    int gone = 0;                                     // tiles whose copies this warp has waited for, and whose place others may have taken
    for (int i = 0; i < mine; i += PAIR) {
        gone = i;
        const unsigned char* tile[PAIR];
        int key0[PAIR];
        bool cut = false;
#pragma unroll
        for (int p = 0; p < PAIR; ++p) {
            const bool here = p == 0 || i + p < mine;
            if (here) ok = ok && i4_warp_wait(&full[warp][(i + p) % STAGES], ((i + p) / STAGES) & 1);
            tile[p] = ring + ((i + p) % STAGES) * TILE;
            // (a last tile alone: the other's keys are ones that nobody sees)
            key0[p] = here ? (tile_lo + begin + warp + (i + p) * warps) * 16 : last_pos + 1;
            cut = cut || key0[p] < inner_lo || key0[p] + 15 > first_pos;
        }
        if (!ok) { if (lane == 0) atomicExch(a.status, 7); break; }
        // ---- scores of keys r and r + 8 (rows of the tile) for query rows 2 l and 2 l + 1
        float s[PAIR][NT][4];
#pragma unroll
        for (int p = 0; p < PAIR; ++p) {
            uint32_t ka[NG], kb[NG];
            load_steps<NG>(tile[p] + 16 * D + r * NG * 4, ka);
            load_steps<NG>(tile[p] + 16 * D + (r + 8) * NG * 4, kb);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[p][nt][0] = s[p][nt][1] = s[p][nt][2] = s[p][nt][3] = 0.f;
            float acc[NT][P][4];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const uint4 w = *reinterpret_cast<const uint4*>(tile[p] + b * 512 + lane * 16);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int c = 2 * b + half;
                    const uint32_t wa = half ? w.z : w.x, wb = half ? w.w : w.y;
#pragma unroll
                    for (int st = 0; st < 2; ++st) {
                        uint32_t a0, a1, a2, a3;
                        if (st) { i4_pairs<C8, 8>(wa, a0, a2); i4_pairs<C8, 8>(wb, a1, a3); }
                        else { i4_pairs<C8, 0>(wa, a0, a2); i4_pairs<C8, 0>(wb, a1, a3); }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int q = 0; q < P; ++q) {
                                if (st == 0 && (c * 32) % G == 0) i4_mma_first(acc[nt][q], a0, a1, a2, a3, qf[nt][q][c][0], qf[nt][q][c][1]);
                                else i4_mma(acc[nt][q], a0, a1, a2, a3, qf[nt][q][c][2 * st], qf[nt][q][c][2 * st + 1]);
                            }
                    }
                    if ((c * 32 + 32) % G == 0) {
                        const int g = c * 32 / G;
                        const float2 fa = i4_step_of<C8>(ka[g]), fb = i4_step_of<C8>(kb[g]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float sa = acc[nt][0][e], sb = acc[nt][0][2 + e];
                                if constexpr (P == 2) { sa += acc[nt][1][e]; sb += acc[nt][1][2 + e]; }
                                s[p][nt][e] = fmaf(fa.x, sa, fmaf(fa.y, qsum[nt][g][e], s[p][nt][e]));
                                s[p][nt][2 + e] = fmaf(fb.x, sb, fmaf(fb.y, qsum[nt][g][e], s[p][nt][2 + e]));
                            }
                    }
                }
            }
        }
        // steps and minima of V; keys outside the block's reach may hold anything
        uint32_t va[PAIR][NG], vb[PAIR][NG];
#pragma unroll
        for (int p = 0; p < PAIR; ++p) {
            load_steps<NG>(tile[p] + 16 * D + 64 * NG + r * NG * 4, va[p]);
            load_steps<NG>(tile[p] + 16 * D + 64 * NG + (r + 8) * NG * 4, vb[p]);
        }
        if (cut) {
#pragma unroll
            for (int p = 0; p < PAIR; ++p) {
                const int key_a = key0[p] + r, key_b = key_a + 8;
                const bool in_a = key_a >= block_lo && key_a <= last_pos, in_b = key_b >= block_lo && key_b <= last_pos;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    // a group that is not a number reaches the rows that see its key, and no others (0 times NaN would)
                    const bool nan_a = isnan(i4_unpack(va[p][g]).x), nan_b = isnan(i4_unpack(vb[p][g]).x);
                    if (__any_sync(0xffffffffu, nan_a || nan_b)) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                if (nan_a && in_a && key_a <= hi[nt][e] && key_a >= lo[nt][e]) oz[nt][g][e] = __int_as_float(0x7fc00000);
                                if (nan_b && in_b && key_b <= hi[nt][e] && key_b >= lo[nt][e]) oz[nt][g][e] = __int_as_float(0x7fc00000);
                            }
                    }
                    if (!in_a || nan_a) va[p][g] = 0;
                    if (!in_b || nan_b) vb[p][g] = 0;
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if (key_a > hi[nt][e] || key_a < lo[nt][e]) s[p][nt][e] = -INFINITY;
                        if (key_b > hi[nt][e] || key_b < lo[nt][e]) s[p][nt][2 + e] = -INFINITY;
                    }
            }
        }
        bool move = false, coarse = false;            // coarse: a row's m lies beyond COARSE (every turn of such a row moves it)
        float mx[NT][2], step_max = 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                mx[nt][e] = fmaxf(s[0][nt][e], s[0][nt][2 + e]);
#pragma unroll
                for (int p = 1; p < PAIR; ++p) mx[nt][e] = fmaxf(mx[nt][e], fmaxf(s[p][nt][e], s[p][nt][2 + e]));
                move = move || mx[nt][e] > high[nt][e];
            }
        float fa[PAIR][NG], fb[PAIR][NG];
#pragma unroll
        for (int p = 0; p < PAIR; ++p)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                fa[p][g] = i4_unpack(va[p][g]).x; fb[p][g] = i4_unpack(vb[p][g]).x;
                step_max = fmaxf(step_max, fmaxf(fabsf(fa[p][g]), fabsf(fb[p][g])));
            }
        move = move || step_max > top;
        if (__any_sync(0xffffffffu, move)) {
            // maxima over the 8 lanes that share l, the largest step over all
#pragma unroll
            for (int w = 16; w > 0; w >>= 1) step_max = fmaxf(step_max, __shfl_xor_sync(0xffffffffu, step_max, w));
            const float before = top;
            // the next power of two: a number's exponent, one up where it has bits below
            if (step_max > top) top = __uint_as_float((__float_as_uint(step_max) + 0x007fffffu) & 0x7f800000u);
            const float offset = log2f(top) - 10.0f, grown = log2f(before) - log2f(top);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = mx[nt][e];
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    const float there = __fmaf_rd(x, row_scale[nt][e], offset);
                    const float now = m[nt][e] == NOTHING ? there : fmaxf(__fsub_rd(m[nt][e], grown), there);
                    const float alpha = m[nt][e] == NOTHING ? 0.0f : exp2f(m[nt][e] - now);
                    m[nt][e] = x == -INFINITY && m[nt][e] == NOTHING ? NOTHING : now;
                    const bool far = fabsf(m[nt][e]) >= COARSE;
                    coarse = coarse || (far && m[nt][e] != NOTHING);
                    high[nt][e] = far ? NOTHING : (now - offset + HEADROOM) / row_scale[nt][e];
                    sum[nt][e] *= alpha;
#pragma unroll
                    for (int g = 0; g < NG; ++g) oz[nt][g][e] *= alpha;
#pragma unroll
                    for (int i2 = 0; i2 < NB * 4; ++i2) { o[nt][i2][e] *= alpha; o[nt][i2][2 + e] *= alpha; }
                }
            coarse = __any_sync(0xffffffffu, coarse);
        }
        float pr[PAIR][NT][4];
#pragma unroll
        for (int p = 0; p < PAIR; ++p)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    pr[p][nt][e] = fmaf(s[p][nt][e], row_scale[nt][e], -m[nt][e]);
                    pr[p][nt][2 + e] = fmaf(s[p][nt][2 + e], row_scale[nt][e], -m[nt][e]);
                }
        if (coarse) {
            const float most = 10.0f - log2f(top) + HEADROOM;
#pragma unroll
            for (int p = 0; p < PAIR; ++p)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) pr[p][nt][e] = i4_min(pr[p][nt][e], most);
        }
#pragma unroll
        for (int p = 0; p < PAIR; ++p)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    pr[p][nt][e] = ce_exp2_fast(pr[p][nt][e]);
                    pr[p][nt][2 + e] = ce_exp2_fast(pr[p][nt][2 + e]);
                    sum[nt][e] += pr[p][nt][e] + pr[p][nt][2 + e];
                }
        // ---- V^T P^T, group by group: the probability carries the step
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int p = 0; p < PAIR; ++p) {
                const uint4 w = *reinterpret_cast<const uint4*>(tile[p] + 8 * D + b * 512 + lane * 16);
                uint32_t bf[NT][P][2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int g = (64 * b + 32 * half) / G;
                    if ((32 * half) % G == 0) {
                        const float za = i4_step_of<C8>(va[p][g]).y, zb = i4_step_of<C8>(vb[p][g]).y;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const float* w4 = pr[p][nt];
                            oz[nt][g][0] = fmaf(w4[0], za, fmaf(w4[2], zb, oz[nt][g][0]));
                            oz[nt][g][1] = fmaf(w4[1], za, fmaf(w4[3], zb, oz[nt][g][1]));
                            float x0 = w4[0] * fa[p][g], x1 = w4[1] * fa[p][g], x2 = w4[2] * fb[p][g], x3 = w4[3] * fb[p][g];
#pragma unroll
                            for (int q = 0; q < P; ++q) {
                                const uint32_t ab = i4_pack(x0, x1), cd = i4_pack(x2, x3);
                                bf[nt][q][0] = transpose8(ab);
                                bf[nt][q][1] = transpose8(cd);
                                if (q + 1 < P) {
                                    const float2 g0 = i4_unpack(ab), g1 = i4_unpack(cd);
                                    x0 -= g0.x; x1 -= g0.y; x2 -= g1.x; x3 -= g1.y;
                                }
                            }
                        }
                    }
                    // the halves of a word are the two halves of the block's channels; two tokens' words side by side
                    const uint32_t pick = half ? 0x7632u : 0x5410u;
                    const uint32_t u = __byte_perm(w.x, w.y, pick), v = __byte_perm(w.z, w.w, pick);
#pragma unroll
                    for (int st = 0; st < 2; ++st) {
                        uint32_t a0, a1, a2, a3;
                        if (st) { i4_pairs<C8, 8>(u, a0, a1); i4_pairs<C8, 8>(v, a2, a3); }
                        else { i4_pairs<C8, 0>(u, a0, a1); i4_pairs<C8, 0>(v, a2, a3); }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int q = 0; q < P; ++q) i4_mma(o[nt][b * 4 + half * 2 + st], a0, a1, a2, a3, bf[nt][q][0], bf[nt][q][1]);
                    }
                }
            }
        __syncwarp();
#pragma unroll
        for (int p = 0; p < PAIR; ++p)
            if (i + p + STAGES < mine) issue(i + p + STAGES);
    }
    if (!ok) {
        // the copies still in flight land in this block's memory: wait for them, with a limit, before it is used for anything else
        for (int i = gone; i < min(gone + STAGES, mine); ++i) i4_wait(&full[warp][i % STAGES], (i / STAGES) & 1);
    }
    __syncthreads();                                  // the rings are free: the warps' outputs take their place

    float* so = reinterpret_cast<float*>(smem);       // [warps][ROWS][D + 4]
    constexpr int LD = D + 4;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = nt * 8 + 2 * l + e;
            float t = sum[nt][e];
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) t += __shfl_xor_sync(0xffffffffu, t, w);
            if (r == 0) { s_m[warp][row] = m[nt][e]; s_l[warp][row] = t; }
            constexpr float even = i4_unit<C8>, odd = even * 0.0625f;
            float zs[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                zs[g] = oz[nt][g][e];
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) zs[g] += __shfl_xor_sync(0xffffffffu, zs[g], w);
            }
#pragma unroll
            for (int i = 0; i < NB * 4; ++i) {
                const int ch = 64 * (i >> 2) + 32 * ((i >> 1) & 1) + 4 * r + 2 * (i & 1), g = (64 * (i >> 2) + 32 * ((i >> 1) & 1)) / G;
                float2 v = make_float2(fmaf(o[nt][i][e], even, zs[g]), fmaf(o[nt][i][2 + e], odd, zs[g]));
                *reinterpret_cast<float2*>(so + (warp * ROWS + row) * LD + ch) = v;
            }
        }
    }
    __syncthreads();
    const bool cluster = a.clustered;
    for (int x = threadIdx.x; x < rows * (D / 4); x += blockDim.x) {
        const int row = x / (D / 4), ch = (x - row * (D / 4)) * 4;
        float M = NOTHING, L = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        auto join = [&](auto all) {                   // (8 or 4 known to the compiler: the loads go out together)
#pragma unroll
            for (int w = 0; w < all(); ++w) M = fmaxf(M, s_m[w][row]);
#pragma unroll
            for (int w = 0; w < all(); ++w) {
                const float f = weight_of(s_m[w][row], s_l[w][row], M);
                const float4 u = *reinterpret_cast<const float4*>(so + (w * ROWS + row) * LD + ch);
                L += s_l[w][row] * f;
                v.x = fmaf(u.x, f, v.x); v.y = fmaf(u.y, f, v.y); v.z = fmaf(u.z, f, v.z); v.w = fmaf(u.w, f, v.w);
            }
        };
        if (warps == WARPS) join(std::integral_constant<int, WARPS>());
        else join(std::integral_constant<int, WARPS / 2>());
        if (cluster) {
            // (warp 0's rows: every number of theirs is read by the thread that replaces it)
            *reinterpret_cast<float4*>(so + row * LD + ch) = v;
            if (ch == 0) { s_join[row][0] = M; s_join[row][1] = L; }
        } else if (a.splits > 1) {
            const size_t at = ((size_t)job_id * a.splits + split) * ROWS + row;
            *reinterpret_cast<float4*>(a.part_o + at * D + ch) = v;
            if (ch == 0) { a.part_ml[2 * at] = M; a.part_ml[2 * at + 1] = L; }
        } else {
            store_row<T>(a, j, row, D, ch, v, L);
        }
    }
    if (!cluster) return;
    // the blocks' runs of keys, in their order: each takes a share of the rows' channels
    cluster_sync();
    const int all = rows * (D / 4);
    for (int x = threadIdx.x * a.splits + split; x < all; x += a.splits * blockDim.x) {
        const int row = x / (D / 4), ch = (x - row * (D / 4)) * 4;
        float M = NOTHING, L = 0.f, ms[8], ls[8];
        float4 us[8], v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 8; ++k) {                 // (one trip to all of them)
            ms[k] = NOTHING; ls[k] = 0.f; us[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k < a.splits) {
                ms[k] = load_cluster(i4_smem(&s_join[row][0]), k);
                ls[k] = load_cluster(i4_smem(&s_join[row][1]), k);
                us[k] = load_cluster4(i4_smem(so + row * LD + ch), k);
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) M = fmaxf(M, ms[k]);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float f = weight_of(ms[k], ls[k], M);
            L += ls[k] * f;
            v.x = fmaf(us[k].x, f, v.x); v.y = fmaf(us[k].y, f, v.y); v.z = fmaf(us[k].z, f, v.z); v.w = fmaf(us[k].w, f, v.w);
        }
        store_row<T>(a, j, row, D, ch, v, L);
    }
    cluster_sync();                                   // nobody leaves while its rows are read
}

// Joins the runs of keys of a row block: a block a row, its warps - up to 8 - a run in turn (a lane four channels), then the warps' sums, all in a fixed order.
// (One warp that reads run after run takes 0.5 us for each.)
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(256) int4_attention_merge_kernel(Args a) {
    ce_pdl_begin();
    constexpr int CH = (D + 127) / 128;
    __shared__ float4 part[8][D / 4];
    __shared__ float part_l[8];
    const int job_id = blockIdx.x / ROWS, row = blockIdx.x - job_id * ROWS, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const Job j = job_of(a, job_id, ROWS);
    const int each = a.nh / a.nkv;
    if (row >= j.tokens * each - j.row0) return;
    const size_t at = (size_t)job_id * a.splits * ROWS + row;
    float M = NOTHING, L = 0.f;
    for (int s = lane; s < a.splits; s += 32) M = fmaxf(M, a.part_ml[2 * (at + (size_t)s * ROWS)]);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, w));
    float4 v[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = warp; s < a.splits; s += warps) {
        const size_t p = at + (size_t)s * ROWS;
        const float ls = a.part_ml[2 * p + 1], f = weight_of(a.part_ml[2 * p], ls, M);
        L += ls * f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int ch = (c * 32 + lane) * 4;
            if (ch >= D || ls == 0.f) continue;       // (a run without a key that the row sees wrote nothing else)
            const float4 u = *reinterpret_cast<const float4*>(a.part_o + p * D + ch);
            v[c].x = fmaf(u.x, f, v[c].x); v[c].y = fmaf(u.y, f, v[c].y); v[c].z = fmaf(u.z, f, v[c].z); v[c].w = fmaf(u.w, f, v[c].w);
        }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
        if ((c * 32 + lane) * 4 < D) part[warp][c * 32 + lane] = v[c];
    if (lane == 0) part_l[warp] = L;
    __syncthreads();
    for (int x = threadIdx.x; x < D / 4; x += blockDim.x) {
        float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
        L = 0.f;
        for (int w = 0; w < warps; ++w) {
            const float4 u = part[w][x];
            L += part_l[w];
            t.x += u.x; t.y += u.y; t.z += u.z; t.w += u.w;
        }
        store_row<T>(a, j, row, D, 4 * x, t, L);
    }
}

template <typename T, int D, int G, int NT>
int run(Args a, int jobs, cudaStream_t stream) {
    constexpr int TILE = i4_cache_tile_bytes(D, G), RING = ring_tiles(TILE) * TILE, OUT = 8 * NT * (D + 4) * 4;
    constexpr int SMEM = WARPS * (RING > OUT ? RING : OUT);
    // 8 warps a block as long as the chip takes all blocks at once, two an SM; then 4, four an SM, whose beginnings and ends (some 4.5 us) hide
    // behind more others: 64 sequences of 8,192 keys in quarters (ops_int4._splits takes thirds there) 134 us for 151, 128 of 30 to 600 22 us for 30 (19 since);
    // one of 2,048 in eighths 8.3 us for 7.5
    const int warps = (long long)jobs * a.splits <= 2 * ce_sm_count() ? WARPS : WARPS / 2;
    static_assert(SMEM <= 220 * 1024, "a block's shared memory");
    static std::atomic<unsigned long long> done{0};
    auto kernel = int4_attention_kernel<T, D, G, NT>;
    cudaError_t e = ce_allow_smem(done, kernel, SMEM);
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[2];
        cfg.gridDim = dim3((unsigned)(jobs * a.splits));
        cfg.blockDim = dim3(warps * 32);
        cfg.dynamicSmemBytes = SMEM / WARPS * warps;
        cfg.stream = stream;
        cfg.attrs = attr;
        a.clustered = a.splits > 1 && !a.part_o;
        a.overlap = ce_pdl_enabled();
        if (a.clustered) {
            attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
            attr[cfg.numAttrs++].val.clusterDim = {(unsigned)a.splits, 1, 1};
            // a grid of more clusters than the chip holds stands alone (ce_clusters_at_once)
            static CeRoom room[2][9];
            a.overlap = a.overlap && jobs <= ce_clusters_at_once(room[warps == WARPS][a.splits], kernel, cfg);
        }
        if (a.overlap) {
            attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
        }
        ce_note("int4_attention_kernel");
        e = cudaLaunchKernelEx(&cfg, kernel, a);
    }
    if (e == cudaSuccess && a.splits > 1 && !a.clustered) {
        ce_note("int4_attention_merge_kernel");
        e = ce_launch(int4_attention_merge_kernel<T, D, 8 * NT>, dim3((unsigned)(jobs * 8 * NT)), dim3(32 * (a.splits < 8 ? a.splits : 8)), 0, stream, a);
    }
    if (e != cudaSuccess) { (void)cudaGetLastError(); return ce_fail(CE_ERR_CUDA, "int4_attention: %s", cudaGetErrorString(e)); }
    return ce_check_launch("int4_attention");
}

template <typename T, int D, int G>
int run_rows(const Args& a, int jobs, int rows, cudaStream_t stream) {
    if constexpr (D <= 128) {
        if (rows == 16) return run<T, D, G, 2>(a, jobs, stream);
    }
    return run<T, D, G, 1>(a, jobs, stream);
}
template <typename T, int D>
int run_group(const Args& a, int group, int jobs, int rows, cudaStream_t stream) {
    return group == 32 ? run_rows<T, D, 32>(a, jobs, rows, stream) : run_rows<T, D, 64>(a, jobs, rows, stream);
}
template <typename T>
int run_type(const Args& a, int d, int group, int jobs, int rows, cudaStream_t stream) {
    switch (d) {
        case 64: return run_group<T, 64>(a, group, jobs, rows, stream);
        case 128: return run_group<T, 128>(a, group, jobs, rows, stream);
        case 192: return run_group<T, 192>(a, group, jobs, rows, stream);
        default: return run_group<T, 256>(a, group, jobs, rows, stream);
    }
}

// rows of a block: 8, or 16 where a KV head has more than 8 query rows to serve and the registers hold them (heads of at most 128)
int block_rows(int each, int d, int tokens) { return d <= 128 && each * tokens > 8 ? 16 : 8; }

}  // namespace

int ce_int4_attention_tc(const void* q, long long q_stride, const void* pages, void* out, const int* seq_slot, const int* q_start, const int* ctx_len,
                         const int* block_table, int* status, const int* tiles, int n_tiles, int nh, int nkv, int d, int group, int page_size,
                         int max_pages, int num_pages, int window, float scale, cudaStream_t stream);

// Rows a block takes, and the row blocks of a one-token sequence (tile 0) or of a tile of 64 tokens (tile 1)
extern "C" int ce_int4_attention_rows(int each, int d, int tile) { return block_rows(each, d, tile ? 64 : 1); }
extern "C" int ce_int4_attention_blocks(int each, int d, int tile) {
    const int rows = block_rows(each, d, tile ? 64 : 1);
    return ((tile ? 64 : 1) * each + rows - 1) / rows;
}

// A call's arguments, 8 bytes each in this order
struct Int4AttentionCall {
    long long dtype;
    const void* q;
    long long q_stride;
    const void* pages;
    void* out;
    const int *seq_slot, *q_start, *ctx_len, *block_table;
    int* status;
    const int* tiles;              // null: ``n`` one-token sequences
    long long n, nh, nkv, d, group, page_size, max_pages, num_pages, window, splits, share;     // without part_o the splits (8 at most) are a cluster; 0: the kernel on tcgen05
    float *part_o, *part_ml;
    double scale;
    void* stream;
};

extern "C" int ce_int4_attention(const Int4AttentionCall* c) {
    const void *q = c->q, *pages = c->pages;
    void* out = c->out;
    const int *seq_slot = c->seq_slot, *q_start = c->q_start, *ctx_len = c->ctx_len, *block_table = c->block_table, *tiles = c->tiles;
    int* status = c->status;
    float *part_o = c->part_o, *part_ml = c->part_ml;
    const long long q_stride = c->q_stride, count = c->n;
    const int dtype = (int)c->dtype, nh = (int)c->nh, nkv = (int)c->nkv, d = (int)c->d, group = (int)c->group, page_size = (int)c->page_size,
              max_pages = (int)c->max_pages, num_pages = (int)c->num_pages, window = (int)c->window, splits = (int)c->splits;
    const float scale = (float)c->scale;
    void* stream = c->stream;
    if (!q || !pages || !out || !seq_slot || !q_start || !ctx_len || !block_table || !status) return ce_fail(CE_ERR_ARG, "int4_attention: null pointer");
    if (dtype != CE_F32 && dtype != CE_BF16) return ce_fail(CE_ERR_ARG, "int4_attention: unknown dtype %d", dtype);
    if (nkv < 1 || nh < 1 || nh % nkv) return ce_fail(CE_ERR_SIZE, "int4_attention: %d heads over %d kv heads", nh, nkv);
    if (d < 64 || d > 256 || d % 64) return ce_fail(CE_ERR_SIZE, "int4_attention: head size %d (64, 128, 192 or 256)", d);
    if (group != 32 && group != 64) return ce_fail(CE_ERR_SIZE, "int4_attention: group %d (32 or 64)", group);
    if (page_size < 16 || page_size % 16) return ce_fail(CE_ERR_SIZE, "int4_attention: page size %d is not a multiple of 16", page_size);
    if (((uintptr_t)pages & 15) != 0) return ce_fail(CE_ERR_ARG, "int4_attention: the pages do not start on a 16-byte boundary");
    const long long sizes[] = {c->nh, c->nkv, c->d, c->group, c->page_size, c->max_pages, c->num_pages, c->window, c->splits};
    for (long long size : sizes)
        if (size < 0 || size > 0x7fffffffll) return ce_fail(CE_ERR_SIZE, "int4_attention: a size of %lld", size);
    if (max_pages < 1 || num_pages < 1) return ce_fail(CE_ERR_SIZE, "int4_attention: bad sizes");
    if (((uintptr_t)out % (dtype == CE_F32 ? 16 : 8)) != 0) return ce_fail(CE_ERR_ARG, "int4_attention: out does not start on a boundary of four elements");
    // (a block's first tile of keys is its number times the share)
    if (c->splits > 1024 || c->share < 0 || c->share > (1ll << 30) / (splits < 1 ? 1 : splits))
        return ce_fail(CE_ERR_SIZE, "int4_attention: %lld shares of %lld tiles of keys", c->splits, c->share);
    if (splits > 8 && (!part_o || !part_ml)) return ce_fail(CE_ERR_ARG, "int4_attention: more than 8 shares of the keys need scratch memory");
    if (!(scale > 0.0f && scale < 0x1p127f)) return ce_fail(CE_ERR_ARG, "int4_attention: a scale that is not a positive number of float32 below 2^127");
    if (count == 0) return CE_OK;
    if (splits == 0) {
        if (dtype != CE_BF16 || !tiles || count < 0 || count > 65535) return ce_fail(CE_ERR_SIZE, "int4_attention: splits of 0 are for tiles of bfloat16");
        return ce_int4_attention_tc(q, q_stride, pages, out, seq_slot, q_start, ctx_len, block_table, status, tiles, (int)count, nh, nkv, d, group, page_size,
                                    max_pages, num_pages, window, scale, (cudaStream_t)stream);
    }
    const int each = nh / nkv, rows = block_rows(each, d, tiles ? 64 : 1), subs = ((tiles ? 64 : 1) * each + rows - 1) / rows;
    const long long jobs = count * nkv * subs;
    if (count < 0 || jobs * splits * 16 > 0x7fffffffll) return ce_fail(CE_ERR_SIZE, "int4_attention: too many rows");
    const int el = dtype == CE_F32 ? 4 : 2;
    Args a{q, out, (const unsigned char*)pages, seq_slot, q_start, ctx_len, block_table, tiles, status, part_o, part_ml, q_stride,
           nh, nkv, page_size, max_pages, num_pages, window, splits, (int)c->share, subs, ((uintptr_t)q % (4 * el)) == 0 && q_stride % 4 == 0, 0, 0, scale};
    return dtype == CE_F32 ? run_type<float>(a, d, group, (int)jobs, rows, (cudaStream_t)stream)
                           : run_type<__nv_bfloat16>(a, d, group, (int)jobs, rows, (cudaStream_t)stream);
}
