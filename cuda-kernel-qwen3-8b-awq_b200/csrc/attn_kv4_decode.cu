// Attention of single tokens over the paged 4-bit cache (attentionKernel, Inference.cu:182-266, intended math; heads grouped over KV heads).
//
//   score_j = c (sk_j sum_d code_jd q_d + mk_j sum_d q_d),  out = sum_j p_j (sv_j code_j + mv_j) / sum_j p_j,  c = scale * log2(e)
//
// The codes go into the tensor cores as they are: a nibble in the low bits of a half is the subnormal code * 2^-24 (or * 2^-20 four bits
// further up), so a mask is all the unpacking there is, products are exact, and scales are applied to fp32 sums.  V's scale is folded into the
// exponent: u_j = score_j + log2(sv_j), P_j = 2^(u_j - max u + 8) enters the second product as fp16 (the largest is between 2^8 and 2^15, so
// the 11 bits reach 22 powers of two below it, whatever the scales are), and the sums of p and p (mv + 8 sv) take P_j / sv_j in fp32.
// The tensor cores cut sums off 2^-23 below their largest term as it is encoded, which for a code in the low bits is 2^-14 times P, and the sum
// of P code is far larger than that of P (code - 8), so that it comes out short: one more product sums P * 8 the same way, and the
// difference goes to fp32 sums in shared memory after sixteen chunks at most (lists of 20 to 41 K tokens: error 3.4e-4 of the outputs' size, after one chunk the same; without the flush 9e-4, without
// either 2e-3; 2.6e-4 with the low terms of P that fp16 rows and groups of four heads at most have, 2.1e-4 being that of the output's own rounding).
//
// A warp works on 32 tokens at a time, two tiles of 16 that bulk copies bring into its own ring of two: S^T = K Q^T (16 tokens x 8 heads
// of the group), then O^T += V^T P^T, with mma.sync m16n8k16: one product a token and KV head is a third of what the warp-level path can
// issue while HBM brings the 136 bytes, and its operands need no pass through tensor memory.
// A group of more than eight heads takes a pass over the cache for every eight.
// 48 requests of 20 to 41 K tokens, 32 heads over 8 KV heads, fp16, 1.66 GB: 312 us, 5.3 TB/s, 0.82 of the measured copy rate (349 in
// sustained use).  16 requests of 16384 tokens: ALU pipe 51 % of active cycles, warp-level tensor pipe 28 %, issue slots 49 %: no unit is saturated.  When the kernel took
// 332 us, copies without products took 272 and products without copies 276: neither alone explains the time.
// The 32-token chunks of all (KV head, request) pairs form one list that is cut into equal parts, one a CTA, whatever the lengths are; the four
// warps of a CTA take its chunks in turn and join their states in shared memory, and pairs that are cut by the border of a CTA are joined
// from the workspace by the last CTA to arrive, in order of the parts: results do not depend on timing.
#include <atomic>

#include "kv4.cuh"
#include "tc05.cuh"

namespace qw3 {

constexpr int KD_WARPS = 4, KD_THREADS = 32 * KD_WARPS, KD_STAGES = 2, KD_CTAS = 3;   // CTAs an SM
constexpr int KD_CHUNK = 32, KD_STAGE_BYTES = 2 * KV4_TILE_BYTES;
constexpr int KD_FLUSH = 16;           // chunks whose products are summed in an accumulator
constexpr int KD_MIN_CHUNKS = 8;       // chunks a CTA takes at least
constexpr int KD_WHOLE = 32;           // pairs of so many chunks are not cut (all cut: one request of 517 tokens 16.4 instead of 12.4 us,
                                       // 128 requests of 100 to 600 32.8 instead of 28.7; requests of 9000 tokens and more the same)
constexpr int KD_PAIR = 6;             // what a pair costs a CTA beside its chunks (q, joining the warps' states), in chunks (1: 48 long ones 309 instead of 303 us)
constexpr int KD_PART = 1024 + 32;     // floats of a partial state: outputs, then (maximum, sum of p, sum of p mv) of eight heads
constexpr int KD_MAX_GRID = 1024;
static_assert(2 * (size_t)KD_MAX_GRID * KD_PART <= WS_PARTIALS && KD_MAX_GRID <= WS_MAX_TILES, "workspace");

struct KdSmem {
    uint8_t ring[KD_WARPS][KD_STAGES][KD_STAGE_BYTES];
    float4 o[KD_WARPS][8][32];        // sums of a warp, in the order of its fragments
    struct { const uint8_t* at[2]; } src[KD_WARPS][32];   // of the chunks that are looked up: the tiles (the second null where it follows the
    int2 tokens[KD_WARPS][32];                            // first), the tokens in them, 16 bits a tile, and the bytes of the first copy
    float4 token[KD_WARPS][KD_CHUNK];  // of the chunk's tokens: scale of K * 2^24, minimum of K, log2 of V's scale, 1 / V's scale
    float mid[KD_WARPS][KD_CHUNK];     // and V's minimum + 8 * scale
    float stat[KD_WARPS][8][3];
    uint64_t bar[KD_WARPS][KD_STAGES];
    int valid[KD_WARPS][KD_STAGES];    // tokens of the two tiles, 16 bits each
    int last;
};

__device__ __forceinline__ float kd_ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float kd_lg2(float x) {
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float kd_rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// V's scale as the logarithm and the reciprocal can take it.  A row of zero bytes, which append never wrote, has 0: it becomes a scale so small that
// the row's codes add nothing.  fp16: one addition, lost in the rounding of every scale from 2^-24 on; the three instructions of bf16, whose floor is
// too small for that, take 357 instead of 355 us for 48 long requests.
template <class T>
__device__ __forceinline__ float kd_scale(float s) {
    using R = RowType<T>;
    return R::FLOOR > 1e-9f ? s + 1.7763568394002505e-15f : s >= 0.0f ? fmaxf(s, R::FLOOR) : NAN;   // 2^-49
}
__device__ __forceinline__ uint32_t kd_transpose(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
// D = A * B
__device__ __forceinline__ void kd_mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

struct KdParams {
    Qw3Kv4Pool pool;
    Qw3AttnKv4Args a;
    int group, q_tiles, heads_t;   // heads a KV head, tiles of eight of them, (KV head, tile) pairs
    long long most_tokens;         // that a row of the table can hold
    float c;
    float* part;
    int* count;
    int* err;
};

// A place in the list of chunks: pair `ht`, request `b`, chunk `c` of the request's `n`.
struct KdPlace {
    int ht, b, c, n;
};

// NARROW: groups of four heads at most, which leave half of a fragment's columns empty.  The lanes of the empty columns take the scores of the
// second tile, so that each has half as many exponentials; fp16 rows use the products' empty columns for
// what the rounding of P to fp16 took off (bf16 rows round the result so much more that it does not show: 1.67e-3 with and without): 48 requests of
// 20 to 41 K tokens 312 us and an error of 2.6e-4, without the low terms 303 and 3.4e-4, without NARROW 315; short requests the same.
template <class T, bool NARROW>
__global__ void __launch_bounds__(KD_THREADS, KD_CTAS) attn_kv4_decode_kernel(KdParams p) {
    extern __shared__ __align__(128) uint8_t kd_smem[];
    KdSmem& sm = *reinterpret_cast<KdSmem*>(kd_smem);
    using R = RowType<T>;
    constexpr bool LOW = NARROW && R::FLOOR > 1e-9f;   // fp16 rows
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int B = p.a.n_req, tiles_page = p.pool.page_size / 16;
    pdl_launch_dependents();
    if (lane == 0) {
        for (int s = 0; s < KD_STAGES; ++s) mbar_init(smem_u32(&sm.bar[warp][s]), 1);
        mbar_fence_init();
    }
    __syncthreads();
    pdl_wait();

    const auto length = [&](int b) {
        const int n = p.a.d_kv_len[b];
        return n < 0 ? 0 : (long long)n > p.most_tokens ? (int)p.most_tokens : n;
    };
    // this CTA's part of the list.  Places are counted twice: in chunks, and, to give all CTAs the same work, with KD_PAIR more for each pair
    long long per_head = 0;
    int busy = 0;   // requests that have tokens
    for (int b = lane; b < B; b += 32) {
        const int n = (length(b) + KD_CHUNK - 1) / KD_CHUNK;
        per_head += n;
        busy += n > 0;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) per_head += __shfl_xor_sync(0xffffffffu, per_head, d);
    busy = __reduce_add_sync(0xffffffffu, busy);
    const long long chunks = per_head * p.heads_t, per_head_w = per_head + (long long)KD_PAIR * busy, total = per_head_w * p.heads_t;
    // so many CTAs that a part is worth starting one, and that joining the parts of a pair does not take longer than they do
    const float balanced = sqrtf(2.0f * (float)chunks * (float)((long long)busy * p.heads_t));
    const long long wanted = min((long long)balanced, chunks / KD_MIN_CHUNKS);
    const int grid = (int)max(1ll, min(wanted, (long long)gridDim.x));
    long long x[2] = {0, 0};        // first chunk and the one behind the last
    KdPlace place = {0, 0, 0, 0};   // of the first
    if (chunks > 0 && (int)blockIdx.x < grid) {
        long long y[2];
        int ht[2];
        bool found[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const long long w = total * (blockIdx.x + e) / grid;
            ht[e] = (int)(w / per_head_w);
            y[e] = w - ht[e] * per_head_w;
            found[e] = w == total;
            x[e] = found[e] ? chunks : ht[e] * per_head;
        }
        long long before = 0;       // chunks of the requests before the thirty-two
        for (int b0 = 0; b0 < B && !(found[0] && found[1]); b0 += 32) {
            const int n = b0 + lane < B ? (length(b0 + lane) + KD_CHUNK - 1) / KD_CHUNK : 0;
            int s = n;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int a = __shfl_up_sync(0xffffffffu, s, d);
                if (lane >= d) s += a;
            }
            const uint32_t any = __ballot_sync(0xffffffffu, n > 0);
            const int ws = s + KD_PAIR * __popc(any & (0xffffffffu >> (31 - lane))), all = __shfl_sync(0xffffffffu, ws, 31);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (!found[e] && y[e] < all) {
                    found[e] = true;
                    const int l = __ffs(__ballot_sync(0xffffffffu, y[e] < ws)) - 1;
                    const int nl = __shfl_sync(0xffffffffu, n, l), sl = __shfl_sync(0xffffffffu, s, l), wl = __shfl_sync(0xffffffffu, ws, l);
                    // behind its first KD_PAIR places a pair is cut, a short one is not
                    const int c = nl <= KD_WHOLE ? 0 : max(0, nl - (wl - (int)y[e]));
                    x[e] += before + (sl - nl) + c;
                    if (e == 0) place = {ht[0], b0 + l, c, nl};
                }
                y[e] -= all;
            }
            before += __shfl_sync(0xffffffffu, s, 31);
        }
    }
    const long long x0 = x[0];
    const int n_mine = (int)(x[1] - x0);   // a list of 2^31 chunks would be 10 TB
    const auto next_request = [&](KdPlace& q) {   // the next one that has chunks
        do {
            if (++q.b == B) {
                q.b = 0;
                if (++q.ht == p.heads_t) {   // never, unless the lengths change under the kernel: then it ends all the same, inside its buffers
                    q.ht = p.heads_t - 1;
                    q.n = 0x7fffffff;
                    return;
                }
            }
            q.n = (length(q.b) + KD_CHUNK - 1) / KD_CHUNK;
        } while (q.n == 0);
    };

    // q of the eight heads, on its way while the copies are prepared
    uint4 w[4];
    const auto load_q = [&] {
        const int kvh = place.ht / p.q_tiles, q_tile = place.ht - kvh * p.q_tiles, h = 8 * q_tile + g;
        const uint4* src_q = reinterpret_cast<const uint4*>(static_cast<const T*>(p.a.d_q) + place.b * p.a.q_stride + (size_t)(kvh * p.group + h) * 128 + 32 * t);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = h < p.group ? src_q[j] : make_uint4(0, 0, 0, 0);
    };
    if (n_mine > 0) load_q();
    const auto rank_of = [&](int b) {   // requests before b that have tokens
        int r = 0;
        for (int i = lane; i < b; i += 32) r += length(i) > 0;
        return __reduce_add_sync(0xffffffffu, r);
    };

    // copies: chunk number k of this warp is number warp + 4 k of the CTA.  Thirty-two are looked up at once, one a lane.
    const int my_chunks = (n_mine - warp + KD_WARPS - 1) / KD_WARPS;
    KdPlace ahead = place;
    int ahead_at = 0, issued = 0;   // `ahead` is the place of the CTA's chunk number ahead_at; chunks issued
    const auto tile_at = [&](const KdPlace& q, int tile) -> const uint8_t* {   // null where the page is outside the pool
        const int in = tile / tiles_page, page = p.a.d_block_table[q.b * p.a.table_stride + in];
        if (page < 0 || page >= p.pool.n_pages) {
            kv4_error(p.err, KV4_ERR_DECODE_PAGE);
            return nullptr;
        }
        return static_cast<const uint8_t*>(p.pool.d_pages) + page * p.pool.page_stride +
               ((long long)(q.ht / p.q_tiles) * tiles_page + (tile - in * tiles_page)) * KV4_TILE_BYTES;
    };
    const auto look_up = [&]() {
        const int k = issued + lane, at = warp + KD_WARPS * k;
        int tokens = 0;
        const uint8_t *src0 = nullptr, *src1 = nullptr;
        KdPlace q = ahead;
        if (k < my_chunks) {
            int left = at - ahead_at;
            while (left >= q.n - q.c) {
                left -= q.n - q.c;
                q.c = 0;
                next_request(q);
            }
            q.c += left;
            const int tile = 2 * q.c, n0 = length(q.b) - 16 * tile, n1 = n0 - 16;
            if (n0 > 0) {
                src0 = tile_at(q, tile);
                if (src0 != nullptr) tokens = min(n0, 16);
            }
            if (n1 > 0) {
                src1 = tile_at(q, tile + 1);
                if (src1 != nullptr) tokens |= min(n1, 16) << 16;
            }
        }
        const bool one = tokens >> 16 != 0 && src1 - src0 == KV4_TILE_BYTES;   // of one page
        sm.src[warp][lane].at[0] = src0;
        sm.src[warp][lane].at[1] = one ? nullptr : src1;
        sm.tokens[warp][lane] = make_int2(tokens, one ? 2 * KV4_TILE_BYTES : (tokens & 0xffff) != 0 ? KV4_TILE_BYTES : 0);
        __syncwarp();
        // the next thirty-two are found from the last of these (used only where there is one)
        ahead.ht = __shfl_sync(0xffffffffu, q.ht, 31);
        ahead.b = __shfl_sync(0xffffffffu, q.b, 31);
        ahead.c = __shfl_sync(0xffffffffu, q.c, 31);
        ahead.n = __shfl_sync(0xffffffffu, q.n, 31);
        ahead_at = warp + KD_WARPS * (issued + 31);
    };
    const auto issue = [&]() {
        const int turn = issued & 31, s = issued % KD_STAGES;
        if (turn == 0) look_up();
        if (elect_one()) {
            const uint32_t bar = smem_u32(&sm.bar[warp][s]), to = smem_u32(sm.ring[warp][s]);
            const int2 n = sm.tokens[warp][turn];
            const uint8_t* const b = sm.src[warp][turn].at[1];
            sm.valid[warp][s] = n.x;
            mbar_expect_tx(bar, n.y + (b != nullptr ? KV4_TILE_BYTES : 0));
            if (n.y != 0) bulk_load(to, sm.src[warp][turn].at[0], n.y, bar);
            if (b != nullptr) bulk_load(to + KV4_TILE_BYTES, b, KV4_TILE_BYTES, bar);
        }
        __syncwarp();
        ++issued;
    };
    for (int s = 0; s < KD_STAGES && issued < my_chunks; ++s) issue();

    // requests without tokens: rows of zeros
    for (int b = blockIdx.x; b < B; b += gridDim.x) {
        const int n = p.a.d_kv_len[b];
        if (tid == 0 && (n < 0 || (long long)n > p.most_tokens)) kv4_error(p.err, KV4_ERR_DECODE_LEN);
        if (length(b) == 0)
            for (int i = tid; i < p.a.heads * 16; i += KD_THREADS) reinterpret_cast<uint4*>(static_cast<T*>(p.a.d_out) + (size_t)b * p.a.heads * 128)[i] = make_uint4(0, 0, 0, 0);
    }

    const int row0 = g ^ ((g >> 1) & 1);   // token of a tile that index g of a fragment stands for (and + 8): neighbours in t are of either parity,
                                           // which halves the bank conflicts of the V rows
    bool ok = true;
    int done = 0, used = 0;   // chunks of the CTA's that are behind, of this warp's
    while (done < n_mine) {
        const int part_end = min(n_mine, done + place.n - place.c);
        const int kvh = place.ht / p.q_tiles, q_tile = place.ht - kvh * p.q_tiles;
        const int nq = min(8, p.group - 8 * q_tile), head0 = kvh * p.group + 8 * q_tile;

        // q of the eight heads: fp16 fragments in the order of the nibbles (bf16: times a power of two of the head's own), and sums
        uint32_t qf[4][4];   // word j of a row: low nibbles k 0..7, 8..15, high nibbles the same
        float f0, f1, qs0, qs1;
        {
            constexpr bool HALF = R::FLOOR > 1e-9f;
            float sum = 0.0f, big = 0.0f, f = p.c;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t u[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 v = R::unpack(u[e]);
                    if (HALF) sum += v.x + v.y;
                    else big = fmaxf(big, fmaxf(fabsf(v.x), fabsf(v.y)));
                }
            }
            if (!HALF) {   // bf16: the largest value of the head goes to [2^14, 2^15); the sum is taken there, before it passes fp32
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                const int ex = (int)(__float_as_uint(big) >> 23);   // biased; 255 for Inf
                int shift = ex == 0 || ex == 255 ? 0 : 127 + 14 - ex;
                shift = min(shift, 100);
                const float up = __uint_as_float((uint32_t)(127 + shift) << 23);
                f *= __uint_as_float((uint32_t)(127 - shift) << 23);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t* u = &w[j].x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 v = R::unpack(u[e]);
                        const float a = v.x * up, b = v.y * up;
                        sum += a + b;
                        u[e] = RowType<__half>::pack(a, b);
                    }
                }
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                qf[j][0] = __byte_perm(w[j].x, w[j].z, 0x5410);
                qf[j][1] = __byte_perm(w[j].y, w[j].w, 0x5410);
                qf[j][2] = __byte_perm(w[j].x, w[j].z, 0x7632);
                qf[j][3] = __byte_perm(w[j].y, w[j].w, 0x7632);
            }
            const int from = 4 * (NARROW ? 2 * (t & 1) : 2 * t);   // of the lane's two heads
            f0 = __shfl_sync(0xffffffffu, f, from);
            f1 = __shfl_sync(0xffffffffu, f, from + 4);
            qs0 = __shfl_sync(0xffffffffu, sum, from);
            qs1 = __shfl_sync(0xffffffffu, sum, from + 4);
        }

        int unflushed = 0;      // chunks in the accumulators
        bool flushed = false;   // sm.o holds sums
        float o[8][4], eight[4];   // dims 16 g + 4 (i / 2) + i % 2 and + 2, heads 2t and 2t + 1: sums of P code, and of P * 8; odd i: 16 times that
        const auto clear = [&] {
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
            eight[0] = eight[1] = eight[2] = eight[3] = 0.0f;
        };
        const auto flush = [&](float r0, float r1) {   // (sums + accumulators) times a factor a head
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float4* const at = &sm.o[warp][i][lane];
                const float4 a = flushed ? *at : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                const float up = i & 1 ? -16.0f : -1.0f, e0 = eight[0], e1 = eight[1];   // all rows of the product are the same
                *at = make_float4((a.x + fmaf(up, e0, o[i][0])) * r0, (a.y + fmaf(up, e1, o[i][1])) * r1, (a.z + fmaf(up, e0, o[i][2])) * r0,
                                  (a.w + fmaf(up, e1, o[i][3])) * r1);
            }
            unflushed = 0;
            flushed = true;
        };
        clear();
        float top0 = -INFINITY, top1 = -INFINITY, z0 = 0.0f, z1 = 0.0f;   // mu + 7, beyond which it has to follow, and mu - 8
        float mu0 = -INFINITY, mu1 = -INFINITY, l0 = 0.0f, l1 = 0.0f, m0 = 0.0f, m1 = 0.0f;

        for (; warp + KD_WARPS * used < part_end; ++used) {
            const int s = used % KD_STAGES;
            const uint32_t bar = smem_u32(&sm.bar[warp][s]), parity = (uint32_t)(used / KD_STAGES) & 1u;
            if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) {
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, parity));
                if (!ok) continue;   // reported below
            }
            const uint8_t* const stage = sm.ring[warp][s];
            {   // lane i: what belongs to token i of the chunk; behind the last one nothing is left but codes, which are finite, times zero
                const uint8_t* const tile = stage + (lane >> 4) * KV4_TILE_BYTES + 4 * (lane & 15);
                const float2 ks = R::unpack(*reinterpret_cast<const uint32_t*>(tile + KV4_KP)), vs = R::unpack(*reinterpret_cast<const uint32_t*>(tile + KV4_VP));
                const int valid = sm.valid[warp][s];
                const float sv = kd_scale<T>(vs.x);
                float4 of = make_float4(ks.x * 16777216.0f, ks.y, kd_lg2(sv), kd_rcp(sv));
                float mid = fmaf(8.0f, sv, vs.y);
                if (valid != (16 | 16 << 16) && (lane & 15) >= (valid >> (lane & 16) & 0xffff)) {
                    of = make_float4(0.0f, 0.0f, -INFINITY, 0.0f);
                    mid = 0.0f;
                }
                sm.token[warp][lane] = of;
                sm.mid[warp][lane] = mid;
            }
            __syncwarp();
            float sum[2][4];     // of a tile: tokens row0, row0 + 8 x heads 2t, 2t + 1
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint8_t* const tile = stage + e * KV4_TILE_BYTES;
                const uint4 ka = *reinterpret_cast<const uint4*>(tile + row0 * 64 + 16 * t), kb = *reinterpret_cast<const uint4*>(tile + row0 * 64 + 512 + 16 * t);
                const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
                float lo[4], hi[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t a8 = wa[j] >> 8, b8 = wb[j] >> 8;
                    if (j == 0) {
                        kd_mma_first(lo, wa[j] & 0x000f000fu, wb[j] & 0x000f000fu, a8 & 0x000f000fu, b8 & 0x000f000fu, qf[j][0], qf[j][1]);
                        kd_mma_first(hi, wa[j] & 0x00f000f0u, wb[j] & 0x00f000f0u, a8 & 0x00f000f0u, b8 & 0x00f000f0u, qf[j][2], qf[j][3]);
                    } else {
                        mma_16816(lo, wa[j] & 0x000f000fu, wb[j] & 0x000f000fu, a8 & 0x000f000fu, b8 & 0x000f000fu, qf[j][0], qf[j][1]);
                        mma_16816(hi, wa[j] & 0x00f000f0u, wb[j] & 0x00f000f0u, a8 & 0x00f000f0u, b8 & 0x00f000f0u, qf[j][2], qf[j][3]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[e][i] = fmaf(hi[i], 0.0625f, lo[i]);
            }
            if (NARROW) {        // lanes of t = 2, 3: the second tile's, of the heads of t = 0, 1
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float other = __shfl_xor_sync(0xffffffffu, sum[1][i], 2);
                    sum[0][i] = t < 2 ? sum[0][i] : other;
                }
            }
            constexpr int TILES = NARROW ? 1 : 2;   // that the lane has values of
            float u[TILES][4], inv[TILES][2];
            float x0m = -INFINITY, x1m = -INFINITY;
#pragma unroll
            for (int e = 0; e < TILES; ++e)
#pragma unroll
                for (int h = 0; h < 2; ++h) {   // token row0 + 8 h
                    const float4 k = sm.token[warp][16 * (NARROW ? t >> 1 : e) + row0 + 8 * h];
                    u[e][2 * h] = fmaf(f0, fmaf(k.x, sum[e][2 * h], k.y * qs0), k.z);
                    u[e][2 * h + 1] = fmaf(f1, fmaf(k.x, sum[e][2 * h + 1], k.y * qs1), k.z);
                    inv[e][h] = k.w;
                    x0m = fmaxf(x0m, u[e][2 * h]);
                    x1m = fmaxf(x1m, u[e][2 * h + 1]);
                }
            if (__any_sync(0xffffffffu, x0m > top0 || x1m > top1)) {   // rare after the first chunks
#pragma unroll
                for (int d = NARROW ? 2 : 4; d < 32; d *= 2) {
                    x0m = fmaxf(x0m, __shfl_xor_sync(0xffffffffu, x0m, d));
                    x1m = fmaxf(x1m, __shfl_xor_sync(0xffffffffu, x1m, d));
                }
                const float n0 = fmaxf(mu0, x0m), n1 = fmaxf(mu1, x1m);
                const float r0 = mu0 == -INFINITY ? 0.0f : kd_ex2(mu0 - n0), r1 = mu1 == -INFINITY ? 0.0f : kd_ex2(mu1 - n1);
                mu0 = n0;
                mu1 = n1;
                top0 = mu0 + 7.0f;
                top1 = mu1 + 7.0f;
                z0 = mu0 == -INFINITY ? 0.0f : mu0 - 8.0f;
                z1 = mu1 == -INFINITY ? 0.0f : mu1 - 8.0f;
                l0 *= r0; m0 *= r0;
                l1 *= r1; m1 *= r1;
                if (flushed || unflushed > 0) {
                    flush(r0, r1);
                    clear();
                }
            }
            if (unflushed == KD_FLUSH) {
                flush(1.0f, 1.0f);
                clear();
            }
            ++unflushed;
            uint32_t pp[TILES][2], low[2], other[2];   // P; LOW: what its rounding took off; what the lane needs from the one opposite
#pragma unroll
            for (int e = 0; e < TILES; ++e)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float mid = sm.mid[warp][16 * (NARROW ? t >> 1 : e) + row0 + 8 * h];
                    const float p0 = kd_ex2(u[e][2 * h] - z0), p1 = kd_ex2(u[e][2 * h + 1] - z1);
                    const float w0 = p0 * inv[e][h], w1 = p1 * inv[e][h];
                    l0 += w0;
                    l1 += w1;
                    m0 = fmaf(w0, mid, m0);
                    m1 = fmaf(w1, mid, m1);
                    pp[e][h] = RowType<__half>::pack(p0, p1);
                    if (LOW) {
                        const float2 rounded = RowType<__half>::unpack(pp[e][h]);
                        low[h] = RowType<__half>::pack(p0 - rounded.x, p1 - rounded.y);
                    } else {
                        low[h] = pp[e][h];
                    }
                    if (NARROW) other[h] = __shfl_xor_sync(0xffffffffu, t < 2 ? low[h] : pp[e][h], 2);
                }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint8_t* const tile = stage + e * KV4_TILE_BYTES + KV4_V;
                uint32_t pf[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) pf[h] = kd_transpose(!NARROW ? pp[e % TILES][h] : t < 2 ? (e == 0 ? pp[0][h] : other[h]) : (e == 0 ? other[h] : low[h]));
                const int ra = 2 * t + (t & 1), rb = 2 * t + (~t & 1);   // tokens of indexes 2t and 2t + 1
                const uint2 a0 = *reinterpret_cast<const uint2*>(tile + ra * 64 + 8 * g), b0 = *reinterpret_cast<const uint2*>(tile + rb * 64 + 8 * g);
                const uint2 a1 = *reinterpret_cast<const uint2*>(tile + ra * 64 + 512 + 8 * g), b1 = *reinterpret_cast<const uint2*>(tile + rb * 64 + 512 + 8 * g);
                mma_16816(eight, 0x00080008u, 0x00080008u, 0x00080008u, 0x00080008u, pf[0], pf[1]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {   // dims 16 g + 4 i .. + 3
                    const int sel = i & 1 ? 0x7632 : 0x5410;
                    const uint32_t x = i < 2 ? __byte_perm(a0.x, b0.x, sel) : __byte_perm(a0.y, b0.y, sel);
                    const uint32_t y = i < 2 ? __byte_perm(a1.x, b1.x, sel) : __byte_perm(a1.y, b1.y, sel);
                    const uint32_t x8 = x >> 8, y8 = y >> 8;
                    mma_16816(o[2 * i], x & 0x000f000fu, x8 & 0x000f000fu, y & 0x000f000fu, y8 & 0x000f000fu, pf[0], pf[1]);
                    mma_16816(o[2 * i + 1], x & 0x00f000f0u, x8 & 0x00f000f0u, y & 0x00f000f0u, y8 & 0x00f000f0u, pf[0], pf[1]);
                }
            }
            __syncwarp();
            if (issued < my_chunks) issue();
        }

        // the states of the four warps, then of the CTAs that share the pair
#pragma unroll
        for (int d = NARROW ? 2 : 4; d < 32; d *= 2) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, d);
            l1 += __shfl_xor_sync(0xffffffffu, l1, d);
            m0 += __shfl_xor_sync(0xffffffffu, m0, d);
            m1 += __shfl_xor_sync(0xffffffffu, m1, d);
        }
        if (!ok) l0 = l1 = NAN;
        if (g == 0 && (!NARROW || t < 2)) {
            float* const st = sm.stat[warp][2 * t];
            st[0] = mu0; st[1] = l0; st[2] = m0;
            st[3] = mu1; st[4] = l1; st[5] = m1;
        }
        flush(1.0f, 1.0f);
        __syncthreads();
        // thread (i, lane): dims 16 g + 4 i .. + 3 of heads 2t and 2t + 1
        const int i = warp, ts = NARROW ? t & 1 : t;   // statistics of its heads
        float top[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, m[2] = {0.0f, 0.0f};
        float4 lo = make_float4(0, 0, 0, 0), hi = make_float4(0, 0, 0, 0);
        const auto add = [&](int h, float mu, float sl, float smv) {   // joins a state's sums of head 2t + h; returns its factor
            const float f = mu == -INFINITY ? 0.0f : kd_ex2(mu - top[h]);
            // a state without tokens adds nothing, one that gave up adds its NaN
            l[h] += mu == -INFINITY ? (sl != sl ? sl : 0.0f) : sl * f;
            m[h] += mu == -INFINITY ? 0.0f : smv * f;
            return f;
        };
        const auto accumulate = [&](float4& to, const float4& from, float fa, float fb) {
            to.x = fmaf(from.x, fa, to.x);
            to.y = fmaf(from.y, fb, to.y);
            to.z = fmaf(from.z, fa, to.z);
            to.w = fmaf(from.w, fb, to.w);
        };
#pragma unroll
        for (int w = 0; w < KD_WARPS; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h) top[h] = fmaxf(top[h], sm.stat[w][2 * ts + h][0]);
#pragma unroll
        for (int w = 0; w < KD_WARPS; ++w) {
            const float* const st = sm.stat[w][2 * ts];
            const float fa = add(0, st[0], st[1], st[2]), fb = add(1, st[3], st[4], st[5]);
            accumulate(lo, sm.o[w][2 * i][lane], fa, fb);
            accumulate(hi, sm.o[w][2 * i + 1][lane], fa, fb);
        }
        if (LOW) {   // the sums of P and of what its rounding took off
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                (&lo.x)[e] += __shfl_xor_sync(0xffffffffu, (&lo.x)[e], 2);
                (&hi.x)[e] += __shfl_xor_sync(0xffffffffu, (&hi.x)[e], 2);
            }
        }
        int first = 0, parts = 1;   // CTAs that have a part of the pair
        if (place.n > KD_WHOLE && (place.c > 0 || done + place.n > n_mine)) {
            // its first chunk in the places that count KD_PAIR for each pair: chunks before it, and the pairs
            const long long start = x0 + done - place.c + (long long)KD_PAIR * ((long long)place.ht * busy + rank_of(place.b) + 1);
            first = owner_of(start, grid, total);
            parts = owner_of(start + place.n - 1, grid, total) - first + 1;
        }
        bool write = true;
        if (parts > 1) {
            const auto slot = [&](int k) { return p.part + (size_t)(k == 0 ? 2 * first + 1 : 2 * (first + k)) * KD_PART; };
            float* const mine = slot((int)blockIdx.x - first);
            reinterpret_cast<float4*>(mine)[(2 * i) * 32 + lane] = lo;
            reinterpret_cast<float4*>(mine)[(2 * i + 1) * 32 + lane] = hi;
            if (warp == 0 && g == 0) {
                float* const st = mine + 1024 + 6 * t;
                st[0] = top[0]; st[1] = l[0]; st[2] = m[0];
                st[3] = top[1]; st[4] = l[1]; st[5] = m[1];
            }
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const int before = atomicAdd(p.count + first, 1);
                sm.last = before == parts - 1;
                if (sm.last) p.count[first] = 0;
            }
            __syncthreads();
            write = sm.last != 0;
            if (write) {
                __threadfence();
                // maxima and factors of the parts, sixty-four at a time, a head and every sixteenth part a thread
                float* const scratch = reinterpret_cast<float*>(sm.o);   // [64][8] factors, [16][8] of the threads
                const int h8 = tid & 7, k8 = tid >> 3;
                float st[4][3], mx = -INFINITY;
                const auto load = [&](int k0) {
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int e = 0; e < 3; ++e) {
                            const int k = k0 + k8 + 16 * u;
                            st[u][e] = k < parts ? __ldcg(slot(k) + 1024 + 3 * h8 + e) : e == 0 ? -INFINITY : 0.0f;
                        }
                };
                for (int k0 = (parts - 1) / 64 * 64; k0 >= 0; k0 -= 64) {   // the first sixty-four stay in registers
                    load(k0);
#pragma unroll
                    for (int u = 0; u < 4; ++u) mx = fmaxf(mx, st[u][0]);
                }
                __syncthreads();   // sm.o has been read
                scratch[512 + tid] = mx;
                __syncthreads();
#pragma unroll
                for (int k = 0; k < 16; ++k) mx = fmaxf(mx, scratch[512 + 8 * k + h8]);
                float sl = 0.0f, smv = 0.0f;
                lo = hi = make_float4(0, 0, 0, 0);
                for (int k0 = 0; k0 < parts; k0 += 64) {
                    if (k0 > 0) {
                        __syncthreads();
                        load(k0);
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) {   // a part without tokens adds nothing, one that gave up adds its NaN
                        const bool none = st[u][0] == -INFINITY;
                        const float f = none ? 0.0f : kd_ex2(st[u][0] - mx);
                        scratch[8 * (k8 + 16 * u) + h8] = f;
                        sl += none ? (st[u][1] != st[u][1] ? st[u][1] : 0.0f) : st[u][1] * f;
                        smv += none ? 0.0f : st[u][2] * f;
                    }
                    __syncthreads();
#pragma unroll 8
                    for (int k = k0; k < min(parts, k0 + 64); ++k) {
                        const float4* const from = reinterpret_cast<const float4*>(slot(k));
                        const float fa = scratch[8 * (k - k0) + 2 * t], fb = scratch[8 * (k - k0) + 2 * t + 1];
                        accumulate(lo, __ldcg(from + (2 * i) * 32 + lane), fa, fb);
                        accumulate(hi, __ldcg(from + (2 * i + 1) * 32 + lane), fa, fb);
                    }
                }
                scratch[512 + tid] = sl;
                scratch[640 + tid] = smv;
                __syncthreads();
                l[0] = l[1] = m[0] = m[1] = 0.0f;
#pragma unroll
                for (int k = 0; k < 16; ++k)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        l[h] += scratch[512 + 8 * k + 2 * t + h];
                        m[h] += scratch[640 + 8 * k + 2 * t + h];
                    }
            }
        }
        if (write) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (2 * t + h >= nq) continue;
                const float r = 1.0f / l[h], a = 16777216.0f, b = 1048576.0f;   // what the nibbles' places stand for
                const float v0 = fmaf(h ? lo.y : lo.x, a, m[h]) * r, v1 = fmaf(h ? hi.y : hi.x, b, m[h]) * r;
                const float v2 = fmaf(h ? lo.w : lo.z, a, m[h]) * r, v3 = fmaf(h ? hi.w : hi.z, b, m[h]) * r;
                T* const dst = static_cast<T*>(p.a.d_out) + ((size_t)place.b * p.a.heads + head0 + 2 * t + h) * 128 + 16 * g + 4 * i;
                const bool any = l[h] != 0.0f;   // no page of the request was inside the pool
                *reinterpret_cast<uint2*>(dst) = any ? make_uint2(R::pack(v0, v1), R::pack(v2, v3)) : make_uint2(0, 0);
            }
        }
        done = part_end;
        if (done < n_mine) {
            place.c = 0;
            next_request(place);
            load_q();
            __syncthreads();   // sm.o and sm.stat are read
        }
    }
    if (!ok) {   // a copy that did not land in time: the ones in flight are waited for
        if (lane == 0) atomicCAS(p.err, 0, 0x30031);
        for (int k = 0; k < KD_STAGES && k < issued; ++k)
            mbar_wait(smem_u32(&sm.bar[warp][(issued - 1 - k) % KD_STAGES]), (uint32_t)((issued - 1 - k) / KD_STAGES) & 1u);
    }
}

}  // namespace qw3

using namespace qw3;

extern "C" int qw3_attn_kv4_decode(const Qw3Kv4Pool* pool, const Qw3AttnKv4Args* a, qw3_ws_t ws, void* stream) {
    const char* who = "qw3_attn_kv4_decode";
    QW3_REQUIRE(a, "%s: null argument", who);
    int rc = kv4_check(who, pool, ws);
    if (rc != QW3_OK) return rc;
    QW3_REQUIRE(a->n_req >= 0, "%s: n_req out of range", who);
    if (a->n_req == 0) return QW3_OK;
    QW3_REQUIRE(a->d_q && a->d_block_table && a->d_kv_len && a->d_out, "%s: null pointer", who);
    QW3_REQUIRE(a->heads > 0 && a->heads <= 4096 && a->heads % pool->kv_heads == 0, "%s: heads must be a multiple of kv_heads", who);
    QW3_REQUIRE(a->q_stride >= (int64_t)a->heads * 128 && a->q_stride % 8 == 0 && a->q_stride < ((int64_t)1 << 31), "%s: q_stride must be a multiple of 8 and hold the heads", who);
    QW3_REQUIRE(a->max_blocks > 0 && a->table_stride >= a->max_blocks, "%s: block table out of range", who);
    QW3_REQUIRE(((reinterpret_cast<uintptr_t>(a->d_q) | reinterpret_cast<uintptr_t>(a->d_out)) & 15) == 0, "%s: q and out must be 16-byte aligned", who);
    QW3_REQUIRE(fabsf(a->scale) <= KV4_MAX_SCALE, "%s: scale must be finite, 2e38 at most", who);
    const Workspace* w = ws_struct(ws);
    KdParams p;
    p.pool = *pool;
    p.a = *a;
    p.group = a->heads / pool->kv_heads;
    p.q_tiles = (p.group + 7) / 8;
    p.heads_t = pool->kv_heads * p.q_tiles;
    p.most_tokens = (long long)a->max_blocks * pool->page_size;
    if (p.most_tokens > 0x7fffffff - 64) p.most_tokens = 0x7fffffff - 64;
    p.c = (float)((a->scale == 0.0f ? 0.08838834764831845 : (double)a->scale) * 1.4426950408889634);
    p.part = w->partials;
    p.count = w->counters;
    p.err = w->err;
    // CTAs that the longest rows of the table could keep busy
    const double most = (double)a->n_req * p.heads_t * (double)((p.most_tokens + KD_CHUNK - 1) / KD_CHUNK) / KD_MIN_CHUNKS;
    int grid = w->sm_count * KD_CTAS;
    if (grid > KD_MAX_GRID) grid = KD_MAX_GRID;
    if (most < grid) grid = most < 1.0 ? 1 : (int)most;
    void (*const kernels[4])(KdParams) = {attn_kv4_decode_kernel<__half, false>, attn_kv4_decode_kernel<__half, true>,
                                          attn_kv4_decode_kernel<__nv_bfloat16, false>, attn_kv4_decode_kernel<__nv_bfloat16, true>};
    const auto kernel = kernels[(pool->dtype == QW3_F16 ? 0 : 2) + (p.group <= 4 ? 1 : 0)];
    static std::atomic<bool> attr_set[64];   // per device: the kernels' shared-memory limit is raised once
    if (w->device >= 64 || !attr_set[w->device].load(std::memory_order_acquire)) {
        for (const auto k : kernels) QW3_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(KdSmem)));
        if (w->device < 64) attr_set[w->device].store(true, std::memory_order_release);
    }
    QW3_CUDA(kv4_launch(kernel, dim3(grid), dim3(KD_THREADS), sizeof(KdSmem), static_cast<cudaStream_t>(stream), ws_pdl(ws), 1, p));
    return QW3_OK;
}
