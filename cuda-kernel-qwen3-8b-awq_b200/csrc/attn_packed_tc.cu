// Causal attention of packed prompts of different lengths, heads grouped over KV heads, on the 5th-generation tensor cores (attentionKernel,
// Inference.cu:182-266, intended math).
//
// The queries of a sequence are its last rows: row i of nq sees keys 0 .. nk - nq + i.  One CTA takes 256 rows as two tiles of 128.  Where the
// group's size has a factor `pack` of two, a row is a (token, head) pair of `pack` heads of the group: they read the same keys, so a tile
// covers 128 / pack tokens, short sequences fill it, and less of the tiles on the diagonal is masked.  Both tiles read the same tiles of 128 keys.
// One CTA an SM, which takes block after block (256 rows of a sequence and a group) from a counter, the blocks with the most keys of a
// sequence first, so that the loads, the first scores and the next block's place are on their way during a block's epilogue.
// Twelve warps:
//   warp 0      takes and finds the blocks; TMA producer: the q rows, K and V tiles (128 keys x 128 dims, two 64-dim halves, 128-byte
//               swizzle), five in a ring
//   warp 1      MMA issuer: S = Q K^T (K-major operands from shared memory), O += P V with P from tensor memory and V MN-major as it lies
//   warp 2      zeroes the V rows behind the sequence in the last tile: they are other sequences' or nobody's, and 0 * NaN is NaN
//   warps 4..7, 8..11   one row a thread of the upper / lower tile: S from tensor memory, online softmax, P back in its place
// Tensor memory, per tile: O 128 columns, S 128, of which P takes the upper half as the exponentials consume it: the keys 64..127 first, so that
// their product runs under the exponentials of the others.  While one tile is in its softmax the tensor cores work for the other.
// 128 keys a tile: an MMA of 128 x 64 x 16 takes 48 cycles of shared-memory reads for 32 of products (with the softmax left out, before CTAs
// were persistent, 4001 rows took 129 us with 64 keys a tile and 110 with 128), one of 128 x 128 x 16 64 for 64.
// P is rounded to the rows' type, whose 8 or 11 bits the result has as well; its sum is taken before.  An fp16 P is kept between 2^8 and
// 2^15 at the row's maximum, so that its normal numbers reach 22 powers of two below.  O is rescaled only when a row's maximum has grown by
// more than 7 (bf16: 8) powers of two.
// 4001 rows, 32 heads over 8 KV heads, bf16: 126 us, 1040 TFLOP/s, 0.62 of the measured rate (137 us in sustained use).  The tensor pipe is active
// in 57 % of active cycles, the exponential unit in 40 %; in an earlier build with timers a softmax warp waited 1140 of some 3660 cycles a tile for scores.
// All waits are bounded, by a second and what 32 rows done again may take: over 250000 keys 1.1 s, and the block behind them waits for that.
// After a wait that gives up the error word is set, the rows that the CTA has begun are written as NaN, blocks that no other CTA takes stay
// as they were, and the CTA leaves when its copies and MMAs in flight are done.
#include <atomic>

#include "kv4.cuh"
#include "tc05.cuh"

namespace qw3 {

constexpr int PK_ROWS = 128, PK_KEYS = 128, PK_STAGES = 5;
constexpr int PK_THREADS = 384;
constexpr int PK_Q_BYTES = PK_ROWS * 256;   // one tile of q rows: two halves of 64 dims
constexpr int PK_KV_BYTES = PK_KEYS * 256;  // one tile of K or V
constexpr long long PK_REDO_TICKS = 32 * 1024;   // a key: four times what a warp was away for that did 32 rows again over 250000 keys
constexpr size_t PK_SMEM = 2 * PK_Q_BYTES + (size_t)PK_STAGES * PK_KV_BYTES + 512;

__device__ __forceinline__ float pk_ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// 2^x for two x up to 30, on the FMA pipe: the exponential unit (16 results a clock and SM) is what the softmax waits for.  x = n + f with n the
// nearest whole number, which 1.5 * 2^23 + x has in its last bits; 2^f by a polynomial of degree 4 that is 1 at 0 (minimax on [-1/2, 1/2] by
// Remez' exchange: relative error 3.6e-6); n is added to the exponent.  Below -127, -Inf included, exactly 0.  Not for NaN:
// a row that sees one has it in its maximum.
__device__ __forceinline__ float2 pk_ex2_fma(float2 x) {
    constexpr float MAGIC = 12582912.0f;
    x = make_float2(fmaxf(x.x, -127.0f), fmaxf(x.y, -127.0f));
    const float2 t = add2(x, make_float2(MAGIC, MAGIC)), n = add2(t, make_float2(-MAGIC, -MAGIC)), f = add2(x, make_float2(-n.x, -n.y));
    float2 p = fma2(make_float2(0.009782911186619846f, 0.009782911186619846f), f, make_float2(0.055976883149044095f, 0.055976883149044095f));
    p = fma2(p, f, make_float2(0.24020711100517408f, 0.24020711100517408f));
    p = fma2(p, f, make_float2(0.693113604482677f, 0.693113604482677f));
    p = fma2(p, f, make_float2(1.0f, 1.0f));
    return make_float2(__uint_as_float(__float_as_uint(t.x) * 8388608u + __float_as_uint(p.x)), __uint_as_float(__float_as_uint(t.y) * 8388608u + __float_as_uint(p.y)));
}

// the largest of three, NaN where one is
__device__ __forceinline__ float pk_max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
constexpr int PK_FMA = 5;   // of sixteen pairs of exponentials, those on the FMA pipe
struct PackedParams {
    Qw3AttnPackedArgs a;
    float c;        // scale * log2(e)
    long long limit;   // clock ticks after which a wait gives up
    int pack;       // heads that share a tile
    int* ticket;    // the next block to be taken, and the CTAs that are done; zero between launches
    int* done;
    int* err;
};
// A block of rows: its sequence's first row and number of rows in q and in k, its number in the sequence (below 0: no more blocks), and
// its first head.
struct PackedBlock {
    int q0, k0, nq, nk, block, head0;
};

// As mbar_wait, with a limit of the call's own.
__device__ __forceinline__ bool packed_wait(uint32_t bar, uint32_t parity, long long limit) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity)) {
        if (clock64() - t0 > limit) return false;
    }
    return true;
}

// One row by a warp, from global memory and in 32-bit arithmetic: rows whose tile holds Inf or NaN in V behind the row, or whose sum of P V passes
// fp32.  The tensor cores multiply what is behind the row by the zeros of the masked probabilities, and the sum is NaN; here nothing past the row's
// last key is read.
template <class T>
__device__ __noinline__ void packed_row(const T* q, const T* k, long long k_stride, const T* v, long long v_stride, int n_keys, float c, T* dst, int lane) {
    using R = RowType<T>;
    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};   // outputs 4 lane .. 4 lane + 3
    for (int k0 = 0; k0 < n_keys; k0 += 32) {
        float s = -INFINITY;
        if (k0 + lane < n_keys) {
            const uint4* kr = reinterpret_cast<const uint4*>(k + (k0 + lane) * k_stride);
            const uint4* qr = reinterpret_cast<const uint4*>(q);
            s = 0.0f;
            for (int i = 0; i < 16; ++i) {
                const uint4 a = qr[i], b = kr[i];
                const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 x = R::unpack(aw[e]), y = R::unpack(bw[e]);
                    s = fmaf(x.y, y.y, fmaf(x.x, y.x, s));
                }
            }
        }
        float mn = fmaxf(m, s);
        for (int d = 16; d > 0; d >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, d));
        const float f = m == -INFINITY ? 0.0f : pk_ex2((m - mn) * c), pr = s == -INFINITY ? 0.0f : pk_ex2((s - mn) * c);
        m = mn;
        l = l * f + pr;   // this lane's keys
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= f;
        for (int j0 = 0; j0 < 32; j0 += 8) {   // eight loads on their way at once
            uint2 w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = k0 + j0 + j < n_keys ? *reinterpret_cast<const uint2*>(v + (k0 + j0 + j) * v_stride + 4 * lane) : make_uint2(0, 0);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float pj = __shfl_sync(0xffffffffu, pr, j0 + j);
                const float2 a = R::unpack(w[j].x), b = R::unpack(w[j].y);
                o[0] = fmaf(pj, a.x, o[0]);
                o[1] = fmaf(pj, a.y, o[1]);
                o[2] = fmaf(pj, b.x, o[2]);
                o[3] = fmaf(pj, b.y, o[3]);
            }
        }
    }
    for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    *reinterpret_cast<uint2*>(dst + 4 * lane) = make_uint2(R::pack(o[0] / l, o[1] / l), R::pack(o[2] / l, o[3] / l));
}

// Which of a warp's rows (`rows`, one a lane: its last key `pos`, its stored result `dst`) have to be done again: those with a value that is not
// finite in a dim where no V row that they see has Inf or NaN.  The others are what the definition gives, however many they are.  One pass
// over V, up to the first such value in every dim that is asked for: 32 keys a step.
template <class T>
__device__ __noinline__ uint32_t packed_spoiled(uint32_t rows, int pos, const T* dst, const T* v, long long v_stride, int lane) {
    using R = RowType<T>;
    const auto bad = [](uint2 w) {   // of the lane's four dims, a bit each
        const float2 a = R::unpack(w.x), b = R::unpack(w.y);
        return (a.x - a.x != 0.0f ? 1u : 0u) | (a.y - a.y != 0.0f ? 2u : 0u) | (b.x - b.x != 0.0f ? 4u : 0u) | (b.y - b.y != 0.0f ? 8u : 0u);
    };
    const auto result = [&](int row) {
        const T* const at = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), row));
        return bad(*reinterpret_cast<const uint2*>(at + 4 * lane));
    };
    uint32_t asked = 0;
    for (uint32_t m = rows; m != 0; m &= m - 1) asked |= result(__ffs(m) - 1);
    const int n = __reduce_max_sync(0xffffffffu, rows >> lane & 1 ? pos + 1 : 0);
    int first[4] = {0x7fffffff, 0x7fffffff, 0x7fffffff, 0x7fffffff};   // key of the first Inf or NaN in a dim
    for (int k0 = 0; k0 < n && __any_sync(0xffffffffu, asked != 0); k0 += 32)
        for (int j0 = 0; j0 < 32; j0 += 8) {
            uint2 w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = k0 + j0 + j < n ? *reinterpret_cast<const uint2*>(v + (k0 + j0 + j) * v_stride + 4 * lane) : make_uint2(0, 0);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t now = bad(w[j]) & asked;
                asked &= ~now;
#pragma unroll
                for (int e = 0; e < 4; ++e) first[e] = now >> e & 1 ? k0 + j0 + j : first[e];
            }
        }
    uint32_t again = 0;
    for (uint32_t m = rows; m != 0; m &= m - 1) {
        const int row = __ffs(m) - 1, last = __shfl_sync(0xffffffffu, pos, row);
        const uint32_t b = result(row);
        bool spoiled = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) spoiled |= (b >> e & 1) != 0 && first[e] > last;
        if (__any_sync(0xffffffffu, spoiled)) again |= 1u << row;
    }
    return again;
}

template <class T>
__global__ void __launch_bounds__(PK_THREADS, 1)
attn_packed_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                   const PackedParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ PackedBlock s_block[2];
    using R = RowType<T>;
    constexpr bool HALF = R::FLOOR > 1e-9f;                        // fp16
    constexpr float SHIFT = HALF ? 8.0f : 0.0f, LAG = HALF ? 7.0f : 8.0f;
    uint8_t* q_s = smem;
    uint8_t* kv_s = q_s + 2 * PK_Q_BYTES;   // a ring: K of a key tile, V of it, K of the next, ..
    uint64_t* bars = reinterpret_cast<uint64_t*>(kv_s + PK_STAGES * PK_KV_BYTES);
    // phases: of a block: q_*, o_* [tile]; of a key tile: s_full, p_full [tile][half]; of every second block: place_* [block & 1]
    const uint32_t q_full = smem_u32(bars), q_empty = q_full + 8, full = q_empty + 8, empty = full + 8 * PK_STAGES, s_full = empty + 8 * PK_STAGES,
                   p_full = s_full + 16, o_full = p_full + 32, o_empty = o_full + 16, place_full = o_empty + 16, place_empty = place_full + 16,
                   drain = place_empty + 16, v_last = drain + 8, v_clean = v_last + 8;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * PK_STAGES + 19);
    volatile int* s_dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const auto wait = [&](uint32_t bar, uint32_t parity) { return packed_wait(bar, parity, p.limit); };

    const auto give_up = [&](int code) {
        atomicCAS(p.err, 0, code);
        *s_dead = 1;
    };
    const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
    const int pack = p.pack, block_tokens = 2 * PK_ROWS / pack, tile_tokens = PK_ROWS / pack;
    const int groups = p.a.heads / pack;
    pdl_launch_dependents();

    if (tid == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        mbar_init(drain, 1);
        mbar_init(v_last, 1);
        mbar_init(v_clean, 1);
        for (int s = 0; s < PK_STAGES; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(o_full + 8 * i, 1);
            mbar_init(o_empty + 8 * i, 4);   // the four warps of the tile
            mbar_init(place_full + 8 * i, 1);
            mbar_init(place_empty + 8 * i, 10);   // warps 1, 2 and the eight of the softmax
        }
        for (int i = 0; i < 4; ++i) mbar_init(p_full + 8 * i, 4);
        *s_dead = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;   // O of the tiles at columns 0 and 128, S at 256 + 128 tile, P at 64 columns of that + 32 half
    pdl_wait();

    // what follows from a block's place
    struct Shape {
        int t0, past, n_keys, n_tiles;   // token i of the block is t0 + i of the sequence's queries; it sees keys 0 .. past + t0 + i
        bool short_last, ragged;         // of the last key tile only the first half has keys; its V has rows that are not the sequence's
    };
    const auto shape_of = [&](const PackedBlock& b) {
        Shape s;
        s.t0 = b.block * block_tokens;
        s.past = b.nk - b.nq;
        s.n_keys = max(0, min(b.nk, s.past + min(s.t0 + block_tokens, b.nq)));
        s.n_tiles = (s.n_keys + PK_KEYS - 1) / PK_KEYS;
        s.short_last = s.n_keys - (s.n_tiles - 1) * PK_KEYS <= PK_KEYS / 2;
        s.ragged = s.n_keys % (PK_KEYS / 2) != 0;
        return s;
    };

    if (warp == 0) {
        const auto sequence = [&](int s, int& q0, int& nq, int& k0, int& nk) {   // false where it is not inside the buffers, which leaves it without rows
            q0 = nq = k0 = nk = 0;
            if (s < 0) return true;
            const int qa = p.a.d_cu_q[s], qb = p.a.d_cu_q[s + 1], ka = p.a.d_cu_k[s], kb = p.a.d_cu_k[s + 1];
            if (qa < 0 || qb < qa || (long long)qb > p.a.q_rows || ka < 0 || kb < ka || (long long)kb > p.a.k_rows) return false;
            q0 = qa; nq = qb - qa; k0 = ka; nk = kb - ka;
            return true;
        };
        if (blockIdx.x == 0)   // the reports
            for (int s = lane; s < p.a.n_seq; s += 32) {
                int q0, nq, k0, nk;
                if (!sequence(s, q0, nq, k0, nk)) kv4_error(p.err, KV4_ERR_PACKED_CU);
            }
        __syncwarp();
        int i = 0, used = 0;                  // tiles asked for, blocks with keys
        int seq0 = p.a.n_seq, passed = 0;     // the search for the next block: sequences below seq0 are left, the others have `passed` blocks
        for (int k = 0;; ++k) {
            PackedBlock b = {0, 0, 0, 0, -1, 0};
            if (*s_dead == 0) {
                const int ticket = __shfl_sync(0xffffffffu, lane == 0 ? atomicAdd(p.ticket, 1) : 0, 0), number = ticket / groups;
                b.head0 = (ticket - number * groups) * pack;
                // the last sequence's last block comes first; the numbers of a CTA grow, so the search goes on where it was
                while (seq0 > 0 && b.block < 0) {
                    int q0, nq, k0, nk;
                    sequence(seq0 - 1 - lane, q0, nq, k0, nk);
                    const int blocks = (nq + block_tokens - 1) / block_tokens;
                    int sum = blocks;
#pragma unroll
                    for (int d = 1; d < 32; d *= 2) {
                        const int x = __shfl_up_sync(0xffffffffu, sum, d);
                        if (lane >= d) sum += x;
                    }
                    const uint32_t hit = __ballot_sync(0xffffffffu, number - passed < sum);
                    if (hit != 0) {
                        const int from = __ffs(hit) - 1;
                        b.q0 = __shfl_sync(0xffffffffu, q0, from);
                        b.k0 = __shfl_sync(0xffffffffu, k0, from);
                        b.nq = __shfl_sync(0xffffffffu, nq, from);
                        b.nk = __shfl_sync(0xffffffffu, nk, from);
                        b.block = __shfl_sync(0xffffffffu, sum - 1 - (number - passed), from);
                    } else {
                        passed += __shfl_sync(0xffffffffu, sum, 31);
                        seq0 -= 32;
                    }
                }
            }
            const uint32_t at = 8 * (k & 1);
            if (k > 1 && !__all_sync(0xffffffffu, wait(place_empty + at, (uint32_t)((k >> 1) - 1) & 1u))) {
                if (lane == 0) give_up(0x30045);
                break;
            }
            if (lane == 0) {
                s_block[k & 1] = b;
                mbar_arrive(place_full + at);
            }
            if (b.block < 0) break;
            const Shape sh = shape_of(b);
            if (sh.n_tiles > 0 && elect_one()) {
                const int kv_head = b.head0 / (p.a.heads / p.a.kv_heads), end = i + 2 * sh.n_tiles;
                bool ok = used == 0 || wait(q_empty, (uint32_t)(used - 1) & 1u);
                const bool q_asked = ok;
                if (ok) {
                    mbar_expect_tx(q_full, 2 * PK_Q_BYTES);
                    for (int t = 0; t < 2; ++t)
                        for (int h = 0; h < 2; ++h)
                            tma_load_3d(smem_u32(q_s + t * PK_Q_BYTES + h * (PK_Q_BYTES / 2)), &tm_q, 64 * h, b.head0, b.q0 + sh.t0 + tile_tokens * t, q_full);
                }
                int n = i;
                for (int j = 0; ok && n < end; ++n) {
                    const int s = n % PK_STAGES, v = (n - i) & 1;
                    if (n >= PK_STAGES) ok = wait(empty + 8 * s, (uint32_t)(n / PK_STAGES - 1) & 1u);
                    if (*s_dead != 0) ok = false;
                    if (!ok) break;
                    mbar_expect_tx(full + 8 * s, PK_KV_BYTES);
                    for (int h = 0; h < 2; ++h)
                        tma_load_3d(smem_u32(kv_s + s * PK_KV_BYTES + h * (PK_KV_BYTES / 2)), v ? &tm_v : &tm_k, 64 * h, b.k0 + j * PK_KEYS, kv_head, full + 8 * s);
                    j += v;
                }
                if (!ok) {
                    give_up(0x30041);
                    if (q_asked) mbar_wait(q_full, (uint32_t)used & 1u);   // the copies in flight
                    for (int m = max(n - PK_STAGES, 0); m < n; ++m) mbar_wait(full + 8 * (m % PK_STAGES), (uint32_t)(m / PK_STAGES) & 1u);
                }
            }
            __syncwarp();
            if (sh.n_tiles > 0) {
                i += 2 * sh.n_tiles;
                ++used;
            }
        }
        // drain: the last release arrivals land before the CTA may leave
        if (*s_dead == 0 && used > 0) {
            bool ok = wait(q_empty, (uint32_t)(used - 1) & 1u);
            for (int m = max(i - PK_STAGES, 0); m < i && ok; ++m) ok = wait(empty + 8 * (m % PK_STAGES), (uint32_t)(m / PK_STAGES) & 1u);
            if (!ok && lane == 0) give_up(0x30046);
        }
        if (lane == 0 && atomicAdd(p.done, 1) == (int)gridDim.x - 1) {   // all CTAs have taken their last ticket
            atomicExch(p.ticket, 0);
            atomicExch(p.done, 0);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (elect_one()) {
            // D = f32, A and B of the rows' type.  S: N = keys, both K-major.  P V: N = 128 dims, V MN-major (bit 16).
            const uint32_t types = (1u << 4) | (HALF ? 0u : (1u << 7) | (1u << 10));
            const uint32_t rows = (uint32_t)(PK_ROWS >> 4) << 24, idesc_o = types | (1u << 16) | ((uint32_t)(128 >> 3) << 17) | rows;
            const uint64_t qd = make_smem_desc(smem_u32(q_s), 16, 1024), kd = make_smem_desc(smem_u32(kv_s), 16, 1024);
            const uint64_t vd = make_smem_desc(smem_u32(kv_s), PK_KV_BYTES / 2, 1024);   // 64-dim halves, 8-key groups
            const auto scores = [&](int t, int i, uint32_t keys, bool last) {   // S of tile t against tile i of the ring
                const int s = i % PK_STAGES;
                const uint32_t idesc = types | (keys >> 3) << 17 | rows;
                const uint64_t a = qd + (uint64_t)(t * (PK_Q_BYTES >> 4)), b = kd + (uint64_t)(s * (PK_KV_BYTES >> 4));
#pragma unroll
                for (int ks = 0; ks < 8; ++ks)
                    umma_f16(tmem + 256 + 128 * t, a + (uint64_t)((ks >> 2) * (PK_Q_BYTES >> 5) + (ks & 3) * 2),
                             b + (uint64_t)((ks >> 2) * (PK_KV_BYTES >> 5) + (ks & 3) * 2), idesc, ks > 0 ? 1u : 0u);
                umma_commit(s_full + 8 * t);
                if (t == 1) umma_commit(empty + 8 * s);
                if (t == 1 && last) umma_commit(q_empty);
            };
            const auto products = [&](int t, int i, int half, bool first) {   // O of tile t += P V of 64 keys
                const uint64_t v = vd + (uint64_t)(i % PK_STAGES * (PK_KV_BYTES >> 4) + half * (64 * 128 >> 4));
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    umma_f16_ts(tmem + 128 * t, tmem + 256 + 128 * t + 64 + 32 * half + 8 * ks, v + (uint64_t)(ks * (2048 >> 4)), idesc_o, first && ks == 0 ? 0u : 1u);
            };
            bool ok = true;
            int i = 0, used = 0, n_a = 0, n_b = 0, n_v = 0;   // tiles of the ring, blocks with keys, halves of P, cleaned tiles so far
            for (int k = 0;; ++k) {
                if (!wait(place_full + 8 * (k & 1), (uint32_t)(k >> 1) & 1u)) {
                    ok = false;
                    break;
                }
                const PackedBlock b = s_block[k & 1];
                mbar_arrive(place_empty + 8 * (k & 1));
                if (b.block < 0) break;
                const Shape sh = shape_of(b);
                if (sh.n_tiles == 0 || !ok) continue;
                const auto tile_wait = [&](int at) { return wait(full + 8 * (at % PK_STAGES), (uint32_t)(at / PK_STAGES) & 1u); };
                const auto keys_of = [&](int j) { return (uint32_t)(j == sh.n_tiles - 1 && sh.short_last ? PK_KEYS / 2 : PK_KEYS); };
                ok = *s_dead == 0 && wait(q_full, (uint32_t)used & 1u) && tile_wait(i);
                if (ok)
                    for (int t = 0; t < 2; ++t) scores(t, i, keys_of(0), sh.n_tiles == 1);
                for (int j = 0; j < sh.n_tiles && ok; ++j) {
                    const bool last = j == sh.n_tiles - 1, both = !last || !sh.short_last, clean = last && sh.ragged;
                    ok = *s_dead == 0 && tile_wait(i + 2 * j + 1);
                    if (ok && clean) mbar_arrive(v_last);
                    for (int t = 0; t < 2 && ok; ++t) {
                        if (j == 0 && used > 0) ok = wait(o_empty + 8 * t, (uint32_t)(used - 1) & 1u);   // the block before has left
                        if (ok && both) {
                            ok = wait(p_full + 16 * t + 8, (uint32_t)n_b & 1u);
                            if (ok && clean && t == 0) ok = wait(v_clean, (uint32_t)n_v & 1u);
                            if (!ok) break;
                            tc_fence_after();
                            products(t, i + 2 * j + 1, 1, j == 0);
                        }
                        if (ok) ok = wait(p_full + 16 * t, (uint32_t)n_a & 1u);
                        if (ok && clean && t == 0 && !both) ok = wait(v_clean, (uint32_t)n_v & 1u);
                        if (!ok) break;
                        tc_fence_after();
                        products(t, i + 2 * j + 1, 0, j == 0 && !both);
                        if (last) umma_commit(o_full + 8 * t);
                        if (t == 1) umma_commit(empty + 8 * ((i + 2 * j + 1) % PK_STAGES));
                        // the next scores: issued after, and so executed after, the products that read P there
                        if (!last) {
                            if (t == 0) ok = tile_wait(i + 2 * j + 2);
                            if (!ok) break;
                            scores(t, i + 2 * j + 2, keys_of(j + 1), j + 2 == sh.n_tiles);
                        }
                    }
                    ++n_a;
                    n_b += both;
                    n_v += clean;
                }
                if (!ok) give_up(0x30042);
                i += 2 * sh.n_tiles;
                ++used;
            }
            if (!ok) give_up(0x30042);
            if (!ok || *s_dead != 0) {   // the MMAs in flight
                umma_commit(drain);
                mbar_wait(drain, 0);
            }
        }
        __syncwarp();
    } else if (warp == 2) {
        int i = 0, n_v = 0;
        for (int k = 0;; ++k) {
            if (!__all_sync(0xffffffffu, wait(place_full + 8 * (k & 1), (uint32_t)(k >> 1) & 1u))) {
                if (lane == 0) give_up(0x30044);
                break;
            }
            const PackedBlock b = s_block[k & 1];
            __syncwarp();
            if (lane == 0) mbar_arrive(place_empty + 8 * (k & 1));
            if (b.block < 0) break;
            const Shape sh = shape_of(b);
            i += 2 * sh.n_tiles;
            if (!sh.ragged || *s_dead != 0) continue;
            const bool ok = __all_sync(0xffffffffu, wait(v_last, (uint32_t)n_v & 1u));   // the issuer has seen the tile land
            ++n_v;
            if (ok) {
                uint8_t* const tile = kv_s + (i - 1) % PK_STAGES * PK_KV_BYTES;
                const int from = sh.n_keys - (sh.n_tiles - 1) * PK_KEYS, n = (sh.short_last ? PK_KEYS / 2 : PK_KEYS) - from;
                for (int e = lane; e < n * 16; e += 32) {   // rows of 128 bytes in either half
                    const int h = e / (n * 8), in = e - h * n * 8;
                    *reinterpret_cast<uint4*>(tile + h * (PK_KV_BYTES / 2) + from * 128 + in * 16) = make_uint4(0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            } else if (lane == 0) {
                give_up(0x30044);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(v_clean);
        }
    } else if (warp >= 4) {
        const int t = (warp - 4) >> 2, q = warp & 3;
        const uint32_t lane_base = tmem + ((uint32_t)(32 * q) << 16);
        const uint32_t o_at = lane_base + 128 * t, s_at = lane_base + 256 + 128 * t, p_at = s_at + 64;
        const int row = 32 * q + lane, token = tile_tokens * t + row / pack;   // of the block
        const int warp_token = tile_tokens * t + 32 * q / pack;                // of the warp's first row
        const float c = p.c;
        bool ok = true;
        int used = 0, n_a = 0;   // blocks with keys, key tiles so far
        for (int k = 0;; ++k) {
            if (!__all_sync(0xffffffffu, wait(place_full + 8 * (k & 1), (uint32_t)(k >> 1) & 1u))) {
                if (lane == 0) give_up(0x30043);
                break;
            }
            const PackedBlock b = s_block[k & 1];
            __syncwarp();
            if (lane == 0) mbar_arrive(place_empty + 8 * (k & 1));
            if (b.block < 0) break;
            const Shape sh = shape_of(b);
            const int pos = min(sh.past + sh.t0 + token, sh.n_keys - 1);                // last key the row sees
            const int pos_first = min(sh.past + sh.t0 + warp_token, sh.n_keys - 1);
            const bool mine = sh.t0 + token < b.nq;
            T* const out = static_cast<T*>(p.a.d_out) + ((size_t)(b.q0 + sh.t0) * p.a.heads + b.head0) * 128;
            T* const dst = out + ((size_t)token * p.a.heads + row % pack) * 128;
            float m = -INFINITY, l = 0.0f;           // m: maximum in use (raw scores)
            float oh = -SHIFT, ol = 0.0f;            // P = 2^(s c - oh - ol)
            bool large = false;                      // m c has no fraction left in fp32: then oh = m c, ol its rounding error, and m is taken off s first
            float2 s[32];
            const auto load = [&](int half, int k0) {   // scores of 64 keys from k0 on
                tmem_ld32(s_at + 64 * half, reinterpret_cast<uint32_t*>(s));
                tmem_ld32(s_at + 64 * half + 32, reinterpret_cast<uint32_t*>(s) + 32);
                tmem_wait_ld();
                if (k0 + 63 > pos_first) {   // some row of the warp does not see all of them
#pragma unroll
                    for (int e = 0; e < 32; ++e) s[e] = make_float2(k0 + 2 * e <= pos ? s[e].x : -INFINITY, k0 + 2 * e + 1 <= pos ? s[e].y : -INFINITY);
                }
            };
            const auto largest = [&] {
                float mx[4] = {s[0].x, s[0].y, s[1].x, s[1].y};
#pragma unroll
                for (int e = 2; e < 32; ++e) mx[e & 3] = pk_max3(mx[e & 3], s[e].x, s[e].y);
                return max_nan(pk_max3(mx[0], mx[1], mx[2]), mx[3]);
            };
            const auto exponentials = [&](int half) {
                if (__any_sync(0xffffffffu, large)) {
                    const float base = large ? m : 0.0f;
#pragma unroll
                    for (int e = 0; e < 32; ++e) s[e] = make_float2(s[e].x - base, s[e].y - base);
                }
                const float off = large ? -SHIFT : oh;
                const float2 c2 = make_float2(c, c), off2 = make_float2(-off, -off);
                float2 ls[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float2 x = fma2(s[16 * h + e], c2, off2);
                        const float2 a = (e * PK_FMA) % 16 + PK_FMA >= 16 ? pk_ex2_fma(x) : make_float2(pk_ex2(x.x), pk_ex2(x.y));
                        ls[e & 1] = add2(ls[e & 1], a);
                        w[e] = R::pack(a.x, a.y);
                    }
                    tmem_st16(p_at + 32 * half + 16 * h, w);
                }
                l += (ls[0].x + ls[0].y) + (ls[1].x + ls[1].y);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 16 * t + 8 * half);
            };
            for (int j = 0; j < sh.n_tiles && ok; ++j) {
                const bool both = j < sh.n_tiles - 1 || !sh.short_last;
                const int k0 = j * PK_KEYS;
                // the scores, and with them the products of the tile before, which were issued earlier
                ok = __all_sync(0xffffffffu, *s_dead == 0 && wait(s_full + 8 * t, (uint32_t)(n_a + j) & 1u));
                if (!ok) break;
                tc_fence_after();
                load(0, k0);
                float mt = largest();
                if (both) {
                    load(1, k0 + 64);
                    mt = max_nan(mt, largest());
                }
                if (__any_sync(0xffffffffu, !((mt - m) * c <= LAG) || large)) {   // rare after the first tile; NaN goes this way too
                    const float mn = max_nan(m, mt), mc = mn == -INFINITY ? 0.0f : mn * c;
                    const bool nl = fabsf(mc) >= 1048576.0f;
                    const float nh = nl ? mc : mc - SHIFT, nlow = nl ? fmaf(mn, c, -mc) - SHIFT : 0.0f;
                    const float f = m == -INFINITY ? 0.0f : pk_ex2((oh - nh) + (ol - nlow));
                    if (j > 0) {
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            uint32_t o[32];
                            tmem_ld32(o_at + 32 * h, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st32(o_at + 32 * h, o);
                        }
                    }
                    l *= f;
                    m = mn;
                    oh = nh;
                    ol = nlow;
                    large = nl;
                }
                if (both) {
                    exponentials(1);
                    load(0, k0);
                }
                exponentials(0);
            }
            n_a += sh.n_tiles;
            if (sh.n_tiles > 0) {
                ok = __all_sync(0xffffffffu, ok && wait(o_full + 8 * t, (uint32_t)used & 1u));
                ++used;
                if (!ok && lane == 0) give_up(0x30043);
            }
            __syncwarp();
            tc_fence_after();
            const float r = pos < 0 ? 0.0f : 1.0f / l;   // a row that sees no key is zeros
            float finite = 0.0f;   // NaN as soon as an output is NaN or Inf
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                uint32_t o[32];
                __syncwarp();
                tmem_ld32(o_at + 32 * h, o);   // of a block without keys: not used
                tmem_wait_ld();
                if (h == 3 && sh.n_tiles > 0) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(o_empty + 8 * t);
                }
                if (mine) {
#pragma unroll
                    for (int e = 0; e < 32; e += 16) {
                        uint32_t w[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float x = __uint_as_float(o[e + 2 * i]) * r, y = __uint_as_float(o[e + 2 * i + 1]) * r;
                            finite = fmaf(x, 0.0f, fmaf(y, 0.0f, finite));
                            w[i] = !ok ? 0x7fff7fffu : pos < 0 ? 0u : R::pack(x, y);
                        }
                        // 32 bytes a lane: every lane writes a row of its own, and a store takes a cycle a row
                        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + 32 * h + e), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                                     "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
                    }
                }
            }
            __syncwarp();   // a row that is done again has been stored
            // a sum that is not finite is that of scores the row sees, and its result is NaN whatever is done
            uint32_t redo = ok ? __ballot_sync(0xffffffffu, mine && pos >= 0 && finite != 0.0f && l - l == 0.0f) : 0u;
            if (redo != 0) {
                const int kv_head = b.head0 / (p.a.heads / p.a.kv_heads);
                const T* const k_rows = static_cast<const T*>(p.a.d_k) + b.k0 * p.a.k_stride + kv_head * 128;
                const T* const v_rows = static_cast<const T*>(p.a.d_v) + b.k0 * p.a.v_stride + kv_head * 128;
                for (redo = packed_spoiled<T>(redo, pos, dst, v_rows, p.a.v_stride, lane); redo != 0; redo &= redo - 1) {
                    const int rr = 32 * q + __ffs(redo) - 1, tok = tile_tokens * t + rr / pack, head = b.head0 + rr % pack;
                    packed_row<T>(static_cast<const T*>(p.a.d_q) + (b.q0 + sh.t0 + tok) * p.a.q_stride + head * 128, k_rows, p.a.k_stride, v_rows, p.a.v_stride,
                                  sh.past + sh.t0 + tok + 1, c, out + ((size_t)tok * p.a.heads + rr % pack) * 128, lane);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <class T>
static int packed_launch(const Qw3AttnPackedArgs& a, const Workspace* ws, bool pdl, cudaStream_t st) {
    PackedParams p;
    p.a = a;
    p.c = (float)((a.scale == 0.0f ? 0.08838834764831845 : (double)a.scale) * 1.4426950408889634);
    const int group = a.heads / a.kv_heads;
    p.pack = group & -group;
    if (p.pack > 16) p.pack = 16;
    p.limit = (1ll << 31) + PK_REDO_TICKS * a.k_rows;
    p.ticket = ws->counters;
    p.done = ws->counters + 1;
    p.err = ws->err;
    CUtensorMap tm_q, tm_k, tm_v;
    const uint64_t qd[3] = {128, (uint64_t)a.heads, (uint64_t)a.q_rows}, qs[2] = {256, (uint64_t)a.q_stride * 2};
    const uint32_t qb[3] = {64, (uint32_t)p.pack, (uint32_t)(PK_ROWS / p.pack)}, kb[3] = {64, PK_KEYS, 1};
    int rc = encode_f16_map(&tm_q, a.d_q, 3, qd, qs, qb);
    if (rc != QW3_OK) return rc;
    if (a.k_rows > 0) {
        const uint64_t kd[3] = {128, (uint64_t)a.k_rows, (uint64_t)a.kv_heads}, ks[2] = {(uint64_t)a.k_stride * 2, 256}, vs[2] = {(uint64_t)a.v_stride * 2, 256};
        rc = encode_f16_map(&tm_k, a.d_k, 3, kd, ks, kb);
        if (rc == QW3_OK) rc = encode_f16_map(&tm_v, a.d_v, 3, kd, vs, kb);
        if (rc != QW3_OK) return rc;
    } else {
        tm_k = tm_v = tm_q;   // no sequence has a key: no copy is made
    }
    static std::atomic<bool> attr_set[64];   // per device: the kernel's shared-memory limit is raised once
    const int dev = ws->device;
    if (dev >= 64 || !attr_set[dev].load(std::memory_order_acquire)) {
        QW3_CUDA(cudaFuncSetAttribute(attn_packed_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PK_SMEM));
        if (dev < 64) attr_set[dev].store(true, std::memory_order_release);
    }
    // every sequence ends with one block that may not be full
    const int64_t block_tokens = 2 * PK_ROWS / p.pack, blocks = (a.q_rows / block_tokens + a.n_seq) * (a.heads / p.pack);
    QW3_REQUIRE(blocks <= 0x7fffffff - ws->sm_count, "qw3_attn_packed: too many rows");
    QW3_CUDA(kv4_launch(attn_packed_kernel<T>, dim3((unsigned)(blocks < ws->sm_count ? blocks : ws->sm_count)), dim3(PK_THREADS), PK_SMEM, st, pdl, 1, tm_q, tm_k, tm_v, p));
    return QW3_OK;
}

// Whether `out` shares bytes with one of `rows` rows of `width` bytes, `stride` bytes apart.
static bool rows_overlap(const void* out, int64_t out_bytes, const void* base, int64_t rows, int64_t width, int64_t stride) {
    if (rows <= 0) return false;   // nor is there a stride
    const int64_t lo = reinterpret_cast<intptr_t>(out) - reinterpret_cast<intptr_t>(base), hi = lo + out_bytes;   // beside the first row
    const int64_t row = lo < width ? 0 : (lo - width) / stride + 1;   // the first that ends behind lo
    return row < rows && row * stride < hi;
}

}  // namespace qw3

using namespace qw3;

extern "C" int qw3_attn_packed(const Qw3AttnPackedArgs* a, qw3_ws_t ws, void* stream) {
    const char* who = "qw3_attn_packed";
    QW3_REQUIRE(a && ws, "%s: null argument", who);
    QW3_REQUIRE(a->head_dim == 128, "%s: head_dim must be 128", who);
    QW3_REQUIRE(a->dtype == QW3_F16 || a->dtype == QW3_BF16, "%s: dtype must be QW3_F16 or QW3_BF16", who);
    QW3_REQUIRE(a->kv_heads > 0 && a->heads > 0 && a->heads <= 4096 && a->heads % a->kv_heads == 0, "%s: heads must be a multiple of kv_heads", who);
    QW3_REQUIRE(a->q_rows >= 0 && a->q_rows <= 0x7fffffff - 1024 && a->k_rows >= 0 && a->k_rows <= 0x7fffffff - 1024 && a->n_seq >= 0, "%s: rows or n_seq out of range", who);
    QW3_REQUIRE(a->scale >= 0.0f && a->scale <= KV4_MAX_SCALE, "%s: scale must be finite, 2e38 at most, and not below 0", who);
    if (a->q_rows == 0 || a->n_seq == 0) return QW3_OK;
    QW3_REQUIRE(a->d_q && a->d_out && a->d_cu_q && a->d_cu_k && (a->k_rows == 0 || (a->d_k && a->d_v)), "%s: null pointer", who);
    const auto stride_ok = [](int64_t s, int heads) { return s >= (int64_t)heads * 128 && s % 8 == 0 && s < ((int64_t)1 << 31); };
    QW3_REQUIRE(stride_ok(a->q_stride, a->heads) && (a->k_rows == 0 || (stride_ok(a->k_stride, a->kv_heads) && stride_ok(a->v_stride, a->kv_heads))),
                "%s: strides must be multiples of 8 and hold the heads", who);
    QW3_REQUIRE(((reinterpret_cast<uintptr_t>(a->d_q) | reinterpret_cast<uintptr_t>(a->d_out) | reinterpret_cast<uintptr_t>(a->d_k) | reinterpret_cast<uintptr_t>(a->d_v)) & 15) == 0,
                "%s: rows must be 16-byte aligned", who);
    QW3_REQUIRE((reinterpret_cast<uintptr_t>(a->d_out) & 31) == 0, "%s: out must be 32-byte aligned", who);
    // blocks run in any order, and rows that are done again read q, k and v after rows have been stored
    const int64_t out_bytes = a->q_rows * a->heads * 256;
    QW3_REQUIRE(!rows_overlap(a->d_out, out_bytes, a->d_q, a->q_rows, a->heads * 256ll, a->q_stride * 2) &&
                    !rows_overlap(a->d_out, out_bytes, a->d_k, a->k_rows, a->kv_heads * 256ll, a->k_stride * 2) &&
                    !rows_overlap(a->d_out, out_bytes, a->d_v, a->k_rows, a->kv_heads * 256ll, a->v_stride * 2),
                "%s: out must not overlap q, k or v", who);
    const int rc = ws_on_device(who, ws);
    if (rc != QW3_OK) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->dtype == QW3_F16 ? packed_launch<__half>(*a, ws_struct(ws), ws_pdl(ws), st) : packed_launch<__nv_bfloat16>(*a, ws_struct(ws), ws_pdl(ws), st);
}
