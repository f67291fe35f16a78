// Paged 4-bit KV cache: pages handed out to requests that grow, rows rotated, quantised and stored, rows read back.
#include <cooperative_groups.h>

#include <type_traits>

#include "kv4.cuh"

namespace qw3 {

// ---- block tables and slots ------------------------------------------------------------------------------------------------------
// One cluster.  Every CTA sums the lengths of all requests for itself (two prefix sums, of new tokens and of new pages, kept in shared
// memory) and checks its share of the pages that will get tokens, the cluster meets, so that outputs may be the inputs' own buffers and a call that
// cannot be served changes nothing, and then its threads fill the lists: a thread takes
// four tokens in a row and finds their request by bisection.  Bound by latency, two dependent rounds of global loads: 10.4 us
// for 7 requests, 14.4 for 250 with 34 K new tokens (launch included, caches cold).
constexpr int PS_THREADS = 512;
constexpr int PS_CLUSTER = 8;   // one CTA instead: the same up to 2500 new tokens of 8 requests (10.2 us), 16.4 instead of 10.2 for 8000, 41 instead of 14.3 for 34000
constexpr int PS_MAX_REQ = 16384;

__global__ void __launch_bounds__(PS_THREADS) page_slots_kernel(const Qw3PageArgs p, int* err) {
    extern __shared__ int ps_smem[];
    __shared__ long long warp_sum[2][PS_THREADS / 32];
    __shared__ int ps_bad;
    const int n = p.n_req, P = p.page_size;
    int* const cu = ps_smem;            // [n + 1] tokens before a request
    int* const off = cu + n + 1;        // [n + 1] pages before a request
    int* const ctx = off + n + 1;       // [n]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = blockIdx.x * PS_THREADS + tid, step = gridDim.x * PS_THREADS;
    const auto cluster = cooperative_groups::this_cluster();
    if (tid == 0) ps_bad = 0;
    pdl_launch_dependents();
    cluster.barrier_arrive();
    pdl_wait();

    const int n_free = *p.d_n_free;
    // the pages that will get tokens are looked at in shares of the CTAs: those to be taken, the first of a thread while the lengths come, and the last
    // ones of requests that go on in them
    const int most_pages = 0x7fffffff / P;
    const int ahead = n_free <= p.free_capacity && first < n_free ? p.d_free[n_free - 1 - first] : 0;
    bool bad_page = false;
    const int each = (n + PS_THREADS - 1) / PS_THREADS, b0 = min(tid * each, n), b1 = min(b0 + each, n);
    long long tokens = 0, pages = 0;
    int bad = 0;
    for (int b = b0; b < b1; ++b) {
        const int c = p.d_ctx_len[b], x = p.d_new_len[b];
        ctx[b] = c;
        if (c < 0 || x < 0) {
            bad = max(bad, 1);
        } else {
            const long long need = ((long long)c + x + P - 1) / P;
            if (need > p.max_blocks) bad = max(bad, 2);
            pages += need - ((long long)c + P - 1) / P;
            tokens += x;
            if (b % PS_CLUSTER == (int)blockIdx.x && x > 0 && c % P != 0 && need <= p.max_blocks) {
                const int page = p.d_block_table[b * p.table_stride + c / P];
                bad_page |= page < 0 || page >= most_pages;
            }
        }
    }
    long long t = tokens, g = pages;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const long long a = __shfl_up_sync(0xffffffffu, t, d), b = __shfl_up_sync(0xffffffffu, g, d);
        if (lane >= d) { t += a; g += b; }
    }
    if (lane == 31) { warp_sum[0][warp] = t; warp_sum[1][warp] = g; }
    const int any1 = __syncthreads_or(bad == 1), any2 = __syncthreads_or(bad == 2);
    long long total = 0, total_pages = 0;
    for (int w = 0; w < PS_THREADS / 32; ++w) {
        if (w == warp) { t += total; g += total_pages; }
        total += warp_sum[0][w];
        total_pages += warp_sum[1][w];
    }
    int code = 0;
    if (any1) code = KV4_ERR_LENGTH;
    else if (any2) code = KV4_ERR_TABLE;
    else if (n_free < 0 || n_free > p.free_capacity || total_pages > n_free) code = KV4_ERR_PAGES;
    else if (total > p.max_tokens) code = KV4_ERR_TOKENS;
    // below, sums fit 32 bits (max_tokens and n_free do)
    if (code == 0) {
        t -= tokens;
        g -= pages;
        for (int b = b0; b < b1; ++b) {
            const int c = ctx[b], x = p.d_new_len[b];
            cu[b] = (int)t;
            off[b] = (int)g;
            t += x;
            g += (c + x + P - 1) / P - (c + P - 1) / P;
        }
    }
    if (tid == 0) { cu[n] = (int)total; off[n] = (int)total_pages; }
    cluster.barrier_wait();   // the others' words are set up
    if (code == 0) {
        for (int i = first; i < (int)total_pages; i += step) {
            const int page = i == first ? ahead : p.d_free[n_free - 1 - i];
            bad_page |= page < 0 || page >= most_pages;
        }
        if (bad_page)
            for (int r = 0; r < PS_CLUSTER; ++r) *cluster.map_shared_rank(&ps_bad, r) = 1;
    }
    // all CTAs have read the lengths, the number of free pages and their share of the pages
    cluster.sync();
    if (code == 0 && *static_cast<volatile int*>(&ps_bad) != 0) code = KV4_ERR_FREE_ID;

    const auto find = [n](const int* starts, int i) {   // the last request that starts at or before i
        int lo = 0, hi = n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (starts[mid] <= i) lo = mid;
            else hi = mid;
        }
        return lo;
    };
    if (code != 0) {
        if (first == 0) {
            kv4_error(err, code);
            *p.d_n_free_out = n_free;
        }
        for (int b = first; b <= n; b += step) {
            p.d_cu[b] = 0;
            if (b < n) p.d_kv_len[b] = ctx[b];
        }
        for (int i = first; i < p.max_tokens; i += step) { p.d_pos[i] = 0; p.d_slot[i] = -1; }
        return;
    }
    if (first == 0) *p.d_n_free_out = n_free - (int)total_pages;
    for (int b = first; b <= n; b += step) {
        p.d_cu[b] = cu[b];
        if (b < n) p.d_kv_len[b] = ctx[b] + cu[b + 1] - cu[b];
    }
    for (int i = first; i < (int)total_pages; i += step) {
        const int b = find(off, i);
        p.d_block_table[b * p.table_stride + (ctx[b] + P - 1) / P + i - off[b]] = p.d_free[n_free - 1 - i];
    }
    for (int i4 = first * 4; i4 < p.max_tokens; i4 += step * 4) {
        int b = i4 < (int)total ? find(cu, i4) : n - 1;
        for (int i = i4; i < min(i4 + 4, p.max_tokens); ++i) {
            int pos = 0, slot = -1;
            if (i < (int)total) {
                while (cu[b + 1] <= i) ++b;
                const int c = ctx[b];
                pos = c + i - cu[b];
                const int block = pos / P, fresh = block - (c + P - 1) / P;
                const int page = fresh >= 0 ? p.d_free[n_free - 1 - (off[b] + fresh)] : p.d_block_table[b * p.table_stride + block];
                slot = page * P + pos % P;
            }
            p.d_pos[i] = pos;
            p.d_slot[i] = slot;
        }
    }
}

// ---- rotation, quantisation, store -----------------------------------------------------------------------------------------------
// A CTA takes the rows of one token, a slice of 96 at most (slices of 16 for few tokens: the same up to 33 tokens, 12.4 instead of
// 10.2 us for 280 tokens of 32 / 32 heads); bulk copies bring them, while slot,
// position and the cosines and sines, which the lanes keep for all heads, are looked up.  A warp takes two rows at a time, eight dims a
// lane.  Products and sums of the rotation are rounded one by one (no contraction), so that a row's codes do not depend on the compiler.  K
// is quantised from the fp32 rotated row, not from its rounding.  Bound by issue slots: 4001 tokens, 32 KV
// heads, bf16, 181 MB: 43 us, 4.2 TB/s.
constexpr int AP_THREADS = 256, AP_WARPS = AP_THREADS / 32, AP_MAX_ROWS = 96;

// Over the lanes of either half-warp.  Two reductions over the whole warp: one with a mask a half would be run half after half.
template <bool MAX>
__device__ __forceinline__ float reduce_half(float a, bool upper) {
    const float none = MAX ? -INFINITY : INFINITY;
    float lo, hi;
    if (MAX) {
        asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(lo) : "f"(upper ? none : a));
        asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(hi) : "f"(upper ? a : none));
    } else {
        asm volatile("redux.sync.min.NaN.f32 %0, %1, 0xffffffff;" : "=f"(lo) : "f"(upper ? none : a));
        asm volatile("redux.sync.min.NaN.f32 %0, %1, 0xffffffff;" : "=f"(hi) : "f"(upper ? a : none));
    }
    return upper ? hi : lo;
}
// a / b rounded to nearest, for normal b and inv = 1 / b rounded to nearest: one correction by the remainder, which is exact (P. Markstein,
// Computation of elementary functions on the IBM RISC System/6000, 1990).  Where a is so small that it underflows, the caller's result is 0.
__device__ __forceinline__ float2 quotient(float2 a, float b, float inv) {
    const float2 i = make_float2(inv, inv), q = mul2(a, i);
    return fma2(fma2(make_float2(-q.x, -q.y), make_float2(b, b), a), i, q);
}

template <class T, bool PAIRS>
__global__ void __launch_bounds__(AP_THREADS, 4)
rope_kv4_append_kernel(const Qw3Kv4Pool pool, const Qw3Kv4AppendArgs p, int* err) {
    using R = RowType<T>;
    extern __shared__ __align__(128) uint4 ap_rows[];
    __shared__ uint64_t bar;
    const int tid = threadIdx.x, l = tid & 15, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const bool second = (tid & 16) != 0;   // row of the warp's two
    const int token = blockIdx.x, kv = pool.kv_heads, P = pool.page_size, rot = p.rot_dim;
    // this CTA's slice: rows q0 .. q1 of q, k0 .. k1 of k and of v
    const int q0 = p.heads * (int)blockIdx.y / (int)gridDim.y, q1 = p.heads * (int)(blockIdx.y + 1) / (int)gridDim.y;
    const int k0 = kv * (int)blockIdx.y / (int)gridDim.y, k1 = kv * (int)(blockIdx.y + 1) / (int)gridDim.y;
    const int nq = q1 - q0, nk = k1 - k0;
    pdl_launch_dependents();
    if (tid == 0) {
        mbar_init(smem_u32(&bar), 1);
        mbar_fence_init();
    }
    pdl_wait();
    if (tid == 0) {
        const T* const row = static_cast<const T*>(p.d_qkv) + (size_t)token * p.qkv_stride;
        const uint32_t b = smem_u32(&bar), to = smem_u32(ap_rows);
        mbar_expect_tx(b, (uint32_t)(nq + 2 * nk) * 256);
        if (nq > 0) bulk_load(to, row + (size_t)q0 * 128, (uint32_t)nq * 256, b);
        if (nk > 0) bulk_load(to + (uint32_t)nq * 256, row + (size_t)(p.heads + k0) * 128, (uint32_t)nk * 256, b);
        if (nk > 0) bulk_load(to + (uint32_t)(nq + nk) * 256, row + (size_t)(p.heads + kv + k0) * 128, (uint32_t)nk * 256, b);
    }
    const int slot = p.d_slot[token];
    const int pos = rot > 0 ? p.d_pos[token] : 0;
    const bool known = rot == 0 || (pos >= 0 && pos < p.max_pos);
    if (!known && tid == 0) kv4_error(err, KV4_ERR_APPEND_POS);
    const int page = slot >= 0 ? slot / P : -1, in_page = slot - page * P;
    if (page >= pool.n_pages && tid == 0) kv4_error(err, KV4_ERR_APPEND_SLOT);
    const bool store = page >= 0 && page < pool.n_pages;
    uint8_t* const tile0 = static_cast<uint8_t*>(pool.d_pages) + (store ? page * pool.page_stride + (in_page >> 4) * KV4_TILE_BYTES : 0);
    const int r_in = in_page & 15;

    float2 cs[4], sn[4];   // pairs: (c, c) and (-s, s) of a pair; halves: of two dims, the sines with the sign that they enter with
    const bool turns = known && 8 * l < rot;
    // halves: lane l holds dims 8l .. 8l+7 of one half, lane `mate` their partners; pairs: four pairs in the lane
    const bool upper = !PAIRS && 16 * l >= rot;
    const int mate = PAIRS ? l : upper ? l - rot / 16 : l + rot / 16;
    if (turns) {
        const size_t at = (size_t)pos * (rot / 2) + (PAIRS ? 4 * l : 8 * (upper ? mate : l));
#pragma unroll
        for (int e = 0; e < (PAIRS ? 4 : 8); e += 4) {
            const float4 c = *reinterpret_cast<const float4*>(p.d_cos + at + e), s = *reinterpret_cast<const float4*>(p.d_sin + at + e);
            if (PAIRS) {
                cs[0] = make_float2(c.x, c.x); cs[1] = make_float2(c.y, c.y); cs[2] = make_float2(c.z, c.z); cs[3] = make_float2(c.w, c.w);
                sn[0] = make_float2(-s.x, s.x); sn[1] = make_float2(-s.y, s.y); sn[2] = make_float2(-s.z, s.z); sn[3] = make_float2(-s.w, s.w);
            } else {
                const float sign = upper ? 1.0f : -1.0f;
                cs[e / 2] = make_float2(c.x, c.y); cs[e / 2 + 1] = make_float2(c.z, c.w);
                sn[e / 2] = make_float2(sign * s.x, sign * s.y); sn[e / 2 + 1] = make_float2(sign * s.z, sign * s.w);
            }
        }
    }
    __syncthreads();
    if (!mbar_wait(smem_u32(&bar), 0)) {
        if (tid == 0) atomicCAS(err, 0, 0x30051);
        mbar_wait(smem_u32(&bar), 0);   // the copy in flight
        return;
    }
    if (!known) return;
    // rows j0 .. of a part (0: q, 1: k, 2: v), `n` of them, which begin at row `at` of the shared memory
    const auto run = [&](auto which, int j0, int n, int at) {
        constexpr int PART = decltype(which)::value;
        for (int i0 = 2 * warp; i0 < n; i0 += 2 * AP_WARPS) {
            const int i = i0 + second, j = j0 + i;
            const bool there = i < n;   // the shuffles need every lane
            const uint4 w = ap_rows[(at + (there ? i : i0)) * 16 + l];
            float2 x[4] = {R::unpack(w.x), R::unpack(w.y), R::unpack(w.z), R::unpack(w.w)};
            if (PART < 2 && rot > 0) {
                float2 y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    y[e] = PAIRS ? make_float2(x[e].y, x[e].x) : make_float2(__shfl_sync(0xffffffffu, x[e].x, mate, 16), __shfl_sync(0xffffffffu, x[e].y, mate, 16));
                if (turns) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)   // scalar products: a packed one would be contracted into the sum
                        x[e] = add2(make_float2(__fmul_rn(x[e].x, cs[e].x), __fmul_rn(x[e].y, cs[e].y)), make_float2(__fmul_rn(y[e].x, sn[e].x), __fmul_rn(y[e].y, sn[e].y)));
                }
            }
            if (PART < 2) {
                T* const to = static_cast<T*>(PART == 0 ? p.d_q_out : p.d_k_out);
                if (there && (PART == 0 || to != nullptr))
                    *reinterpret_cast<uint4*>(to + ((size_t)token * (PART == 0 ? p.heads : kv) + j) * 128 + 8 * l) =
                        make_uint4(R::pack(x[0].x, x[0].y), R::pack(x[1].x, x[1].y), R::pack(x[2].x, x[2].y), R::pack(x[3].x, x[3].y));
            }
            if (PART > 0) {
                float lo = min_nan(x[0].x, x[0].y), hi = max_nan(x[0].x, x[0].y);
#pragma unroll
                for (int e = 1; e < 4; ++e) {
                    lo = min_nan(lo, min_nan(x[e].x, x[e].y));
                    hi = max_nan(hi, max_nan(x[e].x, x[e].y));
                }
                lo = reduce_half<false>(lo, second);
                hi = reduce_half<true>(hi, second);
                // minimum and scale as they are stored: the codes are those of the rounded pair
                const uint32_t m_bits = R::pack(lo, lo) & 0xffffu;
                const float m = R::unpack(m_bits).x, range = __fsub_rn(hi, m);
                float s = R::unpack(R::pack(quotient(make_float2(range, range), 15.0f, 1.0f / 15.0f).x, 0.0f)).x;
                const bool whole = s <= R::CEIL;   // not with Inf or NaN in the row
                s = fminf(fmaxf(s, R::FLOOR), R::CEIL);
                const float inv = __frcp_rn(s);
                // 1.5 * 2^23 + quotient rounds the quotient to the nearest whole number, ties to even (that they are found is why the quotient
                // is rounded correctly), and has it in its last bits
                constexpr float MAGIC = 12582912.0f;
                uint32_t codes = 0;
#pragma unroll
                for (int e = 3; e >= 0; --e) {
                    const float2 c = add2(quotient(add2(x[e], make_float2(-m, -m)), s, inv), make_float2(MAGIC, MAGIC));
                    codes = codes * 16u + __float_as_uint(fminf(fmaxf(c.y, MAGIC), MAGIC + 15.0f));
                    codes = codes * 16u + __float_as_uint(fminf(fmaxf(c.x, MAGIC), MAGIC + 15.0f));
                }
                codes -= 0x4b400000u * 0x11111111u;   // eight times the bits of MAGIC
                if (there && store) {   // a row with Inf or NaN reads back as NaN
                    uint8_t* const tile = tile0 + (size_t)j * (P / 16) * KV4_TILE_BYTES;
                    const uint32_t pair = (R::pack(s, 0.0f) & 0xffffu) | (m_bits << 16);
                    *reinterpret_cast<uint32_t*>(tile + (PART == 1 ? 0 : KV4_V) + r_in * 64 + 4 * l) = whole ? codes : 0u;
                    if (l == 0) *reinterpret_cast<uint32_t*>(tile + (PART == 1 ? KV4_KP : KV4_VP) + r_in * 4) = whole ? pair : (R::pack(1.0f, 0.0f) & 0xffffu) | 0x7fff0000u;
                }
            }
        }
    };
    run(std::integral_constant<int, 0>(), q0, nq, 0);
    run(std::integral_constant<int, 1>(), k0, nk, nq);
    run(std::integral_constant<int, 2>(), k0, nk, nq + nk);
}

// ---- rows read back --------------------------------------------------------------------------------------------------------------
// A half-warp takes four rows at a time: four bytes of codes in, sixteen out, a lane, of K and of V.  A slot below zero gives zeros.  30011
// tokens of 8 KV heads, 156 MB: 30 us, 5.2 TB/s, 0.81 of the measured copy rate (before several rows were loaded
// at once: 43 us).
constexpr int RD_THREADS = 256, RD_GROUPS = RD_THREADS / 16, RD_ROWS = 4;

template <class T>
__global__ void __launch_bounds__(RD_THREADS)
kv4_read_kernel(const Qw3Kv4Pool pool, const int32_t* __restrict__ d_slot, uint32_t rows, T* __restrict__ k_out, T* __restrict__ v_out, int* err) {
    using R = RowType<T>;
    pdl_launch_dependents();
    pdl_wait();
    const int l = threadIdx.x & 15;
    const uint32_t kv = pool.kv_heads, P = pool.page_size, first = blockIdx.x * (RD_GROUPS * RD_ROWS) + (threadIdx.x >> 4);
    uint32_t codes[RD_ROWS][2], pair[RD_ROWS][2];
#pragma unroll
    for (int u = 0; u < RD_ROWS; ++u) {
        const uint32_t i = first + RD_GROUPS * u, token = i / kv, head = i - token * kv;
        const int slot = i < rows ? d_slot[token] : -1;
        const uint32_t page = (uint32_t)slot / P, in_page = (uint32_t)slot - page * P;
        const bool there = slot >= 0 && page < pool.n_pages;
        if (slot >= 0 && !there && l == 0) kv4_error(err, KV4_ERR_READ_SLOT);
        codes[u][0] = codes[u][1] = pair[u][0] = pair[u][1] = 0;
        if (there) {
            const uint8_t* const tile = static_cast<const uint8_t*>(pool.d_pages) + page * pool.page_stride + ((int64_t)head * (P / 16) + (in_page >> 4)) * KV4_TILE_BYTES;
            const uint32_t r = in_page & 15;
            codes[u][0] = *reinterpret_cast<const uint32_t*>(tile + r * 64 + 4 * l);
            codes[u][1] = *reinterpret_cast<const uint32_t*>(tile + KV4_V + r * 64 + 4 * l);
            pair[u][0] = *reinterpret_cast<const uint32_t*>(tile + KV4_KP + r * 4);
            pair[u][1] = *reinterpret_cast<const uint32_t*>(tile + KV4_VP + r * 4);
        }
    }
#pragma unroll
    for (int u = 0; u < RD_ROWS; ++u) {
        const uint32_t i = first + RD_GROUPS * u;
        if (i >= rows) break;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const float2 sm = R::unpack(pair[u][v]);
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)   // code * scale is exact in fp32
                w[e] = R::pack(fmaf((float)(codes[u][v] >> (8 * e) & 15u), sm.x, sm.y), fmaf((float)(codes[u][v] >> (8 * e + 4) & 15u), sm.x, sm.y));
            *reinterpret_cast<uint4*>((v ? v_out : k_out) + (size_t)i * 128 + 8 * l) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// ---- checks ----------------------------------------------------------------------------------------------------------------------
int ws_on_device(const char* who, qw3_ws_t ws) {
    QW3_REQUIRE(ws, "%s: null workspace", who);
    int dev = -1;
    QW3_CUDA(cudaGetDevice(&dev));
    QW3_REQUIRE(dev == ws_struct(ws)->device, "%s: the workspace belongs to device %d, the current device is %d", who, ws_struct(ws)->device, dev);
    return QW3_OK;
}

int kv4_check(const char* who, const Qw3Kv4Pool* pool, qw3_ws_t ws) {
    QW3_REQUIRE(pool && pool->d_pages && ws, "%s: null pool, pages or workspace", who);
    QW3_REQUIRE(pool->head_dim == 128, "%s: head_dim must be 128", who);
    QW3_REQUIRE(pool->dtype == QW3_F16 || pool->dtype == QW3_BF16, "%s: dtype must be QW3_F16 or QW3_BF16", who);
    QW3_REQUIRE(pool->page_size >= 16 && pool->page_size <= 1024 && pool->page_size % 16 == 0, "%s: page_size must be a multiple of 16, 16 to 1024", who);
    QW3_REQUIRE(pool->kv_heads > 0 && pool->kv_heads <= 1024, "%s: kv_heads out of range", who);
    QW3_REQUIRE(pool->n_pages > 0 && pool->n_pages <= 0x7fffffff / pool->page_size, "%s: n_pages out of range (slots have 31 bits)", who);
    QW3_REQUIRE(pool->page_stride >= (int64_t)pool->kv_heads * pool->page_size * 136 && pool->page_stride % 16 == 0 && pool->page_stride < ((int64_t)1 << 40),
                "%s: page_stride must be a multiple of 16 and hold kv_heads * page_size * 136 bytes", who);
    QW3_REQUIRE((reinterpret_cast<uintptr_t>(pool->d_pages) & 15) == 0, "%s: pages must be 16-byte aligned", who);
    return ws_on_device(who, ws);
}

static bool aligned16(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) == 0; }

}  // namespace qw3

using namespace qw3;

extern "C" {

int qw3_page_slots(const Qw3PageArgs* a, qw3_ws_t ws, void* stream) {
    const char* who = "qw3_page_slots";
    QW3_REQUIRE(a && ws, "%s: null argument", who);
    QW3_REQUIRE(a->d_ctx_len && a->d_new_len && a->d_block_table && (a->d_free || a->free_capacity == 0) && a->d_n_free && a->d_n_free_out && a->d_cu && a->d_kv_len, "%s: null pointer", who);
    QW3_REQUIRE(a->max_tokens >= 0 && (a->max_tokens == 0 || (a->d_pos && a->d_slot)), "%s: null pointer or max_tokens out of range", who);
    QW3_REQUIRE(a->max_tokens <= 0x7fffffff - 65536, "%s: max_tokens out of range", who);
    QW3_REQUIRE(a->n_req > 0 && a->n_req <= PS_MAX_REQ, "%s: n_req must be 1 to %d", who, PS_MAX_REQ);
    QW3_REQUIRE(a->page_size >= 16 && a->page_size <= 1024 && a->page_size % 16 == 0, "%s: page_size must be a multiple of 16, 16 to 1024", who);
    QW3_REQUIRE(a->max_blocks > 0 && a->max_blocks <= (0x7fffffff - 1024) / a->page_size && a->table_stride >= a->max_blocks, "%s: block table out of range", who);
    QW3_REQUIRE(a->free_capacity >= 0, "%s: free_capacity out of range", who);
    int rc = ws_on_device(who, ws);
    if (rc != QW3_OK) return rc;
    const size_t smem = (size_t)(3 * a->n_req + 2) * 4;
    if (smem > 48 * 1024) QW3_CUDA(cudaFuncSetAttribute(page_slots_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (3 * PS_MAX_REQ + 2) * 4));
    QW3_CUDA(kv4_launch(page_slots_kernel, dim3(PS_CLUSTER), dim3(PS_THREADS), smem, static_cast<cudaStream_t>(stream), ws_pdl(ws), PS_CLUSTER, *a, ws_struct(ws)->err));
    return QW3_OK;
}

int qw3_rope_kv4_append(const Qw3Kv4Pool* pool, const Qw3Kv4AppendArgs* a, qw3_ws_t ws, void* stream) {
    const char* who = "qw3_rope_kv4_append";
    QW3_REQUIRE(a, "%s: null argument", who);
    int rc = kv4_check(who, pool, ws);
    if (rc != QW3_OK) return rc;
    QW3_REQUIRE(a->tokens >= 0 && a->tokens <= 0x7fffffff, "%s: tokens out of range", who);
    QW3_REQUIRE(a->heads > 0 && a->heads <= 4096, "%s: heads out of range", who);
    QW3_REQUIRE(a->rot_dim >= 0 && a->rot_dim <= 128 && a->rot_dim % 16 == 0, "%s: rot_dim must be a multiple of 16, 0 to 128", who);
    QW3_REQUIRE(a->layout == QW3_ROPE_HALVES || a->layout == QW3_ROPE_PAIRS, "%s: unknown layout", who);
    QW3_REQUIRE(a->reserved == 0, "%s: reserved must be 0", who);
    if (a->tokens == 0) return QW3_OK;
    QW3_REQUIRE(a->d_qkv && a->d_q_out && a->d_slot, "%s: null pointer", who);
    QW3_REQUIRE(a->rot_dim == 0 || (a->d_pos && a->d_cos && a->d_sin && a->max_pos > 0), "%s: positions and tables are needed to rotate", who);
    QW3_REQUIRE(a->qkv_stride >= (int64_t)(a->heads + 2 * pool->kv_heads) * 128 && a->qkv_stride % 8 == 0 && a->qkv_stride < ((int64_t)1 << 31),
                "%s: qkv_stride must be a multiple of 8 and hold heads + 2 kv_heads rows", who);
    QW3_REQUIRE(aligned16(a->d_qkv) && aligned16(a->d_q_out) && aligned16(a->d_k_out) && aligned16(a->d_cos) && aligned16(a->d_sin),
                "%s: rows and tables must be 16-byte aligned", who);
    const auto kernel = pool->dtype == QW3_F16 ? (a->layout == QW3_ROPE_PAIRS ? rope_kv4_append_kernel<__half, true> : rope_kv4_append_kernel<__half, false>)
                                               : (a->layout == QW3_ROPE_PAIRS ? rope_kv4_append_kernel<__nv_bfloat16, true> : rope_kv4_append_kernel<__nv_bfloat16, false>);
    const int rows = a->heads + 2 * pool->kv_heads, slices = (rows + AP_MAX_ROWS - 1) / AP_MAX_ROWS;
    const size_t smem = 256 * ((size_t)(a->heads + slices - 1) / slices + 2 * ((size_t)(pool->kv_heads + slices - 1) / slices));
    QW3_CUDA(kv4_launch(kernel, dim3((unsigned)a->tokens, slices), dim3(AP_THREADS), smem, static_cast<cudaStream_t>(stream), ws_pdl(ws), 1, *pool, *a, ws_struct(ws)->err));
    return QW3_OK;
}

int qw3_kv4_read(const Qw3Kv4Pool* pool, const int32_t* d_slot, int64_t tokens, void* d_k_out, void* d_v_out, qw3_ws_t ws, void* stream) {
    const char* who = "qw3_kv4_read";
    int rc = kv4_check(who, pool, ws);
    if (rc != QW3_OK) return rc;
    QW3_REQUIRE(tokens >= 0 && tokens <= 0x7fffffff, "%s: tokens out of range", who);
    if (tokens == 0) return QW3_OK;
    QW3_REQUIRE(d_slot && d_k_out && d_v_out, "%s: null pointer", who);
    QW3_REQUIRE(aligned16(d_k_out) && aligned16(d_v_out), "%s: rows must be 16-byte aligned", who);
    const int64_t rows = tokens * pool->kv_heads;   // 512 bytes of output each
    QW3_REQUIRE(rows <= 0x7fffffff - RD_GROUPS * RD_ROWS, "%s: too many rows", who);
    const dim3 grid((unsigned)((rows + RD_GROUPS * RD_ROWS - 1) / (RD_GROUPS * RD_ROWS)));
    if (pool->dtype == QW3_F16)
        QW3_CUDA(kv4_launch(kv4_read_kernel<__half>, grid, dim3(RD_THREADS), 0, static_cast<cudaStream_t>(stream), ws_pdl(ws), 1, *pool, d_slot, (uint32_t)rows,
                        static_cast<__half*>(d_k_out), static_cast<__half*>(d_v_out), ws_struct(ws)->err));
    else
        QW3_CUDA(kv4_launch(kv4_read_kernel<__nv_bfloat16>, grid, dim3(RD_THREADS), 0, static_cast<cudaStream_t>(stream), ws_pdl(ws), 1, *pool, d_slot, (uint32_t)rows,
                        static_cast<__nv_bfloat16*>(d_k_out), static_cast<__nv_bfloat16*>(d_v_out), ws_struct(ws)->err));
    return QW3_OK;
}

}  // extern "C"
