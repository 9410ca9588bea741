// Attention of single tokens over pages of 8-bit keys and values (kv8.cuh), bfloat16 queries, head size 128: one stream per
// SM. A load warp keeps a ring of TMA boxes in flight, eight warps work through what has landed with mma.sync.
//
// A row group is a request, a key/value head and up to eight of the query heads that share it. Its keys are cut into units of
// 32 keys aligned to key 0 (8 KB: keys and values). The units of all row groups of the launch form one list, request by request,
// and block b of B takes an equal share of its places (a group has S8_GROUP_COST places more than units, for what a block spends
// on a group besides reading). The n-th unit of a block goes to warp n mod 8.
//
// The products have the keys as their rows, so that no row of a tensor-core tile is padding (a group has at most eight heads, and
// eight is the number of columns): for 16 keys,
//   S^T [16 keys x 8 heads] = K [16 x 128] q^T [128 x 8],      O^T [128 x 8 heads] += V^T [128 x 16] P^T [16 x 8]
// in half precision, which holds every e4m3 value exactly. A lane reads its keys and values 16 bytes at a time. The order of the
// head's entries in the sum of S is free: step s of K takes bytes 4 s .. 4 s + 3 of a lane's 16, and q is laid out to match. Row g of
// a tile is key (g >> 1) + 4 (g & 1), with which eight lanes that read together meet every bank once in TMA's 128-byte swizzle; V's
// lanes read two keys that lie four apart, odd ones in the other order, and a byte permutation makes the pairs of keys that the
// product wants. The queries are brought to a largest magnitude in [1, 4) by a power of two per row (half precision then loses
// only what is below 2^-25 of it).
//
// With t = log2(e) scale q.k and a value's scale 2^v, weights are 2^t and a value's factor is 2^(t + v). Each has its own running
// maximum (m for t, mu for t + v): the sum l of the weights and the factors in half precision (at most 2^8: a maximum is only raised
// when it is passed by 8) both keep their bits whatever the scales of the blocks are. out = O / l * 2^(mu - m).
//
// At the end of a segment (what a block has of a group) the warps' sums are added in shared memory. A whole group is written out;
// of a shared one every block leaves its sums in global memory and counts itself, and the block that counts last adds them in block
// order, writes, and sets the counter back to zero. Nobody waits for anybody. Every wait on an mbarrier is bounded: when one runs
// out the kernel records 1 in *error_flag and goes on without waiting (its output is then wrong; the host reads the flag).
#include "kv8.cuh"
#include "tcgen05.cuh"

#define S8_D 128
#define S8_WARPS 8
#define S8_KEYS 32
#define S8_STAGE_BYTES (2 * S8_KEYS * S8_D)
#define S8_STAGES 20
#define S8_THREADS ((S8_WARPS + 1) * 32)
#define S8_HEADS 8
#define S8_OSTRIDE (S8_D + 4)                        // floats of a row of a warp's sums in shared memory
#define S8_MAX_ROWS 512
#define S8_MAX_BLOCKS 256
#define S8_GROUP_COST 4
#define S8_MIN_SHARE 12
#define S8_PART (S8_HEADS * S8_D + 3 * S8_HEADS)     // floats of a segment's sums: O, m, mu, l

struct Stream8Params {
    const bf16* q;
    bf16* out;
    const unsigned char* pages;
    const int* block_tables;
    const int* ctx_len;
    long q_stride, out_stride, page_bytes;
    int table_stride, num_pages, max_ctx, R, nq, nkv, page_size, box_tokens, window;
    float scale;
    float* partials;                                 // [blocks][2][S8_PART]: the segment that began earlier, the one that goes on later
    unsigned* arrivals;                              // [blocks], zero between launches
    int* error_flag;
};

// Units i0 .. i1 - 1 of the n units of row group (r, h); the group's unit i holds the keys from (first + i) * 32 on.
struct Seg8 {
    int r, h, i0, i1, n, first, ctx;
    long x, x_end;                                   // place of unit i0 in the launch's list; the place behind the segment
    bool ok;
};

__device__ __forceinline__ int s8_first(int ctx, int window) { return window > 0 && ctx > window ? (ctx - window) / S8_KEYS : 0; }
__device__ __forceinline__ int s8_units(int ctx, int window) {
    const int n = (ctx + S8_KEYS - 1) / S8_KEYS - s8_first(ctx, window);
    return n > 0 ? n : 1;                            // every group is somebody's and gets its rows written
}
__device__ __forceinline__ void s8_enter(Seg8& s, long x, long x1) {
    s.x = x;
    s.i0 = 0;
    const long left = x1 - x;
    s.i1 = (long)s.n <= left ? s.n : (int)left;
    s.x_end = (long)(s.n + S8_GROUP_COST) <= left ? x + s.n + S8_GROUP_COST : x1;
}
__device__ __forceinline__ void s8_request(Seg8& s, const int* pre, const int* ctxs, int window) {
    s.ctx = ctxs[s.r];
    s.n = pre[s.r + 1] - pre[s.r] - S8_GROUP_COST;
    s.first = s8_first(s.ctx, window);
}
__device__ __forceinline__ void s8_next(Seg8& s, long x1, const int* pre, const int* ctxs, int groups, int window) {
    if (s.x_end >= x1) {
        s.ok = false;
        return;
    }
    if (++s.h == groups) {
        s.h = 0;
        ++s.r;
        s8_request(s, pre, ctxs, window);
    }
    s8_enter(s, s.x_end, x1);
}
// the first segment with a unit among the places x .. x1 - 1
__device__ __forceinline__ Seg8 s8_open(long x, long x1, const int* pre, const int* ctxs, int R, int groups, int window) {
    Seg8 s;
    s.ok = x < x1;
    s.x = s.x_end = x;
    s.r = s.h = s.i0 = s.i1 = s.first = s.ctx = 0;
    s.n = 1;
    if (!s.ok) return s;
    int lo = 0, hi = R - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((long)groups * pre[mid] <= x) lo = mid; else hi = mid - 1;
    }
    s.r = lo;
    s8_request(s, pre, ctxs, window);
    const int places = s.n + S8_GROUP_COST;
    const long rel = x - (long)groups * pre[lo];
    s.h = (int)(rel / places);
    const int at = (int)(rel - (long)s.h * places);
    const long left = x1 - x;
    s.x_end = (long)(places - at) <= left ? x + (places - at) : x1;
    s.i0 = at;
    s.i1 = (long)(s.n - at) <= left ? s.n : at + (int)left;
    if (s.i0 >= s.i1) s8_next(s, x1, pre, ctxs, groups, window);
    return s;
}

__device__ __forceinline__ void s8_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned s8_transpose(unsigned x) {
    unsigned y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ unsigned s8_half2(float lo, float hi) {
    unsigned r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float s8_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void s8_load_box(void* smem_dst, const CUtensorMap* map, int token, int kvh, int page, uint64_t* bar) {
    const int zero = 0;
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];\n"
        ::"r"(tc_smem_u32(smem_dst)), "l"(map), "r"(tc_smem_u32(bar)), "r"(zero), "r"(token), "r"(kvh), "r"(zero), "r"(page) : "memory");
}

// A warp's running sums for its two heads 2 t4 and 2 t4 + 1: o[m][0], [1]: entry 16 g + 2 m of either head, [2], [3]: the entry after it.
struct Sums8 {
    float o[8][4];
    float m[2], mu[2], l[2];
};

__device__ __forceinline__ float s8_finite(float m) { return m == -INFINITY ? 0.f : m; }

// One unit: `valid` has a bit for every key that counts (not 0), `meta` the scale bytes of its four blocks of eight keys.
__device__ __forceinline__ void s8_unit(const unsigned char* stage, unsigned valid, const unsigned short (&meta)[4], const unsigned (&qf)[8][2],
                                        const float (&f)[2], int lane, int box_shift, Sums8& s) {
    const int g = lane >> 2, t4 = lane & 3;
    const int box_mask = (1 << box_shift) - 1;
    // 16 bytes of key row (kv 0) or value row (kv 1) `key`, piece `c`
    auto piece = [&](int kv, int key, int c) {
        const int i = key & box_mask;
        return *reinterpret_cast<const uint4*>(stage + (((key >> box_shift) * 2 + kv) << (box_shift + 7)) + i * S8_D + ((c ^ (i & 7)) << 4));
    };
    const int row_key = (g >> 1) + ((g & 1) << 2);
    float t[2][4];
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
        float even[4] = {0.f, 0.f, 0.f, 0.f}, odd[4] = {0.f, 0.f, 0.f, 0.f};        // two chains of products
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint4 lo = piece(0, tile * 16 + row_key, half * 4 + t4), hi = piece(0, tile * 16 + 8 + row_key, half * 4 + t4);
            const unsigned a[4] = {lo.x, lo.y, lo.z, lo.w}, b[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int w = 0; w < 4; ++w)
                s8_mma(w & 1 ? odd : even, kv8_half2((unsigned short)a[w]), kv8_half2((unsigned short)b[w]), kv8_half2((unsigned short)(a[w] >> 16)),
                       kv8_half2((unsigned short)(b[w] >> 16)), qf[half * 4 + w][0], qf[half * 4 + w][1]);
        }
        const float k0 = kv8_scale(meta[tile * 2] & 0xffu), k1 = kv8_scale(meta[tile * 2 + 1] & 0xffu);
#pragma unroll
        for (int c = 0; c < 4; ++c) t[tile][c] = (even[c] + odd[c]) * (c < 2 ? k0 : k1) * f[c & 1];
    }
    if (valid != 0xffffffffu) {
#pragma unroll
        for (int tile = 0; tile < 2; ++tile)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (!((valid >> (tile * 16 + (c >> 1) * 8 + row_key)) & 1u)) t[tile][c] = -INFINITY;
    }
    float u[2][4];
#pragma unroll
    for (int tile = 0; tile < 2; ++tile)
#pragma unroll
        for (int c = 0; c < 4; ++c) u[tile][c] = t[tile][c] + (float)((int)(meta[tile * 2 + (c >> 1)] >> 8) - 127);
    float top[2], utop[2];
    bool raise = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(fmaxf(t[0][h], t[0][2 + h]), fmaxf(t[1][h], t[1][2 + h]));
        utop[h] = fmaxf(fmaxf(u[0][h], u[0][2 + h]), fmaxf(u[1][h], u[1][2 + h]));
        raise = raise || top[h] > s.m[h] + 8.f || utop[h] > s.mu[h] + 8.f;
    }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], o));
                utop[h] = fmaxf(utop[h], __shfl_xor_sync(0xffffffffu, utop[h], o));
            }
            const float m = fmaxf(s.m[h], top[h]), mu = fmaxf(s.mu[h], utop[h]);
            s.l[h] *= m == -INFINITY ? 1.f : s8_ex2(s.m[h] - m);
            const float alpha = mu == -INFINITY ? 1.f : s8_ex2(s.mu[h] - mu);
            s.m[h] = m;
            s.mu[h] = mu;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s.o[i][h] *= alpha;
                s.o[i][2 + h] *= alpha;
            }
        }
    }
    const float m0 = s8_finite(s.m[0]), m1 = s8_finite(s.m[1]), mu0 = s8_finite(s.mu[0]), mu1 = s8_finite(s.mu[1]);
    const unsigned sel_lo = g & 1 ? 0x1504u : 0x5140u, sel_hi = g & 1 ? 0x3726u : 0x7362u;
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
        s.l[0] += s8_ex2(t[tile][0] - m0) + s8_ex2(t[tile][2] - m0);
        s.l[1] += s8_ex2(t[tile][1] - m1) + s8_ex2(t[tile][3] - m1);
        const unsigned b0 = s8_transpose(s8_half2(s8_ex2(u[tile][0] - mu0), s8_ex2(u[tile][1] - mu1)));
        const unsigned b1 = s8_transpose(s8_half2(s8_ex2(u[tile][2] - mu0), s8_ex2(u[tile][3] - mu1)));
        // keys t4 and t4 + 4 of both blocks of eight, the lane's own order first
        const int key = tile * 16 + t4 + ((g & 1) << 2);
        uint4 p0 = piece(1, key, g), p1 = piece(1, key ^ 4, g), p2 = piece(1, key + 8, g), p3 = piece(1, (key ^ 4) + 8, g);
        if (valid != 0xffffffffu) {                              // what lies in hidden places may be no number: 0 * NaN
            const uint4 none = make_uint4(0u, 0u, 0u, 0u);
            if (!((valid >> key) & 1u)) p0 = none;
            if (!((valid >> (key ^ 4)) & 1u)) p1 = none;
            if (!((valid >> (key + 8)) & 1u)) p2 = none;
            if (!((valid >> ((key ^ 4) + 8)) & 1u)) p3 = none;
        }
        const unsigned w0[4] = {p0.x, p0.y, p0.z, p0.w}, w1[4] = {p1.x, p1.y, p1.z, p1.w};
        const unsigned w2[4] = {p2.x, p2.y, p2.z, p2.w}, w3[4] = {p3.x, p3.y, p3.z, p3.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const unsigned a = __byte_perm(w0[w], w1[w], sel_lo), b = __byte_perm(w2[w], w3[w], sel_lo);
            s8_mma(s.o[2 * w], kv8_half2((unsigned short)a), kv8_half2((unsigned short)(a >> 16)), kv8_half2((unsigned short)b),
                   kv8_half2((unsigned short)(b >> 16)), b0, b1);
            const unsigned c = __byte_perm(w0[w], w1[w], sel_hi), d = __byte_perm(w2[w], w3[w], sel_hi);
            s8_mma(s.o[2 * w + 1], kv8_half2((unsigned short)c), kv8_half2((unsigned short)(c >> 16)), kv8_half2((unsigned short)d),
                   kv8_half2((unsigned short)(d >> 16)), b0, b1);
        }
    }
}

// Weight of a partial sum under a common maximum. A sum without a finite score has -inf: it is 0, or no number.
__device__ __forceinline__ float s8_weight(float m, float common) { return m == -INFINITY ? 1.f : s8_ex2(m - common); }

// The row's result from its sums. No keys: zeros.
__device__ __forceinline__ float s8_result(float o, float l, float m, float mu) { return l == 0.f ? 0.f : o / l * exp2f(mu - m); }

#define S8_SYNC() asm volatile("bar.sync 1, %0;\n" ::"n"(S8_WARPS * 32) : "memory")

__global__ void __launch_bounds__(S8_THREADS, 1)
decode_kv8_stream_kernel(const __grid_constant__ CUtensorMap map, const Stream8Params p) {
    extern __shared__ unsigned char s8_raw[];
    __shared__ __align__(8) uint64_t full_bar[S8_STAGES], empty_bar[S8_STAGES];
    __shared__ __align__(8) unsigned short metas[S8_STAGES][4];
    __shared__ float wm[S8_WARPS][S8_HEADS], wmu[S8_WARPS][S8_HEADS], wl[S8_WARPS][S8_HEADS];
    __shared__ int pre[S8_MAX_ROWS + 1], ctxs[S8_MAX_ROWS];      // places of the requests before r, for one group; contexts
    __shared__ unsigned arrived_before;
    const uint32_t raw_addr = tc_smem_u32(s8_raw);
    unsigned char* ring = s8_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
    float* Ow = reinterpret_cast<float*>(ring + (size_t)S8_STAGES * S8_STAGE_BYTES);   // [warps][8][S8_OSTRIDE]

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = p.nq / p.nkv, chunks = (G + S8_HEADS - 1) / S8_HEADS, groups = p.nkv * chunks;

    if (tid == 0) {
#pragma unroll
        for (int s = 0; s < S8_STAGES; ++s) {
            mbar_init(&full_bar[s], 2);                          // the boxes, and the scale bytes
            mbar_init(&empty_bar[s], 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&map) : "memory");
        pre[0] = 0;
    }
    pdl_trigger();
    pdl_wait();
    for (int r = tid; r < p.R; r += S8_THREADS) {
        int ctx = p.ctx_len[r];
        ctx = ctx < 0 ? 0 : (ctx < p.max_ctx ? ctx : p.max_ctx);
        ctxs[r] = ctx;
        pre[r + 1] = s8_units(ctx, p.window) + S8_GROUP_COST;
    }
    __syncthreads();
    if (warp == 0) {
        int carry = 0;
        for (int base = 0; base < p.R; base += 32) {
            int val = base + lane < p.R ? pre[base + lane + 1] : 0;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, val, off);
                if (lane >= off) val += up;
            }
            if (base + lane < p.R) pre[base + lane + 1] = val + carry;
            carry += __shfl_sync(0xffffffffu, val, 31);
        }
    }
    __syncthreads();

    const long N = (long)groups * pre[p.R];
    const long most = N / S8_MIN_SHARE > 0 ? N / S8_MIN_SHARE : 1;
    const long blocks = (long)gridDim.x < most ? (long)gridDim.x : most;
    if ((long)blockIdx.x >= blocks) return;
    const long x0 = (long)blockIdx.x * N / blocks, x1 = ((long)blockIdx.x + 1) * N / blocks;
    Seg8 seg = s8_open(x0, x1, pre, ctxs, p.R, groups, p.window);

    if (warp == S8_WARPS) {
        // ---- loads: eight units at a time, lane 4 u + b the block b of eight keys of unit u ----
        const int u = lane >> 2, b = lane & 3;
        const bool boxes = (b * 8) % p.box_tokens == 0;          // this lane issues a box
        const size_t body = (size_t)2 * p.nkv * p.page_size * S8_D;
        int j = 0;                                               // units of the segment that are on their way
        int count = 0, key = 0, kvh = 0, page = -1;              // the coming batch: its units; this lane's block, its page
        auto fetch = [&]() {
            count = 0;
            if (!seg.ok) return;
            count = min(seg.i1 - seg.i0 - j, 8);
            kvh = seg.h / chunks;
            key = (seg.first + seg.i0 + j + u) * S8_KEYS + b * 8;
            page = -1;
            if (u < count && key < seg.ctx) {
                page = p.block_tables[(size_t)seg.r * p.table_stride + key / p.page_size];
                if (page >= p.num_pages) page = -1;
            }
            j += count;
            if (j == seg.i1 - seg.i0) {
                s8_next(seg, x1, pre, ctxs, groups, p.window);
                j = 0;
            }
        };
        fetch();
        unsigned n0 = 0;
        while (count > 0) {
            const int now = count, at = key, head = kvh, id = page;
            unsigned meta = 0xffffu;                             // a page that is missing
            if (id >= 0) {
                const unsigned char* scales = p.pages + (size_t)id * p.page_bytes + body + head;
                meta = scales[0] | (unsigned)scales[p.nkv] << 8;
            }
            fetch();
            if (u < now) {
                const unsigned n = n0 + u, slot = n % S8_STAGES;
                if (n >= S8_STAGES) mbar_wait(&empty_bar[slot], ((n / S8_STAGES) - 1) & 1, p.error_flag);
                if (b == 0) mbar_expect_tx(&full_bar[slot], S8_STAGE_BYTES);
            }
            __syncwarp();
            if (u < now) {
                const unsigned slot = (n0 + u) % S8_STAGES;
                if (boxes)                                       // out of range: the box arrives as zeros
                    s8_load_box(ring + (size_t)slot * S8_STAGE_BYTES + b * 8 * 2 * S8_D, &map, at % p.page_size, head, id >= 0 ? id : p.num_pages,
                                &full_bar[slot]);
                metas[slot][b] = (unsigned short)meta;
            }
            __syncwarp();
            if (u < now && b == 0)
                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(tc_smem_u32(&full_bar[(n0 + u) % S8_STAGES])) : "memory");
            n0 += now;
        }
        return;
    }

    // ---- compute ----
    const int g = lane >> 2, t4 = lane & 3;
    const int box_shift = 31 - __clz(p.box_tokens);
    unsigned n0 = 0;
    while (seg.ok) {
        const int r = seg.r, kvh = seg.h / chunks, head0 = (seg.h % chunks) * S8_HEADS;
        const int heads = min(G - head0, S8_HEADS);
        // this lane's part of query head g: entries 16 t4 .. 16 t4 + 15 of either half
        unsigned qf[8][2];
        float f[2];
        {
            float x[32], amax = 0.f;
            const bf16* q = p.q + (size_t)r * p.q_stride + (size_t)(kvh * G + head0 + g) * S8_D + t4 * 16;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint4 raw = make_uint4(0u, 0u, 0u, 0u);
                if (g < heads) raw = *reinterpret_cast<const uint4*>(q + (i >> 1) * 64 + (i & 1) * 8);
                const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    x[i * 8 + 2 * c] = __uint_as_float(w[c] << 16);
                    x[i * 8 + 2 * c + 1] = __uint_as_float(w[c] & 0xffff0000u);
                }
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) amax = fmaxf(amax, fabsf(x[i]));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            int e = (int)(__float_as_uint(amax) >> 23);          // 2^(e - 127) <= amax < 2^(e - 126)
            e = e < 1 ? 1 : (e > 253 ? 253 : e);
            const float down = kv8_power(127 - e);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                qf[i][0] = s8_half2(x[4 * i] * down, x[4 * i + 1] * down);
                qf[i][1] = s8_half2(x[4 * i + 2] * down, x[4 * i + 3] * down);
            }
            const float back = p.scale * 1.4426950408889634f * kv8_power(e - 127);
            f[0] = __shfl_sync(0xffffffffu, back, t4 * 8);       // of heads 2 t4 and 2 t4 + 1
            f[1] = __shfl_sync(0xffffffffu, back, t4 * 8 + 4);
        }
        Sums8 s;
#pragma unroll
        for (int i = 0; i < 8; ++i) s.o[i][0] = s.o[i][1] = s.o[i][2] = s.o[i][3] = 0.f;
        s.m[0] = s.m[1] = s.mu[0] = s.mu[1] = -INFINITY;
        s.l[0] = s.l[1] = 0.f;
        const int units = seg.i1 - seg.i0;
        const int low = p.window > 0 ? seg.ctx - p.window : 0;   // the first key that counts
        for (int i = (int)((warp - n0) & (S8_WARPS - 1)); i < units; i += S8_WARPS) {
            const unsigned n = n0 + i, slot = n % S8_STAGES;
            mbar_wait(&full_bar[slot], (n / S8_STAGES) & 1, p.error_flag);
            const int key0 = (seg.first + seg.i0 + i) * S8_KEYS;
            const uint2 raw = *reinterpret_cast<const uint2*>(metas[slot]);
            const unsigned short meta[4] = {(unsigned short)raw.x, (unsigned short)(raw.x >> 16), (unsigned short)raw.y, (unsigned short)(raw.y >> 16)};
            unsigned valid = 0xffffffffu;
            if (seg.ctx - key0 < S8_KEYS) valid = seg.ctx > key0 ? (1u << (seg.ctx - key0)) - 1u : 0u;
            if (low > key0) valid = low - key0 < S8_KEYS ? valid & ~((1u << (low - key0)) - 1u) : 0u;
#pragma unroll
            for (int b = 0; b < 4; ++b)
                if (meta[b] == 0xffffu) valid &= ~(0xffu << (8 * b));
            if (valid != 0u) s8_unit(ring + (size_t)slot * S8_STAGE_BYTES, valid, meta, qf, f, lane, box_shift, s);
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(tc_smem_u32(&empty_bar[slot])) : "memory");
        }
        n0 += units;

        // ---- the segment is read: the warps' sums ----
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) s.l[h] += __shfl_xor_sync(0xffffffffu, s.l[h], o);
            float* row = Ow + ((size_t)warp * S8_HEADS + 2 * t4 + h) * S8_OSTRIDE + g * 16;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(row + 4 * i) = make_float4(s.o[2 * i][h], s.o[2 * i][2 + h], s.o[2 * i + 1][h], s.o[2 * i + 1][2 + h]);
            if (g == 0) {
                wm[warp][2 * t4 + h] = s.m[h];
                wmu[warp][2 * t4 + h] = s.mu[h];
                wl[warp][2 * t4 + h] = s.l[h];
            }
        }
        S8_SYNC();
        const bool whole = seg.i0 == 0 && seg.i1 == seg.n;
        int first_block = 0, shared_by = 1;
        float* part = nullptr;
        if (!whole) {
            const long xg = seg.x - seg.i0;                      // the group's first place in the list
            first_block = (int)(((xg + 1) * blocks - 1) / N);    // the last block whose share starts at or before a place
            shared_by = (int)(((xg + seg.n) * blocks - 1) / N) - first_block + 1;
            part = p.partials + ((size_t)blockIdx.x * 2 + (seg.i0 > 0 ? 0 : 1)) * S8_PART;
        }
        const int col = tid & (S8_D - 1);
        bf16* out = p.out + (size_t)r * p.out_stride + (size_t)(kvh * G + head0) * S8_D + col;
        for (int row = tid >> 7; row < heads; row += S8_WARPS * 32 / S8_D) {
            float m = wm[0][row], mu = wmu[0][row];
#pragma unroll
            for (int w = 1; w < S8_WARPS; ++w) {
                m = fmaxf(m, wm[w][row]);
                mu = fmaxf(mu, wmu[w][row]);
            }
            float acc = 0.f, l = 0.f;
#pragma unroll
            for (int w = 0; w < S8_WARPS; ++w) {
                acc = fmaf(Ow[((size_t)w * S8_HEADS + row) * S8_OSTRIDE + col], s8_weight(wmu[w][row], mu), acc);
                l = fmaf(wl[w][row], s8_weight(wm[w][row], m), l);
            }
            if (whole) {
                out[row * S8_D] = __float2bfloat16_rn(s8_result(acc, l, m, mu));
            } else {
                part[row * S8_D + col] = acc;
                if (col == 0) {
                    part[S8_HEADS * S8_D + row] = m;
                    part[S8_HEADS * S8_D + S8_HEADS + row] = mu;
                    part[S8_HEADS * S8_D + 2 * S8_HEADS + row] = l;
                }
            }
        }
        if (!whole) {
            __threadfence();                                     // the sums are visible before the count is
            S8_SYNC();
            if (tid == 0) arrived_before = atomicAdd(&p.arrivals[first_block], 1u);
            S8_SYNC();
            if (arrived_before == (unsigned)(shared_by - 1)) {
                __threadfence();
                // the first block's segment goes on later, the others' began earlier
                auto part_of = [&](int k) { return p.partials + ((size_t)(first_block + k) * 2 + (k == 0 ? 1 : 0)) * S8_PART; };
                float* ml = Ow;                                  // [shared_by][m of 8 rows | mu | l]: at most 256 * 24 floats
                for (int e = tid; e < shared_by * 3 * S8_HEADS; e += S8_WARPS * 32) {
                    const int k = e / (3 * S8_HEADS);
                    ml[e] = __ldcg(part_of(k) + S8_HEADS * S8_D + (e - k * 3 * S8_HEADS));
                }
                S8_SYNC();
                constexpr int ROWS = S8_HEADS * S8_D / (S8_WARPS * 32);          // rows of a thread: 4
                const int row0 = tid >> 7;
                float m[ROWS], mu[ROWS], l[ROWS], acc[ROWS];
#pragma unroll
                for (int i = 0; i < ROWS; ++i) {
                    m[i] = mu[i] = -INFINITY;
                    l[i] = acc[i] = 0.f;
                }
                for (int k = 0; k < shared_by; ++k)
#pragma unroll
                    for (int i = 0; i < ROWS; ++i) {
                        m[i] = fmaxf(m[i], ml[k * 3 * S8_HEADS + row0 + 2 * i]);
                        mu[i] = fmaxf(mu[i], ml[k * 3 * S8_HEADS + S8_HEADS + row0 + 2 * i]);
                    }
                for (int k0 = 0; k0 < shared_by; k0 += 4) {
                    float val[4][ROWS];
#pragma unroll
                    for (int v = 0; v < 4; ++v)
#pragma unroll
                        for (int i = 0; i < ROWS; ++i)
                            val[v][i] = k0 + v < shared_by && row0 + 2 * i < heads ? __ldcg(part_of(k0 + v) + (row0 + 2 * i) * S8_D + col) : 0.f;
#pragma unroll
                    for (int v = 0; v < 4; ++v)
                        if (k0 + v < shared_by)
#pragma unroll
                            for (int i = 0; i < ROWS; ++i) {
                                const float* of = ml + (k0 + v) * 3 * S8_HEADS + row0 + 2 * i;
                                acc[i] = fmaf(val[v][i], s8_weight(of[S8_HEADS], mu[i]), acc[i]);
                                l[i] = fmaf(of[2 * S8_HEADS], s8_weight(of[0], m[i]), l[i]);
                            }
                }
#pragma unroll
                for (int i = 0; i < ROWS; ++i)
                    if (row0 + 2 * i < heads) out[(row0 + 2 * i) * S8_D] = __float2bfloat16_rn(s8_result(acc[i], l[i], m[i], mu[i]));
                if (tid == 0) p.arrivals[first_block] = 0u;      // for the next launch
            }
        }
        S8_SYNC();                                               // the sums are read: the next segment may write its own
        s8_next(seg, x1, pre, ctxs, groups, p.window);
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------
// Sizes the kernel takes (bfloat16 queries whose rows start on 16 bytes), the scratch it needs and its counters, which are zero before
// a launch and after it; launches that may run at the same time need scratch and counters of their own.
LLMP_API int llmp_kv8_stream_supports(int nq, int nkv, int d, int page_size) {
    return d == S8_D && nkv > 0 && nq % nkv == 0 && (page_size == 8 || page_size == 16 || (page_size > 0 && page_size % 32 == 0));
}
LLMP_API long llmp_kv8_stream_scratch_floats() { return (long)S8_MAX_BLOCKS * 2 * S8_PART; }
LLMP_API int llmp_kv8_stream_counters() { return S8_MAX_BLOCKS; }

LLMP_API int llmp_kv8_stream(const void* q, long q_stride, void* out, long out_stride, const void* pages, int num_pages, const int* block_tables,
                             int table_stride, const int* ctx_len, int R, int max_ctx, int nq, int nkv, int page_size, int window, float scale,
                             float* scratch, long scratch_floats, unsigned* counters, int* error_flag, cudaStream_t stream) {
    if (R <= 0) return 0;
    LLMP_REQUIRE(llmp_kv8_stream_supports(nq, nkv, S8_D, page_size), "kv8 attention: %d and %d heads, pages of %d tokens are not for this kernel", nq, nkv, page_size);
    LLMP_REQUIRE(num_pages > 0 && max_ctx > 0 && table_stride > 0, "kv8 attention: bad context %d or tables", max_ctx);
    LLMP_REQUIRE((q_stride % 8) == 0 && ((size_t)q % 16) == 0 && ((size_t)pages % 16) == 0, "kv8 attention: rows must be 16-byte aligned");
    LLMP_REQUIRE(scratch != nullptr && scratch_floats >= llmp_kv8_stream_scratch_floats() && counters != nullptr && error_flag != nullptr,
                 "kv8 attention: scratch, counters and an error flag are needed");
    static int sms = 0;
    if (sms == 0) {
        int dev = 0, n = 0;
        cudaGetDevice(&dev);
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        sms = n <= 0 ? 148 : (n > S8_MAX_BLOCKS ? S8_MAX_BLOCKS : n);
    }
    Stream8Params p;
    p.pages = (const unsigned char*)pages;
    p.q_stride = q_stride; p.out_stride = out_stride; p.page_bytes = kv8_page_bytes(nkv, page_size, S8_D); p.table_stride = table_stride;
    const long held = (long)table_stride * page_size;            // what a row of the tables has room for
    p.num_pages = num_pages; p.max_ctx = held < max_ctx ? (int)held : max_ctx; p.nq = nq; p.nkv = nkv; p.page_size = page_size;
    p.box_tokens = page_size < S8_KEYS ? page_size : S8_KEYS; p.window = window; p.scale = scale; p.partials = scratch; p.arrivals = counters;
    p.error_flag = error_flag;
    EncodeTiledFn encode = llmp_tensor_map_encoder();
    LLMP_REQUIRE(encode != nullptr, "kv8 attention: the driver does not provide cuTensorMapEncodeTiled");
    CUtensorMap map;
    const cuuint64_t row = S8_D, plane = row * page_size;
    const cuuint64_t dims[5] = {S8_D, (cuuint64_t)page_size, (cuuint64_t)nkv, 2, (cuuint64_t)num_pages};
    const cuuint64_t strides[4] = {row, plane, plane * nkv, (cuuint64_t)p.page_bytes};
    const cuuint32_t box[5] = {S8_D, (cuuint32_t)p.box_tokens, 1, 2, 1};
    const cuuint32_t elem[5] = {1, 1, 1, 1, 1};
    const CUresult rc = encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, const_cast<void*>(pages), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    LLMP_REQUIRE(rc == CUDA_SUCCESS, "kv8 attention: cuTensorMapEncodeTiled failed with code %d", (int)rc);
    const size_t smem = (size_t)S8_STAGES * S8_STAGE_BYTES + sizeof(float) * S8_WARPS * S8_HEADS * S8_OSTRIDE + 1024;
    LLMP_ALLOW_SMEM(decode_kv8_stream_kernel, smem);
    for (int r = 0; r < R; r += S8_MAX_ROWS) {                   // launches that follow one another may share scratch and counters
        p.q = (const bf16*)q + (size_t)r * q_stride;
        p.out = (bf16*)out + (size_t)r * out_stride;
        p.block_tables = block_tables + (size_t)r * table_stride;
        p.ctx_len = ctx_len + r;
        p.R = R - r < S8_MAX_ROWS ? R - r : S8_MAX_ROWS;
        llmp_launch_dependent(decode_kv8_stream_kernel, dim3((unsigned)sms), dim3(S8_THREADS), smem, stream, map, p);
    }
    return llmp_check_launch("kv8_stream");
}
