// Attention of single tokens over pages of 8-bit keys and values (kv8.cuh), bfloat16 queries, head size 128: one stream per
// SM. Four warps keep a ring of TMA boxes in flight, eight work through what has landed with mma.sync.
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
// product wants. The queries are brought to a largest magnitude in [1, 4) by a power of two per row: half precision then holds
// every bit of bfloat16's in entries down to 2^-17 of the largest, and smaller ones to 2^-25 of it (one type for both operands, and the sum
// is taken to 2^-24 of its largest terms anyway).
//
// With t = log2(e) scale q.k and a value's scale 2^v, weights are 2^t and a value's factor is 2^(t + v). Each has its own running
// maximum (m for t, mu for t + v): the sum l of the weights and the factors in half precision (at most 2^8: a maximum is only raised
// when it is passed by 8) both keep their bits whatever the scales of the blocks are. out = O / l * 2^(mu - m). A factor is rounded to 2^-11 of
// itself, an eighth of what the result's own rounding to bfloat16 takes (in bfloat16 it would be as much); l is in float32. Against 64 bits the
// results are off by 0.0015 to 0.0017 of their size, as those of the formula in 32 bits rounded once are, to the sixth digit.
//
// At the end of a segment (what a block has of a group) the warps' sums are added in shared memory. A whole group is written out;
// of a shared one every block leaves its sums in global memory and counts itself at its end, and the block that counts last adds them
// in block order, writes, and sets the counter back to zero. Nobody waits for anybody. Every wait on an mbarrier is bounded: when one runs
// out the kernel records 1 in *error_flag and goes on without waiting (its output is then wrong; the host reads the flag).
//
// What bounds it: bytes for many long requests (64 of 8,192 tokens, 32 and 8 heads: 175 us, 6.1 TB/s; 64 ragged ones of up to 4,002:
// 58 us, 5.0 TB/s), for few of them the first boxes' way and the sums over warps and blocks, about 8 us (8 of 2,048: 13.0 us; 1 of 300: 6.6).
// Loading warps of their own against boxes asked for by the warps that compute: one warp issues a box in about 100 ns.
#include "kv8.cuh"
#include "tcgen05.cuh"

#define S8_D 128
#define S8_WARPS 8
#define S8_KEYS 32
#define S8_STAGE_BYTES (2 * S8_KEYS * S8_D)
#define S8_DEPTH 2                                   // units of a warp in shared memory: the one it works on and the next
#define S8_LOADERS 4                                 // warps that load
#define S8_ASK 2                                     // units of a turn of theirs
#define S8_THREADS ((S8_WARPS + S8_LOADERS) * 32)
#define S8_HEADS 8
#define S8_OSTRIDE (S8_D + 4)                        // floats of a row of a warp's sums in shared memory
#define S8_MAX_ROWS 512                              // requests of a launch (their places are summed in shared memory)
#define S8_MAX_BLOCKS 256
#define S8_GROUP_COST 16                             // places of a group besides its units: with 4, 64 ragged requests 70 us (58), one long of 8 20.7 (17.7)
#define S8_MIN_SHARE 12                              // places of a block at least: fewer blocks for short lists, which have less to add up
#define S8_OWN_UNITS 16                              // units of a block at least where a group has blocks of its own
#define S8_EVEN_COST 16                              // what borders inside groups cost a block, in units
// Unit n of a block lies in stage n mod (S8_WARPS S8_DEPTH) and is read by warp n mod S8_WARPS: a stage is always the same warp's. Boxes
// do not land in the order in which they were asked for: were a stage read by two warps in turn, the second could look at its barrier while
// the first's data is still on its way, one phase early, where a wait for a parity cannot tell that from one phase late.
#define S8_PART (S8_HEADS * S8_D + 4 * S8_HEADS)     // floats of a segment's sums: O, then m, mu, l of each row

struct Stream8Params {
    const bf16* q;
    bf16* out;
    const unsigned char* pages;
    const int* block_tables;
    const int* ctx_len;
    long q_stride, out_stride, page_bytes;
    int table_stride, num_pages, max_ctx, R, nq, nkv, page_size, page_shift, window;
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

// One unit, whose boxes hold BOX tokens: `valid` has a bit for every key that counts (not 0), `scales` what its four blocks of eight keys are
// to be multiplied by: the keys' scale, and the exponent of the values'. Keys and values lie as [box][keys, values][token][128], in
// TMA's swizzle (16-byte piece c of token i at c ^ (i & 7)).
template <int BOX>
__device__ __forceinline__ void s8_unit(const unsigned char* stage, unsigned valid, const float2 (&scales)[4], const unsigned (&qf)[8][2],
                                        const float (&f)[2], int lane, Sums8& s) {
    const int g = lane >> 2, t4 = lane & 3;
    const int row_key = (g >> 1) + ((g & 1) << 2);
    auto token = [](int kv, int key) { return ((key / BOX) * 2 + kv) * BOX * S8_D + (key % BOX) * S8_D; };     // of multiples of 8: known here
    const unsigned char* k_at[2] = {stage + row_key * S8_D + ((t4 ^ row_key) << 4), stage + row_key * S8_D + (((4 + t4) ^ row_key) << 4)};
    const int v_key = t4 + ((g & 1) << 2);                       // the lane's own order of keys t4 and t4 + 4
    const unsigned char* v_at[2] = {stage + v_key * S8_D + ((g ^ v_key) << 4), stage + (v_key ^ 4) * S8_D + ((g ^ v_key ^ 4) << 4)};
    auto piece = [](const unsigned char* at) { return *reinterpret_cast<const uint4*>(at); };
    float t[2][4];
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
        float even[4] = {0.f, 0.f, 0.f, 0.f}, odd[4] = {0.f, 0.f, 0.f, 0.f};        // two chains of products
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint4 lo = piece(k_at[half] + token(0, tile * 16)), hi = piece(k_at[half] + token(0, tile * 16 + 8));
            const unsigned a[4] = {lo.x, lo.y, lo.z, lo.w}, b[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int w = 0; w < 4; ++w)
                s8_mma(w & 1 ? odd : even, kv8_half2((unsigned short)a[w]), kv8_half2((unsigned short)b[w]), kv8_half2((unsigned short)(a[w] >> 16)),
                       kv8_half2((unsigned short)(b[w] >> 16)), qf[half * 4 + w][0], qf[half * 4 + w][1]);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) t[tile][c] = (even[c] + odd[c]) * scales[tile * 2 + (c >> 1)].x * f[c & 1];
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
        for (int c = 0; c < 4; ++c) u[tile][c] = t[tile][c] + scales[tile * 2 + (c >> 1)].y;
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
        uint4 p0 = piece(v_at[0] + token(1, tile * 16)), p1 = piece(v_at[1] + token(1, tile * 16));
        uint4 p2 = piece(v_at[0] + token(1, tile * 16 + 8)), p3 = piece(v_at[1] + token(1, tile * 16 + 8));
        if (valid != 0xffffffffu) {                              // what lies in hidden places may be no number: 0 * NaN
            const uint4 none = make_uint4(0u, 0u, 0u, 0u);
            const int key = tile * 16 + v_key;
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

// Four columns of a row's result from its sums (8-byte aligned).
__device__ __forceinline__ void s8_store(bf16* out, float4 o, float l, float m, float mu) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(s8_result(o.x, l, m, mu), s8_result(o.y, l, m, mu));
    const __nv_bfloat162 b = __floats2bfloat162_rn(s8_result(o.z, l, m, mu), s8_result(o.w, l, m, mu));
    *reinterpret_cast<uint2*>(out) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
}

// A group of `heads` rows from row (r, head) on that the blocks first_block .. first_block + by - 1 share (by 0: none).
struct Shared8 {
    int first_block, by, heads, r, head;
};

#define S8_SYNC() asm volatile("bar.sync 1, %0;\n" ::"n"(S8_WARPS * 32) : "memory")       // of the warps that compute

template <int BOX>
__global__ void __launch_bounds__(S8_THREADS, 1)
decode_kv8_stream_kernel(const __grid_constant__ CUtensorMap map, const Stream8Params p) {
    extern __shared__ unsigned char s8_raw[];
    __shared__ __align__(8) uint64_t full_bar[S8_WARPS * S8_DEPTH], empty_bar[S8_WARPS * S8_DEPTH];      // stage d * S8_WARPS + w: warp w's
    __shared__ __align__(16) float2 unit_scales[S8_WARPS * S8_DEPTH][4];
    __shared__ float wm[S8_WARPS][S8_HEADS], wmu[S8_WARPS][S8_HEADS], wl[S8_WARPS][S8_HEADS];
    __shared__ int pre[S8_MAX_ROWS + 1], ctxs[S8_MAX_ROWS];      // places of the requests before r, for one group; contexts
    __shared__ int longest;
    __shared__ Shared8 shared[2];                                // this block's part of a group that began earlier, of one that goes on later
    const uint32_t raw_addr = tc_smem_u32(s8_raw);
    unsigned char* ring = s8_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
    float* Ow = reinterpret_cast<float*>(ring + (size_t)S8_WARPS * S8_DEPTH * S8_STAGE_BYTES);      // [warps][8][S8_OSTRIDE]

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = p.nq / p.nkv, chunks = (G + S8_HEADS - 1) / S8_HEADS, groups = p.nkv * chunks;

    if (tid < S8_WARPS * S8_DEPTH) {
        mbar_init(&full_bar[tid], 2);                            // the boxes, and the scales
        mbar_init(&empty_bar[tid], 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (tid == 32) asm volatile("prefetch.tensormap [%0];\n" ::"l"(&map) : "memory");
    if (tid == 0) pre[0] = 0;
    if (tid < 2) shared[tid].by = 0;
    pdl_trigger();
    pdl_wait();
    if (warp == 0) {                                             // places, their running sums, the longest group
        int carry = 0, most = 0;
        for (int base = 0; base < p.R; base += 32) {
            int val = 0;
            if (base + lane < p.R) {
                int ctx = p.ctx_len[base + lane];
                ctx = ctx < 0 ? 0 : (ctx < p.max_ctx ? ctx : p.max_ctx);
                ctxs[base + lane] = ctx;
                val = s8_units(ctx, p.window) + S8_GROUP_COST;
            }
            most = max(most, val);
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, val, off);
                if (lane >= off) val += up;
            }
            if (base + lane < p.R) pre[base + lane + 1] = val + carry;
            carry += __shfl_sync(0xffffffffu, val, 31);
        }
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) longest = most - S8_GROUP_COST;
    }
    __syncthreads();

    // How the list is dealt out: evenly, or (few groups of about the same length) every group to `split` blocks of its own, which
    // spares most blocks a second group and the borders that fall inside groups.
    const long N = (long)groups * pre[p.R];
    const long most = N / S8_MIN_SHARE > 0 ? N / S8_MIN_SHARE : 1;
    const long blocks = (long)gridDim.x < most ? (long)gridDim.x : most;
    const int all = p.R * groups;
    int split = 0;
    if (all <= (int)gridDim.x) {
        split = min((int)gridDim.x / all, (longest + S8_OWN_UNITS - 1) / S8_OWN_UNITS);
        if ((longest + split - 1) / split > N / blocks + S8_EVEN_COST) split = 0;
    }
    Seg8 seg;
    long x1 = 0;
    if (split > 0) {
        const int group = blockIdx.x / split, part = blockIdx.x % split;
        if (group >= all) return;
        seg.r = group / groups;
        seg.h = group % groups;
        s8_request(seg, pre, ctxs, p.window);
        const int own = min(split, (seg.n + S8_OWN_UNITS - 1) / S8_OWN_UNITS);   // a short group takes fewer
        if (part >= own) return;
        seg.i0 = (int)((long)seg.n * part / own);
        seg.i1 = (int)((long)seg.n * (part + 1) / own);
        seg.ok = true;
        seg.x = seg.x_end = x1 = 0;
        if (tid == 0 && own > 1) shared[part == 0 ? 1 : 0] = Shared8{group * split, own, 0, 0, 0};
    } else {
        if ((long)blockIdx.x >= blocks) return;
        x1 = ((long)blockIdx.x + 1) * N / blocks;
        seg = s8_open((long)blockIdx.x * N / blocks, x1, pre, ctxs, p.R, groups, p.window);
    }

    if (warp >= S8_WARPS) {
        // ---- loads: warp l of S8_LOADERS serves the units n with n mod S8_LOADERS = l, a few at a time: lane 4 u + b sees to block b of
        // eight keys of the u-th of them. Page numbers are asked for two turns ahead, scale bytes one, so that neither is waited for
        // while boxes could be on their way. ----
        const int u = lane >> 2, b = lane & 3;
        const bool boxes = (b * 8) % BOX == 0;                   // this lane issues a box
        const size_t body = (size_t)2 * p.nkv * p.page_size * S8_D;
        struct Ask {
            int key, head, page;
            bool ok;
        };
        unsigned n_ahead = (unsigned)(warp - S8_WARPS) + u * S8_LOADERS;         // this lane's coming unit, counted from the block's first
        unsigned before = 0;                                     // units of the block before `seg`
        auto fetch = [&]() {
            Ask t;
            while (seg.ok && n_ahead - before >= (unsigned)(seg.i1 - seg.i0)) {
                before += seg.i1 - seg.i0;
                s8_next(seg, x1, pre, ctxs, groups, p.window);
            }
            t.ok = seg.ok && u < S8_ASK;
            t.page = -1;
            t.key = (seg.first + seg.i0 + (int)(n_ahead - before)) * S8_KEYS + b * 8;
            t.head = seg.h / chunks;
            if (t.ok && t.key < seg.ctx) t.page = p.block_tables[(size_t)seg.r * p.table_stride + (t.key >> p.page_shift)];
            n_ahead += S8_LOADERS * S8_ASK;
            return t;
        };
        unsigned ek = 0u, ev = 0u;
        auto scales = [&](Ask& t) {
            if (t.page >= p.num_pages) t.page = -1;
            if (t.page >= 0) {
                const unsigned char* at = p.pages + (size_t)t.page * p.page_bytes + body + t.head;
                ek = at[0];
                ev = at[p.nkv];
            }
        };
        unsigned n = n_ahead;
        Ask now = fetch(), next = fetch();
        scales(now);
        while (__any_sync(0xffffffffu, now.ok)) {
            const Ask after = fetch();
            const unsigned slot = n % (S8_WARPS * S8_DEPTH), round = n / (S8_WARPS * S8_DEPTH);
            if (now.ok) {
                if (round > 0) mbar_wait(&empty_bar[slot], (round - 1) & 1, p.error_flag);
                if (b == 0) mbar_expect_tx(&full_bar[slot], S8_STAGE_BYTES);
            }
            __syncwarp();
            if (now.ok && boxes)                                 // out of range: the box arrives as zeros
                s8_load_box(ring + (size_t)slot * S8_STAGE_BYTES + b * 8 * 2 * S8_D, &map, now.key & (p.page_size - 1), now.head,
                            now.page >= 0 ? now.page : p.num_pages, &full_bar[slot]);
            if (now.ok) unit_scales[slot][b] = make_float2(now.page >= 0 ? kv8_scale(ek) : -1.f, (float)((int)ev - 127));      // -1: a page that is missing
            __syncwarp();
            if (now.ok && b == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(tc_smem_u32(&full_bar[slot])) : "memory");
            n += S8_LOADERS * S8_ASK;
            now = next;
            next = after;
            scales(now);
        }
        return;
    }

    // ---- compute: unit n of the block is warp n mod S8_WARPS's ----
    const int g = lane >> 2, t4 = lane & 3;
    int at = warp;                                               // the coming unit of `seg`, counted from its i0
    unsigned k = 0;                                              // this warp's units so far
    uint4 q_raw[4];                                              // entries 16 t4 .. 16 t4 + 15 of either half of query head g
    auto ask_q = [&](const Seg8& of) {
        const int head = (of.h % chunks) * S8_HEADS + g;         // within the group that shares a key/value head
        const bf16* q = p.q + (size_t)of.r * p.q_stride + (size_t)(of.h / chunks * G + head) * S8_D + t4 * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            q_raw[i] = make_uint4(0u, 0u, 0u, 0u);
            if (of.ok && head < G) q_raw[i] = *reinterpret_cast<const uint4*>(q + (i >> 1) * 64 + (i & 1) * 8);
        }
    };
    ask_q(seg);
    while (seg.ok) {
        const int r = seg.r, kvh = seg.h / chunks, head0 = (seg.h % chunks) * S8_HEADS;
        const int heads = min(G - head0, S8_HEADS);
        // this lane's part of query head g, which was asked for before the segment before this one ended
        unsigned qf[8][2];
        float f[2];
        {
            float x[32], amax = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned w[4] = {q_raw[i].x, q_raw[i].y, q_raw[i].z, q_raw[i].w};
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
        for (; at < units; at += S8_WARPS, ++k) {
            const unsigned slot = k % S8_DEPTH * S8_WARPS + warp;
            mbar_wait(&full_bar[slot], (k / S8_DEPTH) & 1, p.error_flag);
            const float4 s01 = reinterpret_cast<const float4*>(unit_scales[slot])[0], s23 = reinterpret_cast<const float4*>(unit_scales[slot])[1];
            const float2 scales[4] = {make_float2(s01.x, s01.y), make_float2(s01.z, s01.w), make_float2(s23.x, s23.y), make_float2(s23.z, s23.w)};
            const int key0 = (seg.first + seg.i0 + at) * S8_KEYS;
            unsigned valid = 0xffffffffu;
            if (seg.ctx - key0 < S8_KEYS) valid = seg.ctx > key0 ? (1u << (seg.ctx - key0)) - 1u : 0u;
            if (low > key0) valid = low - key0 < S8_KEYS ? valid & ~((1u << (low - key0)) - 1u) : 0u;
#pragma unroll
            for (int b = 0; b < 4; ++b)
                if (scales[b].x < 0.f) valid &= ~(0xffu << (8 * b));
            if (valid != 0u) s8_unit<BOX>(ring + (size_t)slot * S8_STAGE_BYTES, valid, scales, qf, f, lane, s);
            __syncwarp();                                        // the stage is read: it may be filled again
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(tc_smem_u32(&empty_bar[slot])) : "memory");
        }
        at -= units;

        // ---- the segment is read: the warps' maxima, then their sums under the largest ----
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (g == 0) {
                wm[warp][2 * t4 + h] = s.m[h];
                wmu[warp][2 * t4 + h] = s.mu[h];
            }
        S8_SYNC();
        float top[2], utop[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            top[h] = utop[h] = -INFINITY;
#pragma unroll
            for (int w = 0; w < S8_WARPS; ++w) {
                top[h] = fmaxf(top[h], wm[w][2 * t4 + h]);
                utop[h] = fmaxf(utop[h], wmu[w][2 * t4 + h]);
            }
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) s.l[h] += __shfl_xor_sync(0xffffffffu, s.l[h], o);
            const float weight = s8_weight(s.mu[h], utop[h]);
            float* row = Ow + ((size_t)warp * S8_HEADS + 2 * t4 + h) * S8_OSTRIDE + g * 16;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(row + 4 * i) = make_float4(s.o[2 * i][h] * weight, s.o[2 * i][2 + h] * weight, s.o[2 * i + 1][h] * weight,
                                                                      s.o[2 * i + 1][2 + h] * weight);
            if (g == 0) wl[warp][2 * t4 + h] = s.l[h] * s8_weight(s.m[h], top[h]);
        }
        S8_SYNC();
        Seg8 after = seg;
        s8_next(after, x1, pre, ctxs, groups, p.window);
        ask_q(after);
        const bool whole = seg.i0 == 0 && seg.i1 == seg.n;
        if (!whole && tid == 0) {
            Shared8& of = shared[seg.i0 > 0 ? 0 : 1];
            if (split == 0) {
                const long xg = seg.x - seg.i0;                  // the group's first place in the list
                of.first_block = (int)(((xg + 1) * blocks - 1) / N);     // the last block whose share starts at or before a place
                of.by = (int)(((xg + seg.n) * blocks - 1) / N) - of.first_block + 1;
            }
            of.heads = heads;
            of.r = r;
            of.head = kvh * G + head0;
        }
        if (warp < heads) {                                      // a warp takes a row, a lane four columns
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            float l = 0.f, m = -INFINITY, mu = -INFINITY;
#pragma unroll
            for (int w = 0; w < S8_WARPS; ++w) {
                const float4 v = *reinterpret_cast<const float4*>(Ow + ((size_t)w * S8_HEADS + warp) * S8_OSTRIDE + lane * 4);
                o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
                l += wl[w][warp];
                m = fmaxf(m, wm[w][warp]);
                mu = fmaxf(mu, wmu[w][warp]);
            }
            if (whole) {
                s8_store(p.out + (size_t)r * p.out_stride + (size_t)(kvh * G + head0 + warp) * S8_D + lane * 4, o, l, m, mu);
            } else {
                float* part = p.partials + ((size_t)blockIdx.x * 2 + (seg.i0 > 0 ? 0 : 1)) * S8_PART;
                *reinterpret_cast<float4*>(part + warp * S8_D + lane * 4) = o;
                if (lane == 0) *reinterpret_cast<float4*>(part + S8_HEADS * S8_D + warp * 4) = make_float4(m, mu, l, 0.f);
            }
        }
        S8_SYNC();                                               // the sums are read: the next segment may write its own
        seg = after;
    }

    // ---- groups that this block shares with others: counted once all its own are read (one thread's fence covers what the block
    // wrote before the barrier), and those added up that it is the last to count on ----
    S8_SYNC();
    if (tid < 2 && shared[tid].by > 0) {
        __threadfence();
        const unsigned before = atomicAdd(&p.arrivals[shared[tid].first_block], 1u);
        __threadfence();
        if (before != (unsigned)(shared[tid].by - 1)) shared[tid].by = 0;
    }
    S8_SYNC();
    for (int which = 0; which < 2; ++which) {
        const Shared8 of = shared[which];
        if (of.by == 0 || warp >= of.heads) continue;
        // the first block's segment goes on later, the others' began earlier
        auto part_of = [&](int b) { return p.partials + ((size_t)(of.first_block + b) * 2 + (b == 0 ? 1 : 0)) * S8_PART; };
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f, m = -INFINITY, mu = -INFINITY;
        for (int b0 = 0; b0 < of.by; b0 += 4) {                  // four blocks at a time, what they left on its way together
            float4 v[4], ml[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                ml[b] = make_float4(-INFINITY, -INFINITY, 0.f, 0.f);
                v[b] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (b0 + b < of.by) {
                    v[b] = __ldcg(reinterpret_cast<const float4*>(part_of(b0 + b) + warp * S8_D) + lane);
                    ml[b] = __ldcg(reinterpret_cast<const float4*>(part_of(b0 + b) + S8_HEADS * S8_D) + warp);
                }
            }
            float m_new = m, mu_new = mu;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                m_new = fmaxf(m_new, ml[b].x);
                mu_new = fmaxf(mu_new, ml[b].y);
            }
            l *= s8_weight(m, m_new);
            const float old = s8_weight(mu, mu_new);
            o.x *= old; o.y *= old; o.z *= old; o.w *= old;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                l = fmaf(ml[b].z, s8_weight(ml[b].x, m_new), l);
                const float w = s8_weight(ml[b].y, mu_new);
                o.x = fmaf(v[b].x, w, o.x); o.y = fmaf(v[b].y, w, o.y); o.z = fmaf(v[b].z, w, o.z); o.w = fmaf(v[b].w, w, o.w);
            }
            m = m_new;
            mu = mu_new;
        }
        s8_store(p.out + (size_t)of.r * p.out_stride + (size_t)(of.head + warp) * S8_D + lane * 4, o, l, m, mu);
        if (tid == 0) p.arrivals[of.first_block] = 0u;           // for the next launch
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------
// Sizes the kernel takes (bfloat16 queries whose rows start on 16 bytes), the scratch it needs and its counters, which are zero before
// a launch and after it; launches that may run at the same time need scratch and counters of their own.
LLMP_API int llmp_kv8_stream_supports(int nq, int nkv, int d, int page_size) {
    return d == S8_D && nq > 0 && nkv > 0 && nq % nkv == 0 && page_size >= 8 && (page_size & (page_size - 1)) == 0;
}
LLMP_API long llmp_kv8_stream_scratch_floats() { return (long)S8_MAX_BLOCKS * 2 * S8_PART; }
LLMP_API int llmp_kv8_stream_counters() { return S8_MAX_BLOCKS; }

LLMP_API int llmp_kv8_stream(const void* q, long q_stride, void* out, long out_stride, const void* pages, int num_pages, const int* block_tables,
                             int table_stride, const int* ctx_len, int R, int max_ctx, int nq, int nkv, int page_size, int window, float scale,
                             float* scratch, long scratch_floats, unsigned* counters, int* error_flag, cudaStream_t stream) {
    if (R <= 0) return 0;
    LLMP_REQUIRE(llmp_kv8_stream_supports(nq, nkv, S8_D, page_size), "kv8 attention: %d and %d heads, pages of %d tokens are not for this kernel", nq, nkv, page_size);
    LLMP_REQUIRE(num_pages > 0 && max_ctx > 0 && table_stride > 0, "kv8 attention: bad context %d or tables", max_ctx);
    LLMP_REQUIRE((q_stride % 8) == 0 && ((size_t)q % 16) == 0 && ((size_t)pages % 16) == 0 && ((size_t)out % 8) == 0 && (out_stride % 4) == 0, "kv8 attention: rows must be 16-byte aligned");
    LLMP_REQUIRE(scratch != nullptr && scratch_floats >= llmp_kv8_stream_scratch_floats() && counters != nullptr && error_flag != nullptr,
                 "kv8 attention: scratch, counters and an error flag are needed");
    static int blocks = 0;
    if (blocks == 0) {
        int dev = 0, n = 0;
        cudaGetDevice(&dev);
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        n = n <= 0 ? 148 : n;
        blocks = n > S8_MAX_BLOCKS ? S8_MAX_BLOCKS : n;
    }
    Stream8Params p;
    p.pages = (const unsigned char*)pages;
    p.q_stride = q_stride; p.out_stride = out_stride; p.page_bytes = kv8_page_bytes(nkv, page_size, S8_D); p.table_stride = table_stride;
    const long held = (long)table_stride * page_size;            // what a row of the tables has room for
    p.num_pages = num_pages; p.max_ctx = held < max_ctx ? (int)held : max_ctx; p.nq = nq; p.nkv = nkv; p.page_size = page_size;
    p.page_shift = 31 - __builtin_clz((unsigned)page_size); p.window = window; p.scale = scale; p.partials = scratch; p.arrivals = counters;
    p.error_flag = error_flag;
    const int box_tokens = page_size < S8_KEYS ? page_size : S8_KEYS;
    EncodeTiledFn encode = llmp_tensor_map_encoder();
    LLMP_REQUIRE(encode != nullptr, "kv8 attention: the driver does not provide cuTensorMapEncodeTiled");
    CUtensorMap map;
    const cuuint64_t row = S8_D, plane = row * page_size;
    const cuuint64_t dims[5] = {S8_D, (cuuint64_t)page_size, (cuuint64_t)nkv, 2, (cuuint64_t)num_pages};
    const cuuint64_t strides[4] = {row, plane, plane * nkv, (cuuint64_t)p.page_bytes};
    const cuuint32_t box[5] = {S8_D, (cuuint32_t)box_tokens, 1, 2, 1};
    const cuuint32_t elem[5] = {1, 1, 1, 1, 1};
    const CUresult rc = encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, const_cast<void*>(pages), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    LLMP_REQUIRE(rc == CUDA_SUCCESS, "kv8 attention: cuTensorMapEncodeTiled failed with code %d", (int)rc);
    const size_t smem = (size_t)S8_WARPS * S8_DEPTH * S8_STAGE_BYTES + sizeof(float) * S8_WARPS * S8_HEADS * S8_OSTRIDE + 1024;
    const auto kernel = box_tokens == 8 ? decode_kv8_stream_kernel<8> : box_tokens == 16 ? decode_kv8_stream_kernel<16> : decode_kv8_stream_kernel<32>;
    if (box_tokens == 8) LLMP_ALLOW_SMEM(decode_kv8_stream_kernel<8>, smem);
    else if (box_tokens == 16) LLMP_ALLOW_SMEM(decode_kv8_stream_kernel<16>, smem);
    else LLMP_ALLOW_SMEM(decode_kv8_stream_kernel<32>, smem);
    for (int r = 0; r < R; r += S8_MAX_ROWS) {                   // launches that follow one another may share scratch and counters
        p.q = (const bf16*)q + (size_t)r * q_stride;
        p.out = (bf16*)out + (size_t)r * out_stride;
        p.block_tables = block_tables + (size_t)r * table_stride;
        p.ctx_len = ctx_len + r;
        p.R = R - r < S8_MAX_ROWS ? R - r : S8_MAX_ROWS;
        llmp_launch_dependent(kernel, dim3((unsigned)blocks), dim3(S8_THREADS), smem, stream, map, p);
    }
    return llmp_check_launch("kv8_stream");
}
