// Causal attention of prompt portions over pages of 8-bit keys and values (kv8.cuh) on the fifth-generation tensor cores: bfloat16
// queries, head size 128, as llmp_paged_attention over pages of bfloat16.
//
// A block takes 256 query rows of one request and one key/value head (a row is a token and a query head of the group, the head running
// fastest) as two tiles of 128, and walks tiles of 128 keys. All products are in half precision, which holds every e4m3 value (and 2^-8 of it) exactly:
//   unpack       six warps turn a tile's bytes into half precision, laid out as operands; both row tiles use what is unpacked once. By
//                shifts and masks: the conversion instruction is as slow as the exponentials and shares their unit
//   S = Q K^T    Q, K in shared memory (128-byte swizzle, K-major), S in tensor memory
//   softmax      a thread has a row: it reads S from tensor memory twice (maxima; factors), 32 columns at a time, and writes its factors
//                over S. The loops stay short and what is rare stands outside them (masks, weights that factors do not give, values that
//                are no number), since the instructions of four roles do not come fast enough otherwise: 2,048 tokens behind 14,000
//                took 771 us with 64 columns a turn and all of it inside, 741 with 32, 649 so; one pass, with the rescaling inside, 744
//   O += P V     P read from tensor memory, V in shared memory MN-major, O in tensor memory
// While one row tile is in its softmax the tensor cores work for the other. The two tiles' S and O fill the tensor memory (512 columns).
// What bounds it: a row tile's chain of S, maxima, factors, P V, one after another, 5,000 clocks a key tile, of them the softmax 3,100 and
// the products 1,030. 2,048 tokens (32 heads) 66 us, 0.52 PFLOP/s; behind 14,000 649 us, 0.78 PFLOP/s; 40 behind 8,000 30.7 us.
//
// With t = log2(e) scale q.k and a value's scale 2^v, weights are 2^t and the factor of a value's bytes is 2^(t + v). As in
// attention_decode_kv8_stream.cu each has its own maximum, m and mu, raised to a whole number when it is passed by more than 12: factors
// are held in half precision relative to 2^mu, the sum l of the weights in float32 relative to 2^m, and out = O / l * 2^(mu - m). The keys
// of a page have one scale, so a weight is its factor times 2^(mu - m - v), a power of two; only where that is beyond 2^100 are the weights
// computed apart. Queries are brought to a largest magnitude in
// [1, 4) by a power of two per row, which takes the sign of the scale along.
//
// Roundings: factors to half precision, 2^-11 of themselves (bfloat16 operands would take 2^-8 and as many cycles); queries as in
// attention_decode_kv8_stream.cu; l and O in float32. Against 64 bits 2,048 tokens are off by 0.00164 of their size, the formula in 32 bits
// rounded once by 0.00163, portions through unpacked bfloat16 pages, whose weights are bfloat16, by 0.0020.
//
// What cannot be seen does not matter: bytes behind the context and in missing pages are zeros as operands; those that are no number are
// too, and the rows that see their key become no number by their l, in every entry of the head.
//
// Roles: warps 0-3 and 4-7 softmax of the two row tiles, 8-13 unpacking, 14 loads (TMA, a page and head in a box, keys and values
// together), 15 issues the products. Few rows over many keys: an item of the list is a part of a row tile's keys and leaves its sums
// in global memory, and prompt_kv8_merge_kernel adds them up. Every wait on an mbarrier is bounded: when one runs out the kernel records
// 1 in *error_flag and goes on without waiting (its output is then wrong; the host reads the flag).
#include "kv8.cuh"
#include "prefill_tc.cuh"
#include "tcgen05.cuh"

#define P8_D 128
#define P8_ROWS 128                                  // of a row tile
#define P8_KEYS 128
#define P8_THREADS 512
#define P8_STAGES 2                                  // tiles of bytes on their way or being unpacked, keys and values each
#define P8_UNPACK 6                                  // warps that unpack
#define P8_PIECES 3                                  // 16 bytes each that a lane unpacks side by side
#define P8_HALF (P8_ROWS * 128)                      // bytes of 128 rows of 64 entries in half precision
#define P8_RAW (P8_KEYS * P8_D)                      // bytes of a tile's keys, or values
#define P8_SLOTS 8                                   // places for a tile's scales, which live until its softmax is done
#define P8_PART (P8_D + 4)                           // floats of a row's sums: O, m, mu, l

struct Prompt8Params {
    const bf16* q;
    bf16* out;
    const unsigned char* pages;
    const int* block_tables;
    const int* q_start;
    const int* ctx_len;
    const int* items;                                // [num_items][4]: request, first token, part | parts << 16, place of the item's sums
    float* partials;                                 // [places][nkv][256][P8_PART]
    long q_stride, out_stride, page_bytes;
    int table_stride, num_pages, nq, nkv, page_size, page_shift, window, tokens;
    float scale;
    int* error_flag;
};

__device__ __forceinline__ void p8_load_box(void* smem_dst, const CUtensorMap* map, int token, int kvh, int kv, int page, uint64_t* bar) {
    const int zero = 0;
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];\n"
        ::"r"(tc_smem_u32(smem_dst)), "l"(map), "r"(tc_smem_u32(bar)), "r"(zero), "r"(token), "r"(kvh), "r"(kv), "r"(page) : "memory");
}

// Instruction descriptor of kind::f16 with half-precision operands and float32 sums, M x N.
__host__ __device__ constexpr uint32_t p8_idesc(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

// Shared-memory descriptor of an MN-major operand in the 128-byte swizzle: rows of 64 contiguous entries, one per K index, eight of
// them 1024 bytes, the next 64 entries P8_HALF further.
__device__ __forceinline__ uint64_t p8_desc_mn(uint32_t smem_addr) {
    return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)(P8_HALF >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}

__device__ __forceinline__ void p8_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(tc_smem_u32(bar)) : "memory");
}
// One lane of a warp that executes this together: 1 there, 0 in the others.
__device__ __forceinline__ uint32_t p8_elect() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(one));
    return one;
}
// Products and their commit by the thread whose `one` is not 0; the warp comes along. D[tmem] (+)= A[smem] B[smem]; A[tmem] B[smem].
__device__ __forceinline__ void p8_mma(uint32_t one, uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %5, 0;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
                 ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(one) : "memory");
}
__device__ __forceinline__ void p8_mma_p(uint32_t one, uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %5, 0;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
                 ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(one) : "memory");
}
__device__ __forceinline__ void p8_commit(uint32_t one, uint64_t* bar) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n"
                 ::"r"(tc_smem_u32(bar)), "r"(one) : "memory");
}
__device__ __forceinline__ unsigned p8_half2(float lo, float hi) {
    unsigned r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// 2^n for whole numbers -126 <= n <= 127 in a float, by its bits.
__device__ __forceinline__ float p8_power(float n) { return __int_as_float((__float_as_int(n + 12582912.f) + 127) << 23); }

__device__ __forceinline__ float p8_max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Pairs of floats in one instruction: x * c + add, and a + b.
__device__ __forceinline__ float2 p8_fma2(float2 x, float2 c, float2 add) {
    float2 r;
    asm("{\n\t.reg .b64 x, c, a, r;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 c, {%4, %5};\n\tmov.b64 a, {%6, %7};\n\t"
        "fma.rn.f32x2 r, x, c, a;\n\tmov.b64 {%0, %1}, r;\n\t}\n" : "=f"(r.x), "=f"(r.y) : "f"(x.x), "f"(x.y), "f"(c.x), "f"(c.y), "f"(add.x), "f"(add.y));
    return r;
}
__device__ __forceinline__ float2 p8_add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, r;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 r, x, y;\n\tmov.b64 {%0, %1}, r;\n\t}\n"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}

// All ones in the bytes that are no number (0x7f and 0xff).
__device__ __forceinline__ unsigned p8_no_number(unsigned w) { return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu; }

// Waits for this thread's tensor-memory loads. What they brought is named as changed by it: else the compiler may use the registers, which
// it takes to be loaded where the load stands, before the wait.
__device__ __forceinline__ void p8_wait_ld(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                   "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                   "+r"(r[28]) :: "memory");
    asm volatile("" : "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) :: "memory");
}

// The largest t and t + v of 32 scores (hidden ones are -inf). `scales`: of the 32 / BLOCK blocks they belong to, every BLOCK / 8th: the
// keys' scale, the exponent of the values' (-inf: a page that is missing).
template <int BLOCK> __device__ __forceinline__ void p8_top(const uint32_t (&x)[32], const float2* scales, float f, float& t_top, float& u_top, float& v_low) {
#pragma unroll
    for (int b = 0; b < 32; b += BLOCK) {
        const float2 s = scales[b / 8];
        float top = fmaxf(__uint_as_float(x[b]), __uint_as_float(x[b + 1]));
#pragma unroll
        for (int i = 2; i < BLOCK; i += 2) top = p8_max3(top, __uint_as_float(x[b + i]), __uint_as_float(x[b + i + 1]));
        const float t = s.y == -INFINITY ? -INFINITY : top * fmaxf(s.x * f, 1e-38f);
        t_top = fmaxf(t_top, t);
        u_top = fmaxf(u_top, t + s.y);
        v_low = fminf(v_low, s.y == -INFINITY ? INFINITY : s.y);
    }
}

// 32 scores -> 16 pairs of factors; returns the sum of their weights relative to 2^m.
template <int BLOCK>
__device__ __forceinline__ float p8_factors(const uint32_t (&x)[32], const float2* scales, float f, float m, float mu, uint32_t (&pk)[16]) {
    float l = 0.f;
#pragma unroll
    for (int b = 0; b < 32; b += BLOCK) {
        const float2 s = scales[b / 8];
        const float c = fmaxf(s.x * f, 1e-38f), add = s.y - mu;  // (not 0: a hidden score stays -inf)
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < BLOCK; i += 2) {
            const float2 u = p8_fma2(make_float2(__uint_as_float(x[b + i]), __uint_as_float(x[b + i + 1])), make_float2(c, c), make_float2(add, add));
            const float2 v = make_float2(fa_ex2(u.x), fa_ex2(u.y));
            sum = i == 0 ? v : p8_add2(sum, v);
            pk[(b + i) / 2] = p8_half2(v.x, v.y);
        }
        const float n = mu - m - s.y;                            // weight = factor * 2^n; beyond 2^100 they are p8_far's
        l = fmaf(sum.x + sum.y, n <= 100.f ? p8_power(fmaxf(n, -126.f)) : 0.f, l);
    }
    return l;
}

// The sum of the weights that p8_factors leaves out: factors too small for float32 although their weights are not.
template <int BLOCK> __device__ __forceinline__ float p8_far(const uint32_t (&x)[32], const float2* scales, float f, float m, float mu) {
    float l = 0.f;
#pragma unroll
    for (int b = 0; b < 32; b += BLOCK) {
        const float2 s = scales[b / 8];
        if (mu - m - s.y > 100.f && s.y > -INFINITY) {
            const float c = fmaxf(s.x * f, 1e-38f);
#pragma unroll
            for (int i = 0; i < BLOCK; ++i) l += fa_ex2(fmaf(__uint_as_float(x[b + i]), c, -m));
        }
    }
    return l;
}

template <int BOX>
__global__ void __launch_bounds__(P8_THREADS, 1)
prompt_kv8_kernel(const __grid_constant__ CUtensorMap map, const Prompt8Params p) {
    extern __shared__ unsigned char p8_raw[];
    __shared__ __align__(8) uint64_t raw_full[2][P8_STAGES], raw_free[2][P8_STAGES], k_full[2], k_free[2], v_full, v_free, s_full[2], p_full[2][2], o_done[2];
    __shared__ __align__(16) float2 scales[P8_SLOTS][16];
    __shared__ __align__(16) unsigned no_number[P8_SLOTS][4];            // keys of a tile whose values hold NaN
    __shared__ uint32_t tmem_slot;
    const uint32_t raw_addr = tc_smem_u32(p8_raw);
    unsigned char* Qs = p8_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);     // [2 tiles][2 halves][128 rows][128 bytes]
    unsigned char* Ks = Qs + 4 * P8_HALF;                        // [2 key tiles][2 halves][128 keys][128 bytes]
    unsigned char* Vs = Ks + 4 * P8_HALF;                        // [2 halves][128 keys][128 bytes]
    unsigned char* raw = Vs + 2 * P8_HALF;                       // [keys, values][P8_STAGES][128 keys][128 bytes]

    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);      // (known to be one number for the warp: the roles do not diverge)
    if (warp == 8 && lane == 0) {
        for (int i = 0; i < P8_STAGES; ++i) {
            mbar_init(&raw_full[0][i], 2);                       // the boxes, and the scales
            mbar_init(&raw_full[1][i], 1);
            mbar_init(&raw_free[0][i], P8_UNPACK);
            mbar_init(&raw_free[1][i], P8_UNPACK);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], P8_UNPACK);
            mbar_init(&k_free[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i][0], 4);
            mbar_init(&p_full[i][1], 4);
            mbar_init(&o_done[i], 1);
        }
        mbar_init(&v_full, P8_UNPACK);
        mbar_init(&v_free, 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&map) : "memory");
    }
    if (warp == 15) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tc_smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    pdl_trigger();
    pdl_wait();

    // ---- what the item is ----
    const int4 item = reinterpret_cast<const int4*>(p.items)[blockIdx.x / (unsigned)p.nkv];
    const int kvh = (int)(blockIdx.x % (unsigned)p.nkv), r = item.x, tok0 = item.y, part = item.z & 0xffff, parts = item.z >> 16;
    const int G = p.nq / p.nkv;
    const int q_begin = p.q_start[r], q_len = p.q_start[r + 1] - q_begin;
    const int ctx = min(p.ctx_len[r], p.table_stride << p.page_shift), pos0 = p.ctx_len[r] - q_len;
    const int ntok = min(q_len - tok0, p.tokens);
    const int rows = ntok * G;
    const int* table = p.block_tables + (size_t)r * p.table_stride;
    // keys of the whole row tile, and this part's tiles of them; a row tile of 128 rows sees none beyond its last row's position
    const int low = p.window > 0 ? max(pos0 + tok0 - p.window + 1, 0) : 0;
    const int tile0 = low / P8_KEYS, all_tiles = (pos0 + tok0 + ntok - 1) / P8_KEYS + 1 - tile0;
    const int each = all_tiles / parts, more = all_tiles - each * parts;         // the first `more` parts have one more
    const int t_begin = tile0 + each * part + min(part, more), t_end = t_begin + each + (part < more);
    int n[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int last_row = min(rows, (t + 1) * P8_ROWS) - 1;   // of the tile; below its first: the tile has no rows
        n[t] = last_row < t * P8_ROWS ? 0 : max(min(t_end, (pos0 + tok0 + last_row / G) / P8_KEYS + 1) - t_begin, 0);
    }
    const int tiles = max(n[0], n[1]);

    // ---- a softmax thread's row: its queries into shared memory ----
    const int mine = warp >> 2, row = tid & (P8_ROWS - 1);       // row tile and row, of warps 0 .. 7
    float f = 0.f;
    if (warp < 8) {
        const int index = mine * P8_ROWS + row;
        uint4 v[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) v[c] = make_uint4(0u, 0u, 0u, 0u);
        if (index < rows) {
            const uint4* q = reinterpret_cast<const uint4*>(p.q + (size_t)(q_begin + tok0 + index / G) * p.q_stride + (size_t)(kvh * G + index % G) * P8_D);
#pragma unroll
            for (int c = 0; c < 16; ++c) v[c] = q[c];
        }
        float amax = 0.f;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
            const unsigned w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
        }
        int e = (int)(__float_as_uint(amax) >> 23);              // 2^(e - 127) <= amax < 2^(e - 126)
        e = e < 1 ? 1 : (e > 253 ? 253 : e);
        const float down = p.scale < 0.f ? -kv8_power(127 - e) : kv8_power(127 - e);
        f = fabsf(p.scale) * 1.4426950408889634f * kv8_power(e - 127);
        unsigned char* to = Qs + (size_t)mine * 2 * P8_HALF + row * 128;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
            const unsigned w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
            unsigned h[4];
#pragma unroll
            for (int i = 0; i < 4; i += 2) {                     // entries 0, 2 and 1, 3 of four, as the keys are unpacked
                h[i] = p8_half2(__uint_as_float(w[i] << 16) * down, __uint_as_float(w[i + 1] << 16) * down);
                h[i + 1] = p8_half2(__uint_as_float(w[i] & 0xffff0000u) * down, __uint_as_float(w[i + 1] & 0xffff0000u) * down);
            }
            *reinterpret_cast<uint4*>(to + (c >> 3) * P8_HALF + (((c & 7) ^ (row & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    }
    fa_fence_before();
    __syncthreads();
    fa_fence_after();
    const uint32_t tmem = tmem_slot;                             // S of the tiles in columns 0 and 128, O in 256 and 384

    if (warp == 15) {
        // ---- products: the whole warp walks along, one thread issues (addresses then stay in uniform registers: with the
        // loop in one thread's branch eight products took 450 to 950 clocks to issue, a third of a key tile's time) ----
        constexpr uint32_t idesc_s = p8_idesc(P8_ROWS, P8_KEYS), idesc_o = p8_idesc(P8_ROWS, P8_D) | (1u << 16);      // V is MN-major
        const uint32_t one = p8_elect();
        // (an operand further on in shared memory: its address in units of 16 bytes, in the descriptor's low bits)
        const uint64_t q_desc = umma_desc(tc_smem_u32(Qs)), k_desc = umma_desc(tc_smem_u32(Ks)), v_desc = p8_desc_mn(tc_smem_u32(Vs));
        const int last_t = n[1] > 0 ? 1 : 0;
        // S of row tile t and key tile j; the first of the row tiles waits for the keys, the last frees them
        auto scores = [&](int t, int j) {
            if (t == 0 || j >= n[0]) mbar_wait(&k_full[j & 1], (j >> 1) & 1, p.error_flag);
            // S lies where the P of the key tile before is: products into other columns keep no order among themselves
            if (j > 0) mbar_wait(&o_done[t], (j - 1) & 1, p.error_flag);
            fa_fence_after();
            const uint64_t q_at = q_desc + (uint32_t)t * (2 * P8_HALF >> 4), k_at = k_desc + (uint32_t)(j & 1) * (2 * P8_HALF >> 4);
#pragma unroll
            for (int k = 0; k < P8_D / 16; ++k) {
                const uint32_t off = ((uint32_t)(k >> 2) * P8_HALF + (uint32_t)(k & 3) * 32) >> 4;
                p8_mma(one, tmem + t * 128, q_at + off, k_at + off, idesc_s, k != 0 ? 1u : 0u);
            }
            p8_commit(one, &s_full[t]);
            if (t == last_t || (t == 0 && j >= n[1])) p8_commit(one, &k_free[j & 1]);
        };
#pragma unroll 1
        for (int j = -1; j < tiles; ++j) {
#pragma unroll 1
            for (int t = 0; t < 2; ++t) {
                const int count = t == 0 ? n[0] : n[1];
                if (j >= count) continue;
                if (j < 0) {
                    if (count > 0) scores(t, 0);
                    continue;
                }
                if (t == 0 || j >= n[0]) mbar_wait(&v_full, j & 1, p.error_flag);
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    mbar_wait(&p_full[t][half], j & 1, p.error_flag);
                    fa_fence_after();
#pragma unroll
                    for (int k = 0; k < P8_KEYS / 32; ++k)       // 16 keys a product: 8 columns of P, 2 KB of V
                        p8_mma_p(one, tmem + 256 + t * 128, tmem + t * 128 + half * 32 + k * 8, v_desc + (uint32_t)((half * 4 + k) * 2048 >> 4), idesc_o, (j | half | k) != 0 ? 1u : 0u);
                }
                p8_commit(one, &o_done[t]);
                if (t == last_t || (t == 0 && j >= n[1])) p8_commit(one, &v_free);
                if (j + 1 < count) scores(t, j + 1);
            }
        }
    } else if (warp == 14) {
        // ---- loads: lane b < 16 sees to block b of eight keys; page numbers are asked for two tiles before their boxes, scale bytes one ----
        const bool boxes = lane < 16 && (lane * 8) % BOX == 0;
        const size_t body = (size_t)2 * p.nkv * p.page_size * P8_D;
        auto find = [&](int j) {
            const int key = (t_begin + j) * P8_KEYS + lane * 8;
            return j < tiles && lane < 16 && key < ctx ? table[key >> p.page_shift] : -1;
        };
        unsigned ek = 0u, ev = 0u;
        auto ask = [&](int& page) {
            if (page >= p.num_pages) page = -1;
            if (page >= 0) {
                const unsigned char* at = p.pages + (size_t)page * p.page_bytes + body + kvh;
                ek = at[0];
                ev = at[p.nkv];
            }
        };
        // one tile's keys or values; out of range: the box arrives as zeros
        auto load = [&](int kv, int j, int page) {
            const int stage = j % P8_STAGES;
            if (j >= P8_STAGES) mbar_wait(&raw_free[kv][stage], (j / P8_STAGES - 1) & 1, p.error_flag);
            if (lane == 0) mbar_expect_tx(&raw_full[kv][stage], P8_RAW);
            __syncwarp();
            if (boxes)
                p8_load_box(raw + (kv * P8_STAGES + stage) * P8_RAW + lane * 8 * P8_D, &map, ((t_begin + j) * P8_KEYS + lane * 8) & (p.page_size - 1), kvh, kv,
                            page >= 0 ? page : p.num_pages, &raw_full[kv][stage]);
        };
        int now = find(0), next = find(1), before = -1;
        ask(now);
#pragma unroll 1
        for (int j = 0; tiles > 0 && j <= tiles; ++j) {          // in the order in which they are unpacked: keys a tile ahead of values
            if (j < tiles) {
                const int after = find(j + 2);
                load(0, j, now);
                if (lane < 16)                                   // (a block of zeros may have any scale; the operands are 2^-8 of the bytes' values)
                    scales[j % P8_SLOTS][lane] = now >= 0 ? make_float2((ek == 0u ? 1.f : kv8_scale(ek)) * 256.f, (float)((int)ev - 119)) : make_float2(1.f, -INFINITY);
                if (lane < 4) no_number[j % P8_SLOTS][lane] = 0u;
                __syncwarp();
                if (lane == 0) p8_arrive(&raw_full[0][j % P8_STAGES]);
                if (j > 0) load(1, j - 1, before);
                before = now;
                now = next;
                next = after;
                ask(now);
            } else {
                load(1, j - 1, before);
            }
        }
    } else if (warp >= 8) {
        // ---- unpacking ----
        // Eight lanes take a key: lane c of them its entries 16 c .. 16 c + 15.
        const int first = tid - 256, piece = first & 7, half = piece >> 2, at = (piece & 3) * 2;
        // Keys are unpacked a tile ahead of values: K 0, K 1, V 0, K 2, V 1 .. : a tile's keys then wait for nobody, and its
        // values are due only when its softmax is done.
#pragma unroll 1
        for (int step = 0; step <= 2 * tiles; ++step) {
            const int kv = step > 0 && (step & 1) == 0, j = kv ? step / 2 - 1 : (step + 1) / 2;
            if (j == tiles) continue;
            const unsigned char* src = raw + (kv * P8_STAGES + j % P8_STAGES) * P8_RAW;
            const float2* of = scales[j % P8_SLOTS];
            mbar_wait(&raw_full[kv][j % P8_STAGES], j / P8_STAGES & 1, p.error_flag);
            const int there = ctx - (t_begin + j) * P8_KEYS;     // keys of the tile that exist
            const bool whole = there >= P8_KEYS && __all_sync(0xffffffffu, of[lane & 15].y > -INFINITY);
            if (kv == 0 && j > 1) mbar_wait(&k_free[j & 1], ((j >> 1) - 1) & 1, p.error_flag);
            if (kv == 1 && j > 0) mbar_wait(&v_free, (j - 1) & 1, p.error_flag);
            unsigned char* dst = (kv == 0 ? Ks + (j & 1) * 2 * P8_HALF : Vs) + half * P8_HALF;
#pragma unroll 1
            for (int key0 = first >> 3; key0 < P8_KEYS; key0 += P8_PIECES * P8_UNPACK * 4) {
                uint4 w[P8_PIECES];
                unsigned any = 0u;
#pragma unroll
                for (int u = 0; u < P8_PIECES; ++u) {
                    const int key = key0 + u * P8_UNPACK * 4;
                    w[u] = make_uint4(0u, 0u, 0u, 0u);
                    if (key < P8_KEYS) w[u] = *reinterpret_cast<const uint4*>(src + key * P8_D + ((piece ^ (key & 7)) << 4));
                }
                if (!whole) {
#pragma unroll
                    for (int u = 0; u < P8_PIECES; ++u) {        // not there: zeros, for factors of zero
                        const int key = key0 + u * P8_UNPACK * 4;
                        if (key >= there || of[min(key, P8_KEYS - 1) / 8].y == -INFINITY) w[u] = make_uint4(0u, 0u, 0u, 0u);
                    }
                }
#pragma unroll
                for (int u = 0; u < P8_PIECES; ++u)
                    any |= ((w[u].x & 0x7f7f7f7fu) + 0x01010101u) | ((w[u].y & 0x7f7f7f7fu) + 0x01010101u) | ((w[u].z & 0x7f7f7f7fu) + 0x01010101u) |
                           ((w[u].w & 0x7f7f7f7fu) + 0x01010101u);
                if (__builtin_expect(any & 0x80808080u, 0)) {            // what is no number: zeros as values, and the key is noted
#pragma unroll 1
                    for (int u = 0; u < P8_PIECES; ++u) {
                        const int key = key0 + u * P8_UNPACK * 4;
                        uint4 x = u == 0 ? w[0] : u == 1 ? w[1] : w[2];
                        const unsigned bad[4] = {p8_no_number(x.x), p8_no_number(x.y), p8_no_number(x.z), p8_no_number(x.w)};
                        if ((bad[0] | bad[1] | bad[2] | bad[3]) == 0u) continue;
                        x = make_uint4(x.x & ~bad[0], x.y & ~bad[1], x.z & ~bad[2], x.w & ~bad[3]);
                        if (u == 0) w[0] = x;
                        if (u == 1) w[1] = x;
                        if (u == 2) w[2] = x;
                        atomicOr(&no_number[j % P8_SLOTS][key >> 5], 1u << (key & 31));
                    }
                }
#pragma unroll
                for (int u = 0; u < P8_PIECES; ++u) {
                    const int key = key0 + u * P8_UNPACK * 4;
                    const unsigned b[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
                    unsigned h[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {                // a byte seeeemmm is s0eeeemmm0000000 in half precision, times 2^8; of four bytes the pairs 0, 2 and 1, 3
                        h[2 * i] = ((b[i] << 7) & 0x3f803f80u) | ((b[i] << 8) & 0x80008000u);
                        h[2 * i + 1] = ((b[i] >> 1) & 0x3f803f80u) | (b[i] & 0x80008000u);
                    }
                    // (lanes of the second half of the head store their second piece first: the halves lie in the same banks)
                    const uint4 lo = make_uint4(h[0], h[1], h[2], h[3]), hi = make_uint4(h[4], h[5], h[6], h[7]);
                    if (key < P8_KEYS) {
                        *reinterpret_cast<uint4*>(dst + key * 128 + (((at + half) ^ (key & 7)) << 4)) = half ? hi : lo;
                        *reinterpret_cast<uint4*>(dst + key * 128 + (((at + 1 - half) ^ (key & 7)) << 4)) = half ? lo : hi;
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                p8_arrive(kv == 0 ? &k_full[j & 1] : &v_full);
                p8_arrive(&raw_free[kv][j % P8_STAGES]);
            }
        }
    } else {
        // ---- softmax ----
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + mine * 128, to = tmem + lanes + 256 + mine * 128;
        const int index = mine * P8_ROWS + row;
        const bool live = index < rows;
        const int pos = live ? pos0 + tok0 + index / G : -1;     // -1: a row that does not exist sees nothing
        const int first = p.window > 0 ? pos - p.window + 1 : 0;
        // positions of the tile's first and last row: what no key tile has to be masked for
        const int pos_first = pos0 + tok0 + mine * P8_ROWS / G, pos_last = pos0 + tok0 + (min(rows, (mine + 1) * P8_ROWS) - 1) / G;
        float m = -INFINITY, mu = -INFINITY, l = 0.f;
        const int count = n[mine];
        uint32_t x[32], y[32], pk[16];
        constexpr int BLOCK = BOX;
        for (int j = 0; j < count; ++j) {
            const int j0 = (t_begin + j) * P8_KEYS;
            const float2* of = scales[j % P8_SLOTS];
            const bool mask = j0 + P8_KEYS - 1 > pos_first || (p.window > 0 && j0 < pos_last - p.window + 1) || rows < (mine + 1) * P8_ROWS;
            mbar_wait(&s_full[mine], j & 1, p.error_flag);       // P V of the key tile before is done as well: it was issued before
            fa_fence_after();
            if (mask) {                                          // what is hidden is written over S, once
#pragma unroll 1
                for (int c = 0; c < P8_KEYS; c += 32) {
                    FA_TMEM_LD32(ts + c, x, 0);
                    p8_wait_ld(x);
                    fa_mask32(x, j0 + c, pos, first);
                    FA_TMEM_ST32(ts + c, x, 0);
                }
                fa_tmem_wait_st();
            }
            float t_top = -INFINITY, u_top = -INFINITY, v_low = INFINITY;
#pragma unroll 1
            for (int c = 0; c < P8_KEYS; c += 64) {
                FA_TMEM_LD32(ts + c, x, 0);
                p8_wait_ld(x);
                FA_TMEM_LD32(ts + c + 32, y, 0);
                p8_top<BLOCK>(x, of + c / 8, f, t_top, u_top, v_low);
                p8_wait_ld(y);
                p8_top<BLOCK>(y, of + c / 8 + 4, f, t_top, u_top, v_low);
            }
            if (t_top > m + 12.f) {
                const float to_m = ceilf(t_top);
                l *= m == -INFINITY ? 0.f : fa_ex2(m - to_m);
                m = to_m;
            }
            float alpha = 1.f;
            const bool raise = u_top > mu + 12.f;
            if (raise) {
                const float to_mu = ceilf(u_top);
                alpha = fa_ex2(mu - to_mu);                      // 0 the first time
                mu = to_mu;
            }
            if (j > 0 && __any_sync(0xffffffffu, raise)) {
#pragma unroll 1
                for (int c = 0; c < P8_D; c += 32) {
                    FA_TMEM_LD32(to + c, x, 0);
                    p8_wait_ld(x);
#pragma unroll
                    for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * alpha);
                    FA_TMEM_ST32(to + c, x, 0);
                }
            }
            const float m_now = m == -INFINITY ? 0.f : m, mu_now = mu == -INFINITY ? 0.f : mu;
            if (__any_sync(0xffffffffu, mu_now - m_now - v_low > 100.f)) {
#pragma unroll 1
                for (int c = 0; c < P8_KEYS; c += 32) {
                    FA_TMEM_LD32(ts + c, x, 0);
                    p8_wait_ld(x);
                    l += p8_far<BLOCK>(x, of + c / 8, f, m_now, mu_now);
                }
            }
#pragma unroll 1
            for (int c = 0; c < P8_KEYS; c += 32) {
                FA_TMEM_LD32(ts + c, x, 0);
                p8_wait_ld(x);
                l += p8_factors<BLOCK>(x, of + c / 8, f, m_now, mu_now, pk);
                FA_TMEM_ST16(ts + c / 2, pk);
                if (c & 32) {                                    // half of the keys: their product may begin (661 -> 657 us)
                    fa_tmem_wait_st();
                    fa_fence_before();
                    __syncwarp();
                    if (lane == 0) p8_arrive(&p_full[mine][c >> 6]);
                }
            }
            // values that are no number: looked at once the tile's values are unpacked, which the next wait stands behind
            if (j > 0) {
                const int before = (j - 1) % P8_SLOTS, k0 = j0 - P8_KEYS;
                const uint4 bad = *reinterpret_cast<const uint4*>(no_number[before]);
                if (__builtin_expect((bad.x | bad.y | bad.z | bad.w) != 0u, 0)) {
#pragma unroll 1
                    for (int i = 0; i < P8_KEYS; ++i)
                        if ((no_number[before][i >> 5] >> (i & 31) & 1u) && k0 + i >= first && k0 + i <= pos) l = __int_as_float(0x7fffffff);
                }
            }
        }
        if (count > 0) mbar_wait(&o_done[mine], (count - 1) & 1, p.error_flag);
        fa_fence_after();
        if (count > 0) {
            const int before = (count - 1) % P8_SLOTS, k0 = (t_begin + count - 1) * P8_KEYS;
            const uint4 bad = *reinterpret_cast<const uint4*>(no_number[before]);
            if ((bad.x | bad.y | bad.z | bad.w) != 0u) {
#pragma unroll 1
                for (int i = 0; i < P8_KEYS; ++i)
                    if ((no_number[before][i >> 5] >> (i & 31) & 1u) && k0 + i >= first && k0 + i <= pos) l = __int_as_float(0x7fffffff);
            }
        }
        const float inv = l == 0.f ? 0.f : exp2f(mu - m) / l;    // no keys: zeros
        bf16* out = p.out + (size_t)(q_begin + tok0 + (live ? index / G : 0)) * p.out_stride + (size_t)(kvh * G + index % G) * P8_D;
        uint32_t a[32];
        float* sums = p.partials + (((size_t)item.w * p.nkv + kvh) * (2 * P8_ROWS) + index) * P8_PART;
#pragma unroll
        for (int c = 0; c < P8_D; c += 32) {
            if (count > 0) {
                FA_TMEM_LD32(to + c, a, 0);
                p8_wait_ld(a);
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) a[i] = 0u;
            }
            if (!live) continue;
#pragma unroll
            for (int i = 0; i < 32; i += 4) {                    // columns 0, 2, 1, 3 of four, as the values are unpacked
                const uint32_t swapped = a[i + 1];
                a[i + 1] = a[i + 2];
                a[i + 2] = swapped;
            }
            if (parts == 1) {
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    uint4 v;
                    v.x = fa_pack(__uint_as_float(a[i]) * inv, __uint_as_float(a[i + 1]) * inv);
                    v.y = fa_pack(__uint_as_float(a[i + 2]) * inv, __uint_as_float(a[i + 3]) * inv);
                    v.z = fa_pack(__uint_as_float(a[i + 4]) * inv, __uint_as_float(a[i + 5]) * inv);
                    v.w = fa_pack(__uint_as_float(a[i + 6]) * inv, __uint_as_float(a[i + 7]) * inv);
                    *reinterpret_cast<uint4*>(out + c + i) = v;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(sums + c + i) = make_uint4(a[i], a[i + 1], a[i + 2], a[i + 3]);
            }
        }
        if (live && parts > 1) *reinterpret_cast<float4*>(sums + P8_D) = make_float4(m, mu, l, 0.f);
    }
    fa_fence_before();
    __syncthreads();
    if (warp == 15) {
        fa_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
    }
}

// Weight of a part's sum under a common maximum. One without a finite score has -inf: it is 0, or no number.
__device__ __forceinline__ float p8_weight(float m, float common) { return m == -INFINITY ? 1.f : fa_ex2(m - common); }

// A row of a row tile whose keys came in parts, a warp each: the parts' sums in order. `shared` [n][4]: request, first token, parts, first place.
__global__ void __launch_bounds__(256) prompt_kv8_merge_kernel(const Prompt8Params p, const int* shared) {
    pdl_trigger();
    pdl_wait();
    const int4 of = reinterpret_cast<const int4*>(shared)[blockIdx.y];
    const int kvh = blockIdx.z, index = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int G = p.nq / p.nkv, q_begin = p.q_start[of.x], ntok = min(p.q_start[of.x + 1] - q_begin - of.y, p.tokens);
    if (index >= ntok * G) return;
    auto sums = [&](int part) { return p.partials + (((size_t)(of.w + part) * p.nkv + kvh) * (2 * P8_ROWS) + index) * P8_PART; };
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, mu = -INFINITY, l = 0.f;
    for (int p0 = 0; p0 < of.z; p0 += 4) {                       // four parts on their way together
        float4 v[4], s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            s[i] = make_float4(-INFINITY, -INFINITY, 0.f, 0.f);
            if (p0 + i < of.z) {
                v[i] = __ldcg(reinterpret_cast<const float4*>(sums(p0 + i)) + lane);
                s[i] = __ldcg(reinterpret_cast<const float4*>(sums(p0 + i) + P8_D));
            }
        }
        const float m_new = fmaxf(fmaxf(fmaxf(s[0].x, s[1].x), fmaxf(s[2].x, s[3].x)), m);
        const float mu_new = fmaxf(fmaxf(fmaxf(s[0].y, s[1].y), fmaxf(s[2].y, s[3].y)), mu);
        l *= p8_weight(m, m_new);
        const float old = p8_weight(mu, mu_new);
        o.x *= old; o.y *= old; o.z *= old; o.w *= old;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            l = fmaf(s[i].z, p8_weight(s[i].x, m_new), l);
            const float w = p8_weight(s[i].y, mu_new);
            o.x = fmaf(v[i].x, w, o.x); o.y = fmaf(v[i].y, w, o.y); o.z = fmaf(v[i].z, w, o.z); o.w = fmaf(v[i].w, w, o.w);
        }
        m = m_new;
        mu = mu_new;
    }
    const float inv = l == 0.f ? 0.f : exp2f(mu - m) / l;
    bf16* out = p.out + (size_t)(q_begin + of.y + index / G) * p.out_stride + (size_t)(kvh * G + index % G) * P8_D + lane * 4;
    *reinterpret_cast<uint2*>(out) = make_uint2(fa_pack(o.x * inv, o.y * inv), fa_pack(o.z * inv, o.w * inv));
}

// ---- host side ---------------------------------------------------------------------------------------------------------------
LLMP_API int llmp_kv8_prompt_supports(int nq, int nkv, int d, int page_size) {
    return d == P8_D && nq > 0 && nkv > 0 && nq % nkv == 0 && nq / nkv <= P8_ROWS && page_size >= 8 && (page_size & (page_size - 1)) == 0;
}
// Query tokens of an item, and floats of a place for its sums (all key/value heads).
LLMP_API int llmp_kv8_prompt_tokens(int nq, int nkv) { return nkv <= 0 || nq < nkv ? 0 : 2 * P8_ROWS / (nq / nkv); }
LLMP_API long llmp_kv8_prompt_place_floats(int nkv) { return (long)nkv * 2 * P8_ROWS * P8_PART; }

// items: [num_items][4] as in Prompt8Params; shared: [num_shared][4] as in prompt_kv8_merge_kernel; partials: the items' places.
LLMP_API int llmp_kv8_prompt(const void* q, long q_stride, void* out, long out_stride, const void* pages, int num_pages, const int* block_tables,
                             int table_stride, const int* q_start, const int* ctx_len, const int* items, int num_items, const int* shared,
                             int num_shared, float* partials, int nq, int nkv, int page_size, int window, float scale, int* error_flag,
                             cudaStream_t stream) {
    if (num_items <= 0) return 0;
    LLMP_REQUIRE(llmp_kv8_prompt_supports(nq, nkv, P8_D, page_size), "kv8 prompt attention: %d and %d heads, pages of %d tokens are not for this kernel", nq, nkv, page_size);
    LLMP_REQUIRE((q_stride % 8) == 0 && (out_stride % 8) == 0 && ((size_t)q % 16) == 0 && ((size_t)out % 16) == 0 && ((size_t)pages % 16) == 0 &&
                 ((size_t)items % 16) == 0 && ((size_t)shared % 16) == 0, "kv8 prompt attention: rows and lists must be 16-byte aligned");
    LLMP_REQUIRE(error_flag != nullptr && num_pages > 0 && table_stride > 0, "kv8 prompt attention: an error flag, pages and tables are needed");
    LLMP_REQUIRE(num_shared == 0 || (partials != nullptr && shared != nullptr), "kv8 prompt attention: shared items need places for their sums");
    LLMP_REQUIRE((long)num_items * nkv < (1L << 31) && num_shared <= 65535 && nkv <= 65535, "kv8 prompt attention: too many items");
    Prompt8Params p;
    p.q = (const bf16*)q; p.out = (bf16*)out; p.pages = (const unsigned char*)pages; p.block_tables = block_tables; p.q_start = q_start;
    p.ctx_len = ctx_len; p.items = items; p.partials = partials; p.q_stride = q_stride; p.out_stride = out_stride;
    p.page_bytes = kv8_page_bytes(nkv, page_size, P8_D); p.table_stride = table_stride; p.num_pages = num_pages; p.nq = nq; p.nkv = nkv;
    p.page_size = page_size; p.page_shift = 31 - __builtin_clz((unsigned)page_size); p.window = window; p.tokens = llmp_kv8_prompt_tokens(nq, nkv);
    p.scale = scale; p.error_flag = error_flag;
    const int box_tokens = page_size < 32 ? page_size : 32;
    EncodeTiledFn encode = llmp_tensor_map_encoder();
    LLMP_REQUIRE(encode != nullptr, "kv8 prompt attention: the driver does not provide cuTensorMapEncodeTiled");
    CUtensorMap map;
    const cuuint64_t row = P8_D, plane = row * page_size;
    const cuuint64_t dims[5] = {P8_D, (cuuint64_t)page_size, (cuuint64_t)nkv, 2, (cuuint64_t)num_pages};
    const cuuint64_t strides[4] = {row, plane, plane * nkv, (cuuint64_t)p.page_bytes};
    const cuuint32_t box[5] = {P8_D, (cuuint32_t)box_tokens, 1, 1, 1};
    const cuuint32_t elem[5] = {1, 1, 1, 1, 1};
    const CUresult rc = encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, const_cast<void*>(pages), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    LLMP_REQUIRE(rc == CUDA_SUCCESS, "kv8 prompt attention: cuTensorMapEncodeTiled failed with code %d", (int)rc);
    const size_t smem = 10 * (size_t)P8_HALF + 2 * P8_STAGES * (size_t)P8_RAW + 1024;
    const auto kernel = box_tokens == 8 ? prompt_kv8_kernel<8> : box_tokens == 16 ? prompt_kv8_kernel<16> : prompt_kv8_kernel<32>;
    if (box_tokens == 8) LLMP_ALLOW_SMEM(prompt_kv8_kernel<8>, smem);
    else if (box_tokens == 16) LLMP_ALLOW_SMEM(prompt_kv8_kernel<16>, smem);
    else LLMP_ALLOW_SMEM(prompt_kv8_kernel<32>, smem);
    llmp_launch_dependent(kernel, dim3((unsigned)num_items * nkv), dim3(P8_THREADS), smem, stream, map, p);
    if (num_shared > 0) llmp_launch_dependent(prompt_kv8_merge_kernel, dim3(2 * P8_ROWS / 8, num_shared, nkv), dim3(256), 0, stream, p, shared);
    return llmp_check_launch("kv8_prompt");
}
