// Attention of single tokens over pages of 8-bit keys and values (kv8.cuh): row r of q belongs to request r, at position
// ctx_len[r] - 1. This file holds the kernel that takes every size and either type of q, on the CUDA cores, and the entry point.
//
//   o = sum_j w_j v_j / sum_j w_j,   w_j = exp(scale q.k_j - m),   k_j = 2^(ek - 127) * bytes, v_j = 2^(ev - 127) * bytes
//
// Keys are cut into splits of the same number of keys for all requests; block (split, key/value head and heads of its group,
// request) walks its split in tiles of 64 keys with a running maximum and sum and leaves an unnormalised partial, which
// kv8_merge_kernel adds up in the order of the splits. The scales are applied in float32: to the score for a key, to the
// weight for a value. What bounds it: the tiles of a split follow one another, and the merge is a launch (4 requests of up to 700
// tokens in float32, a window of 333, 6 and 2 heads of 80: 8.9 us); the sizes that are served most have the streaming kernel.
#include "kv8.cuh"

#define D8_TILE 64
#define D8_THREADS 128
#define D8_MAX_HEADS 8                               // query heads per block
#define D8_MAX_ACC 8                                 // column pairs per thread
#define D8_MAX_SPLITS 1024

struct Decode8Params {
    const void* q;
    const unsigned char* pages;
    const int* block_tables;
    const int* ctx_len;
    float* part_o;                                   // [R, nq, splits, d]
    float* part_ml;                                  // [R, nq, splits, 2]
    long q_stride, page_bytes;
    int table_stride, num_pages, max_ctx;
    int nq, nkv, d, page_size, window;
    int heads_per_block, head_chunks, splits, split_keys;
    float scale;
};

__device__ __forceinline__ void d8_copy16(void* smem_dst, const void* src, bool valid) {
    const unsigned dst = (unsigned)__cvta_generic_to_shared(smem_dst);
    const int bytes = valid ? 16 : 0;                // 0: nothing is read, the 16 bytes become zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// The context the kernels see: never beyond what the tables and the launch's bound hold.
__device__ __forceinline__ int d8_context(const int* ctx_len, int r, int max_ctx) {
    const int ctx = ctx_len[r];
    return ctx < 0 ? 0 : (ctx < max_ctx ? ctx : max_ctx);
}

template <typename T>
__global__ void __launch_bounds__(D8_THREADS) decode_kv8_kernel(const Decode8Params p) {
    extern __shared__ __align__(16) unsigned char d8_smem[];
    const int d = p.d, kstride = d + 16;                         // padded key row: rows begin in different banks
    unsigned char* Ks = d8_smem;                                 // [64][kstride]
    unsigned char* Vs = Ks + D8_TILE * kstride;                  // [64][d]
    float* Qs = reinterpret_cast<float*>(Vs + D8_TILE * d);      // [heads][d]
    float* Ss = Qs + D8_MAX_HEADS * d;                           // [heads][64]
    __shared__ float k_scale[D8_TILE], v_scale[D8_TILE];
    __shared__ long long key_off[D8_TILE];                       // offset of the key's row, or -1
    __shared__ float row_m[D8_MAX_HEADS], row_l[D8_MAX_HEADS], row_a[D8_MAX_HEADS];
    pdl_trigger();
    pdl_wait();

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int kvh = blockIdx.y / p.head_chunks, chunk = blockIdx.y % p.head_chunks;
    const int r = blockIdx.z, G = p.nq / p.nkv, head0 = chunk * p.heads_per_block;
    const int heads = min(G - head0, p.heads_per_block);
    const int ctx = d8_context(p.ctx_len, r, p.max_ctx);
    int lo = blockIdx.x * p.split_keys;
    if (lo >= ctx) return;
    const int hi = min(lo + p.split_keys, ctx);
    if (p.window > 0) lo = max(lo, ctx - p.window);              // may pass hi: an empty split
    const T* q = reinterpret_cast<const T*>(p.q) + (size_t)r * p.q_stride + (size_t)(kvh * G + head0) * d;
    const int* table = p.block_tables + (size_t)r * p.table_stride;
    const size_t plane = (size_t)p.nkv * p.page_size * d;        // from a key's row to the value's
    const int pieces = d / 16;

    for (int e = tid; e < heads * d; e += D8_THREADS) Qs[e] = to_float(q[e]);
    if (tid < D8_MAX_HEADS) {
        row_m[tid] = -INFINITY;
        row_l[tid] = 0.f;
    }
    float acc[D8_MAX_ACC][2];
#pragma unroll
    for (int i = 0; i < D8_MAX_ACC; ++i) acc[i][0] = acc[i][1] = 0.f;
    const int pairs = heads * d / 2;

    for (int j0 = lo / D8_TILE * D8_TILE; j0 < hi; j0 += D8_TILE) {
        __syncthreads();                                         // the tile before is read
        if (tid < D8_TILE) {
            const int j = j0 + tid;
            const int page = j >= lo && j < hi ? table[j / p.page_size] : -1;
            const bool there = page >= 0 && page < p.num_pages;
            const size_t base = (size_t)(there ? page : 0) * p.page_bytes;
            key_off[tid] = there ? (long long)(base + ((size_t)kvh * p.page_size + j % p.page_size) * d) : -1;
            k_scale[tid] = there ? kv8_scale(p.pages[base + 2 * plane + kvh]) : 0.f;
            v_scale[tid] = there ? kv8_scale(p.pages[base + 2 * plane + p.nkv + kvh]) : 0.f;
        }
        __syncthreads();
        for (int e = tid; e < D8_TILE * pieces; e += D8_THREADS) {
            const int key = e / pieces, c = (e % pieces) * 16;
            const long long off = key_off[key];
            const unsigned char* src = off >= 0 ? p.pages + off + c : p.pages;
            d8_copy16(Ks + key * kstride + c, src, off >= 0);
            d8_copy16(Vs + key * d + c, off >= 0 ? src + plane : src, off >= 0);
        }
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;\n" ::: "memory");
        __syncthreads();
        {                                                        // scores: thread -> key tid % 64, every other head
            const int key = tid % D8_TILE;
            for (int h = tid / D8_TILE; h < heads; h += D8_THREADS / D8_TILE) {
                const unsigned char* krow = Ks + key * kstride;
                const float* qrow = Qs + h * d;
                float s = 0.f;
                for (int c = 0; c < d; c += 16) {
                    const uint4 raw = *reinterpret_cast<const uint4*>(krow + c);
                    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float f[4];
                        kv8_unpack4(w[i], f);
#pragma unroll
                        for (int j = 0; j < 4; ++j) s = fmaf(qrow[c + 4 * i + j], f[j], s);
                    }
                }
                Ss[h * D8_TILE + key] = key_off[key] >= 0 ? s * k_scale[key] * p.scale : -INFINITY;
            }
        }
        __syncthreads();
        for (int h = warp; h < heads; h += D8_THREADS / 32) {
            const float s0 = Ss[h * D8_TILE + lane], s1 = Ss[h * D8_TILE + lane + 32];
            const float m_old = row_m[h], m_new = fmaxf(m_old, warp_max(fmaxf(s0, s1)));
            const float m = m_new > -INFINITY ? m_new : 0.f;     // nothing but hidden keys and NaN so far
            const float p0 = s0 == -INFINITY ? 0.f : expf(s0 - m), p1 = s1 == -INFINITY ? 0.f : expf(s1 - m);
            const float alpha = m_old > -INFINITY ? expf(m_old - m) : 1.f;
            const float sum = warp_sum(p0 + p1);
            Ss[h * D8_TILE + lane] = p0 * v_scale[lane];
            Ss[h * D8_TILE + lane + 32] = p1 * v_scale[lane + 32];
            if (lane == 0) {
                row_m[h] = m_new;
                row_l[h] = row_l[h] * alpha + sum;
                row_a[h] = alpha;
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < D8_MAX_ACC; ++i) {                   // a thread owns (head, column pair) tid, tid + 128, ...
            const int idx = tid + i * D8_THREADS;
            if (idx < pairs) {
                const int h = idx / (d / 2), c = (idx % (d / 2)) * 2;
                const float alpha = row_a[h];
                float a0 = acc[i][0] * alpha, a1 = acc[i][1] * alpha;
                const float* prow = Ss + h * D8_TILE;
#pragma unroll 8
                for (int key = 0; key < D8_TILE; ++key) {
                    const float2 v = kv8_unpack2(*reinterpret_cast<const unsigned short*>(Vs + key * d + c));
                    a0 = fmaf(prow[key], v.x, a0);
                    a1 = fmaf(prow[key], v.y, a1);
                }
                acc[i][0] = a0;
                acc[i][1] = a1;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < D8_MAX_ACC; ++i) {
        const int idx = tid + i * D8_THREADS;
        if (idx < pairs) {
            const int h = idx / (d / 2), c = (idx % (d / 2)) * 2;
            float* dst = p.part_o + (((size_t)r * p.nq + kvh * G + head0 + h) * p.splits + blockIdx.x) * d + c;
            dst[0] = acc[i][0];
            dst[1] = acc[i][1];
        }
    }
    if (tid < heads) {
        float* ml = p.part_ml + (((size_t)r * p.nq + kvh * G + head0 + tid) * p.splits + blockIdx.x) * 2;
        ml[0] = row_m[tid];
        ml[1] = row_l[tid];
    }
}

// One block per (query head, request): the weights exp(m_s - m) of the splits once, then groups of d / 4 threads sum every so many-th
// split, four columns a thread, and the groups' sums are added in their order. A split without a finite score has left m = -inf: its sums are zeros, or NaN where its keys were.
template <typename T>
__global__ void __launch_bounds__(D8_THREADS) kv8_merge_kernel(const Decode8Params p, T* __restrict__ out, long out_stride) {
    __shared__ float weight[D8_MAX_SPLITS];
    __shared__ float4 sums[D8_THREADS];
    __shared__ float scratch[32];
    pdl_trigger();
    pdl_wait();
    const int r = blockIdx.y, h = blockIdx.x;
    const int ctx = d8_context(p.ctx_len, r, p.max_ctx);
    const int splits = (ctx + p.split_keys - 1) / p.split_keys;
    const float* ml = p.part_ml + ((size_t)r * p.nq + h) * p.splits * 2;
    const float* po = p.part_o + ((size_t)r * p.nq + h) * p.splits * p.d;
    float m = -INFINITY;
    for (int s = threadIdx.x; s < splits; s += D8_THREADS) m = fmaxf(m, ml[2 * s]);
    m = block_max(m, scratch);
    float l = 0.f;
    for (int s = threadIdx.x; s < splits; s += D8_THREADS) {
        const float w = ml[2 * s] > -INFINITY ? expf(ml[2 * s] - m) : 1.f;
        weight[s] = w;
        l += ml[2 * s + 1] * w;
    }
    l = block_sum(l, scratch);
    __syncthreads();
    const float inv = l != 0.f ? 1.f / l : 0.f;                  // no keys: zeros
    const int lanes = p.d / 4, groups = D8_THREADS / lanes, group = threadIdx.x / lanes, c = threadIdx.x % lanes;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (group < groups) {
#pragma unroll 4
        for (int s = group; s < splits; s += groups) {
            const float4 v = reinterpret_cast<const float4*>(po + (size_t)s * p.d)[c];
            const float w = weight[s];
            o.x = fmaf(v.x, w, o.x); o.y = fmaf(v.y, w, o.y); o.z = fmaf(v.z, w, o.z); o.w = fmaf(v.w, w, o.w);
        }
        sums[threadIdx.x] = o;
    }
    __syncthreads();
    if (group == 0) {
        for (int g = 1; g < groups; ++g) {
            const float4 v = sums[g * lanes + c];
            o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
        }
        T* to = out + (size_t)r * out_stride + (size_t)h * p.d + c * 4;
        to[0] = from_float<T>(o.x * inv); to[1] = from_float<T>(o.y * inv); to[2] = from_float<T>(o.z * inv); to[3] = from_float<T>(o.w * inv);
    }
}

// Keys per split for a bound on the contexts: a tile (12 and 2 heads of 64, bfloat16: one request of 300 tokens 9.6 us, with two tiles 14;
// 8 of 4,100 20.7 and 28.6; 4 of 8,000 21.6 and 28.4), two where there are many partials to write and add up (10 ragged ones of up to 16,000:
// 41.8 and 37.8), or as many more as keep the partials of a row few.
static int d8_split_keys(long max_ctx) {
    long keys = max_ctx <= 8192 ? 64 : 128;
    while ((max_ctx + keys - 1) / keys > D8_MAX_SPLITS) keys *= 2;
    return (int)keys;
}

LLMP_API long llmp_kv8_decode_scratch_floats(int R, int nq, int d, int max_ctx) {
    const long keys = d8_split_keys(max_ctx), splits = (max_ctx + keys - 1) / keys;
    return (long)R * nq * (splits > 0 ? splits : 1) * (d + 2);
}

LLMP_API int llmp_kv8_decode(const void* q, long q_stride, void* out, long out_stride, int dtype, const void* pages, int num_pages,
                             const int* block_tables, int table_stride, const int* ctx_len, int R, int max_ctx, int nq, int nkv, int d,
                             int page_size, int window, float scale, float* scratch, long scratch_floats, cudaStream_t stream) {
    if (R <= 0) return 0;
    LLMP_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "kv8 attention: %d query heads cannot share %d key/value heads", nq, nkv);
    LLMP_REQUIRE(d >= 16 && d <= 256 && d % 16 == 0, "kv8 attention: head size %d is not a multiple of 16 in 16..256", d);
    LLMP_REQUIRE(page_size > 0 && num_pages > 0 && max_ctx > 0 && table_stride > 0, "kv8 attention: bad page size %d or context %d", page_size, max_ctx);
    LLMP_REQUIRE(R <= 65535, "kv8 attention: too many rows %d", R);
    LLMP_REQUIRE(((size_t)pages % 16) == 0, "kv8 attention: pages must be 16-byte aligned");
    LLMP_REQUIRE(llmp_kv8_decode_scratch_floats(R, nq, d, max_ctx) <= scratch_floats, "kv8 attention: scratch of %ld floats is too small", scratch_floats);
    Decode8Params p;
    const int G = nq / nkv;
    int hpb = G < D8_MAX_HEADS ? G : D8_MAX_HEADS;
    while (hpb > 1 && hpb * d / 2 > D8_MAX_ACC * D8_THREADS) --hpb;
    p.heads_per_block = hpb;
    p.head_chunks = (G + hpb - 1) / hpb;
    LLMP_REQUIRE((long)nkv * p.head_chunks <= 65535, "kv8 attention: too many heads");
    p.split_keys = d8_split_keys(max_ctx);
    p.splits = (max_ctx + p.split_keys - 1) / p.split_keys;
    p.q = q; p.pages = (const unsigned char*)pages; p.block_tables = block_tables; p.ctx_len = ctx_len; p.q_stride = q_stride;
    p.page_bytes = kv8_page_bytes(nkv, page_size, d); p.table_stride = table_stride; p.num_pages = num_pages;
    const long held = (long)table_stride * page_size;            // what a row of the tables has room for
    p.max_ctx = held < max_ctx ? (int)held : max_ctx;
    p.nq = nq; p.nkv = nkv; p.d = d; p.page_size = page_size; p.window = window; p.scale = scale;
    p.part_o = scratch;
    p.part_ml = scratch + (size_t)R * nq * p.splits * d;
    const size_t smem = (size_t)D8_TILE * (2 * d + 16) + sizeof(float) * D8_MAX_HEADS * (d + D8_TILE);
    const dim3 grid(p.splits, nkv * p.head_chunks, R), merge(nq, R);
    if (dtype == LLMP_F32) {
        llmp_launch_dependent(decode_kv8_kernel<float>, grid, dim3(D8_THREADS), smem, stream, p);
        llmp_launch_dependent(kv8_merge_kernel<float>, merge, dim3(D8_THREADS), 0, stream, p, (float*)out, out_stride);
    } else {
        llmp_launch_dependent(decode_kv8_kernel<bf16>, grid, dim3(D8_THREADS), smem, stream, p);
        llmp_launch_dependent(kv8_merge_kernel<bf16>, merge, dim3(D8_THREADS), 0, stream, p, (bf16*)out, out_stride);
    }
    return llmp_check_launch("kv8_decode");
}
