// Writing and unpacking pages of 8-bit keys and values (kv8.cuh), and copying pages of any cache.
#include "kv8.cuh"

#define KV8_WARPS 4

// ---- storing -----------------------------------------------------------------------------------------------------------
// Rows of k and v [tokens, nkv * d] go to their slots (page * page_size + offset; negative or beyond the pages: nowhere). A run is the
// consecutive rows of one page (rows without a slot between them aside). Per run and block (keys or values of one head):
//   need = smallest scale that holds the run's largest finite magnitude
//   e    = need, or the block's scale where that is larger and the run begins behind the page's first token
//   values held before the run's first offset, if e has grown:  q <- nearest(q * 2^(old - e))
//   the run's values:  q <- nearest(x * 2^(127 - e)), infinities and NaN to "no number"
// One warp owns a run of a block, so nothing is shared; rows of one page that are not neighbours would be two runs that
// write the same block at once. What lies behind the run in its page stays as it is.
//
// Latency bounds it (a warp has 4 KB to read and 2 KB to write): a warp reads the slots of its rows side by side and finds the runs
// that begin among them by votes, and asks for a whole page of 16 tokens at once, which stays in registers from the search for the
// largest to the rounding. 2,478 rows of 8 heads: 40 us with slots and rows read one after another, 14.6 so
// (ncu, cold caches), 10.5 in a captured graph.
struct StoreParams {
    const void* k;
    const void* v;
    const int* slots;
    unsigned char* pages;
    long k_stride, v_stride, page_bytes;
    int N, nkv, d, page_size, num_pages, rows_per_block, wide;
};

// Eight entries of a row, as they lie there. `wide`: they start on 16 bytes.
template <typename T> struct Eight {
    uint4 raw[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p, int wide) {
        if (wide) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(raw)[i] = p[i];
        }
    }
    __device__ __forceinline__ void none() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ float at(int i) const {
        const unsigned w = reinterpret_cast<const unsigned*>(raw)[sizeof(T) == 4 ? i : i >> 1];
        return __uint_as_float(sizeof(T) == 4 ? w : (i & 1 ? w & 0xffff0000u : w << 16));
    }
    __device__ __forceinline__ float largest(float amax) const {         // of the finite ones
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = fabsf(at(i));
            if (a < INFINITY) amax = fmaxf(amax, a);
        }
        return amax;
    }
    __device__ __forceinline__ uint2 round(float up) const {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = fabsf(at(i)) < INFINITY ? at(i) * up : __int_as_float(0x7fffffff);
        return make_uint2(kv8_pack4(x[0], x[1], x[2], x[3]), kv8_pack4(x[4], x[5], x[6], x[7]));
    }
};

template <typename T>
__global__ void __launch_bounds__(KV8_WARPS * 32) kv8_store_kernel(const StoreParams p) {
    constexpr int HELD = 8;                                      // pieces of eight entries a lane holds: 16 tokens of 128 entries a warp
    pdl_trigger();
    pdl_wait();                                                  // the rows, and what the pages hold, are complete
    const int lane = threadIdx.x & 31;
    const int unit = blockIdx.y * KV8_WARPS + (threadIdx.x >> 5);        // keys or values of one head
    if (unit >= 2 * p.nkv) return;
    const bool values = unit >= p.nkv;
    const T* src = reinterpret_cast<const T*>(values ? p.v : p.k) + (size_t)(values ? unit - p.nkv : unit) * p.d;
    const size_t stride = values ? p.v_stride : p.k_stride;
    const int slots_end = p.num_pages * p.page_size, pieces = p.d / 8;
    auto slot_of = [&](int row) {
        const int s = row < p.N ? p.slots[row] : -1;
        return s < slots_end ? s : -1;
    };
    // the runs that begin among this block's rows
    const int base = blockIdx.x * p.rows_per_block, window = min(p.rows_per_block, p.N - base);
    const int slot = lane < window ? slot_of(base + lane) : -1;
    const int page_here = slot < 0 ? -1 : slot / p.page_size;
    const unsigned live = __ballot_sync(0xffffffffu, slot >= 0);
    const unsigned lower = live & ((1u << lane) - 1u);
    int page_before = __shfl_sync(0xffffffffu, page_here, lower ? 31 - __clz(lower) : 0);
    if (slot >= 0 && !lower) {                                   // the first of them: the last row before the block that has a slot
        int row = base - 1, s = -1;
        for (; row >= 0 && (s = slot_of(row)) < 0; --row) {}
        page_before = s < 0 ? -1 : s / p.page_size;
    }
    for (unsigned starts = __ballot_sync(0xffffffffu, slot >= 0 && page_before != page_here); starts; starts &= starts - 1u) {
        const int begin = __ffs(starts) - 1;
        const int page = __shfl_sync(0xffffffffu, page_here, begin), first = base + begin;
        // the run's end, the lowest of its offsets, and whether they ascend (no slot twice)
        int end = first, lowest = p.page_size, last = -1;
        bool ordered = true;
        for (bool more = true; more;) {
            const int s = slot_of(end + lane);
            const bool other = end + lane >= p.N || (s >= 0 && s / p.page_size != page);
            const unsigned stop = __ballot_sync(0xffffffffu, other);
            const int count = stop ? __ffs(stop) - 1 : 32;
            const bool in = lane < count && s >= 0;
            if (in) lowest = min(lowest, s % p.page_size);
            const unsigned ins = __ballot_sync(0xffffffffu, in), lower = ins & ((1u << lane) - 1u);
            const int before = __shfl_sync(0xffffffffu, s, lower ? 31 - __clz(lower) : 0);
            if (in && s <= (lower ? before : last)) ordered = false;
            if (ins) last = __shfl_sync(0xffffffffu, s, 31 - __clz(ins));
            end += count;
            more = !stop;
        }
        lowest = __reduce_min_sync(0xffffffffu, lowest);
        ordered = __all_sync(0xffffffffu, ordered);
        unsigned char* block = p.pages + (size_t)page * p.page_bytes + (size_t)unit * p.page_size * p.d;
        unsigned char* scale = p.pages + (size_t)page * p.page_bytes + (size_t)2 * p.nkv * p.page_size * p.d + unit;
        const int count = (end - first) * pieces;
        const int old = lowest > 0 ? *scale : 0;
        // piece i of the run: entries 8 (i mod pieces) .. of its row i / pieces
        Eight<T> held[HELD];
        int to[HELD];                                            // where in the block it goes; -1: nowhere
        auto ask = [&](int i, Eight<T>& x) {
            x.none();
            if (i >= count) return -1;
            const int row = first + i / pieces, c = i % pieces * 8;
            const int s = slot_of(row);
            if (s < 0) return -1;
            x.load(src + (size_t)row * stride + c, p.wide);
            return s % p.page_size * p.d + c;
        };
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < HELD; ++j) to[j] = ask(j * 32 + lane, held[j]);
#pragma unroll
        for (int j = 0; j < HELD; ++j) amax = held[j].largest(amax);
        for (int i = HELD * 32 + lane; i < count; i += 32) {
            Eight<T> x;
            ask(i, x);
            amax = x.largest(amax);
        }
        amax = warp_max(amax);
        int e = kv8_needed(amax);
        if (lowest > 0 && old >= e) {
            e = old;
        } else if (lowest > 0) {                                 // the tokens before the run move to the larger scale
            const float down = kv8_power(max(old - e, -126));
            for (int i = lane; i < lowest * pieces; i += 32) {
                uint2* at = reinterpret_cast<uint2*>(block) + i;
                const uint2 w = *at;
                float a[4], b[4];
                kv8_unpack4(w.x, a);
                kv8_unpack4(w.y, b);
                *at = make_uint2(kv8_pack4(a[0] * down, a[1] * down, a[2] * down, a[3] * down),
                                 kv8_pack4(b[0] * down, b[1] * down, b[2] * down, b[3] * down));
            }
        }
        __syncwarp();
        if (lane == 0) *scale = (unsigned char)e;
        const float up = kv8_power(127 - e);
        if (!ordered) {                                          // row by row: of a slot's rows the last one stays
            for (int row = first; row < end; ++row) {
                for (int c = lane; c < pieces; c += 32) {
                    Eight<T> x;
                    const int at = ask((row - first) * pieces + c, x);
                    if (at >= 0) *reinterpret_cast<uint2*>(block + at) = x.round(up);
                }
                __syncwarp();
            }
            continue;
        }
#pragma unroll
        for (int j = 0; j < HELD; ++j)
            if (to[j] >= 0) *reinterpret_cast<uint2*>(block + to[j]) = held[j].round(up);
        for (int i = HELD * 32 + lane; i < count; i += 32) {
            Eight<T> x;
            const int at = ask(i, x);
            if (at >= 0) *reinterpret_cast<uint2*>(block + at) = x.round(up);
        }
    }
}

static int kv8_check_sizes(const char* what, const void* pages, int num_pages, int nkv, int d, int page_size) {
    LLMP_REQUIRE(nkv > 0 && num_pages > 0 && page_size > 0, "%s: bad sizes (%d heads, %d pages of %d tokens)", what, nkv, num_pages, page_size);
    LLMP_REQUIRE(d >= 16 && d <= 256 && d % 16 == 0, "%s: head size %d is not a multiple of 16 in 16..256", what, d);
    LLMP_REQUIRE(((size_t)pages % 16) == 0, "%s: pages must be 16-byte aligned", what);
    LLMP_REQUIRE((long)num_pages * page_size < (1L << 31), "%s: token slots pass 32 bits", what);
    return 0;
}

LLMP_API long llmp_kv8_page_bytes(int nkv, int page_size, int d) { return kv8_page_bytes(nkv, page_size, d); }

LLMP_API int llmp_kv8_store(const void* k, long k_stride, const void* v, long v_stride, int dtype, const int* slots, void* pages,
                            int num_pages, int N, int nkv, int d, int page_size, cudaStream_t stream) {
    if (N <= 0) return 0;
    if (kv8_check_sizes("kv8_store", pages, num_pages, nkv, d, page_size)) return 1;
    StoreParams p;
    p.k = k; p.v = v; p.slots = slots; p.pages = (unsigned char*)pages; p.k_stride = k_stride; p.v_stride = v_stride;
    p.page_bytes = kv8_page_bytes(nkv, page_size, d); p.N = N; p.nkv = nkv; p.d = d; p.page_size = page_size; p.num_pages = num_pages;
    const long row16 = dtype == LLMP_F32 ? 4 : 8;                // entries of 16 bytes
    p.wide = ((size_t)k % 16) == 0 && ((size_t)v % 16) == 0 && k_stride % row16 == 0 && v_stride % row16 == 0;
    p.rows_per_block = N <= 256 ? 1 : 16;                        // few rows: mostly single tokens, a run each
    const dim3 grid((N + p.rows_per_block - 1) / p.rows_per_block, (2 * nkv + KV8_WARPS - 1) / KV8_WARPS);
    LLMP_REQUIRE(grid.y <= 65535, "kv8_store: too many heads");
    if (dtype == LLMP_F32) llmp_launch_dependent(kv8_store_kernel<float>, grid, dim3(KV8_WARPS * 32), 0, stream, p);
    else llmp_launch_dependent(kv8_store_kernel<bf16>, grid, dim3(KV8_WARPS * 32), 0, stream, p);
    return llmp_check_launch("kv8_store");
}

// ---- unpacking ---------------------------------------------------------------------------------------------------------
// Page i of out [n, 2, nkv, page_size, d] gets the values of the page in entry index[i] of the block tables [R, table_stride];
// zeros for tokens behind the request's context and for a missing page. A thread takes 16 keys and the 16 values at the same place, exact in
// either type; the threads of a token and head are 2^row_shift neighbours of one warp (some idle where d / 16 is no power of two). Bound by
// the bytes it writes, which the attention kernel then reads from L2: 2,048 tokens of 8 heads of 128 5.6 us, 16,000 18.3.
//
// `hide`: for attention kernels that multiply what a row does not see by 0. Where a value of a token and head is no number, it becomes 0 and
// the token's keys of that head become no numbers: its scores are then masked, or seen, like any others.
struct GatherParams {
    const unsigned char* pages;
    const int* tables;
    const int* ctx_len;
    const int* index;
    void* out;
    long page_bytes;
    int n, table_stride, entries, nkv, d, page_size, num_pages, row_shift, hide;
};

// All ones in the bytes that are no number (0x7f and 0xff).
__device__ __forceinline__ unsigned kv8_no_number(unsigned w) { return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu; }

// 16 values of a page times their scale.
__device__ __forceinline__ void kv8_write16(float* dst, uint4 raw, float s) {
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        float q[4];
        kv8_unpack4(w[c], q);
        reinterpret_cast<float4*>(dst)[c] = make_float4(q[0] * s, q[1] * s, q[2] * s, q[3] * s);
    }
}
__device__ __forceinline__ void kv8_write16(bf16* dst, uint4 raw, float s) {
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
    unsigned h[8];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        float q[4];
        kv8_unpack4(w[c], q);
        const __nv_bfloat162 lo = __floats2bfloat162_rn(q[0] * s, q[1] * s), hi = __floats2bfloat162_rn(q[2] * s, q[3] * s);
        h[2 * c] = *reinterpret_cast<const unsigned*>(&lo);
        h[2 * c + 1] = *reinterpret_cast<const unsigned*>(&hi);
    }
    reinterpret_cast<uint4*>(dst)[0] = make_uint4(h[0], h[1], h[2], h[3]);
    reinterpret_cast<uint4*>(dst)[1] = make_uint4(h[4], h[5], h[6], h[7]);
}

template <typename T>
__global__ void __launch_bounds__(256) kv8_gather_kernel(const GatherParams p) {
    pdl_trigger();
    pdl_wait();
    const int i = blockIdx.x, lane = threadIdx.x & 31;
    const int entry = p.index[i];
    const bool known = entry >= 0 && entry < p.entries;
    int page = known ? p.tables[entry] : -1;
    if (page >= p.num_pages) page = -1;
    const int token0 = known ? entry % p.table_stride * p.page_size : 0;
    const int there = page >= 0 ? p.ctx_len[entry / p.table_stride] - token0 : 0;      // tokens of the page that exist
    const unsigned char* src = p.pages + (size_t)(page < 0 ? 0 : page) * p.page_bytes;
    const int rows = p.nkv * p.page_size, half = rows * p.d;     // (head, token) of keys, or of values
    const unsigned row_lanes = (p.row_shift == 4 ? 0xffffu : (1u << (1 << p.row_shift)) - 1u) << (lane >> p.row_shift << p.row_shift);
    T* out = reinterpret_cast<T*>(p.out) + (size_t)i * 2 * half;
    for (int at = blockIdx.y * blockDim.x + threadIdx.x; (at - lane) >> p.row_shift < rows; at += gridDim.y * blockDim.x) {      // (warps stay together)
        const int row = at >> p.row_shift, c = (at & ((1 << p.row_shift) - 1)) * 16;
        const bool mine = row < rows && c < p.d;
        uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
        float ks = 0.f, vs = 0.f;
        if (mine && row % p.page_size < there) {
            const int head = row / p.page_size;
            k = *reinterpret_cast<const uint4*>(src + (size_t)row * p.d + c);
            v = *reinterpret_cast<const uint4*>(src + half + (size_t)row * p.d + c);
            ks = kv8_scale(src[2 * (size_t)half + head]);
            vs = kv8_scale(src[2 * (size_t)half + p.nkv + head]);
        }
        if (p.hide) {
            const uint4 bad = make_uint4(kv8_no_number(v.x), kv8_no_number(v.y), kv8_no_number(v.z), kv8_no_number(v.w));
            v = make_uint4(v.x & ~bad.x, v.y & ~bad.y, v.z & ~bad.z, v.w & ~bad.w);
            if (__ballot_sync(0xffffffffu, (bad.x | bad.y | bad.z | bad.w) != 0u) & row_lanes) k = make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);
        }
        if (mine) {
            kv8_write16(out + (size_t)row * p.d + c, k, ks);
            kv8_write16(out + half + (size_t)row * p.d + c, v, vs);
        }
    }
}

LLMP_API int llmp_kv8_gather(const void* pages, int num_pages, const int* tables, int R, int table_stride, const int* ctx_len,
                             const int* index, int n, void* out, int dtype, int nkv, int d, int page_size, int hide, cudaStream_t stream) {
    if (n <= 0) return 0;
    if (kv8_check_sizes("kv8_gather", pages, num_pages, nkv, d, page_size)) return 1;
    LLMP_REQUIRE(((size_t)out % 16) == 0, "kv8_gather: the output must be 16-byte aligned");
    LLMP_REQUIRE(table_stride > 0 && (long)R * table_stride < (1L << 31), "kv8_gather: bad block tables");
    LLMP_REQUIRE(2L * nkv * page_size * d < (1L << 31), "kv8_gather: a page of %d tokens is too large", page_size);
    GatherParams p;
    p.pages = (const unsigned char*)pages; p.tables = tables; p.ctx_len = ctx_len; p.index = index; p.out = out;
    p.page_bytes = kv8_page_bytes(nkv, page_size, d); p.n = n; p.table_stride = table_stride; p.entries = R * table_stride;
    p.nkv = nkv; p.d = d; p.page_size = page_size; p.num_pages = num_pages; p.hide = hide;
    p.row_shift = 0;
    while ((16 << p.row_shift) < d) ++p.row_shift;
    const long threads = (long)nkv * page_size << p.row_shift;
    const long blocks = (threads + 255) / 256;                   // one turn a thread (16,000 tokens 18.3 us; two 20.7, four 23.6)
    const dim3 grid(n, (unsigned)(blocks < 64 ? blocks : 64));
    if (dtype == LLMP_F32) llmp_launch_dependent(kv8_gather_kernel<float>, grid, dim3(256), 0, stream, p);
    else llmp_launch_dependent(kv8_gather_kernel<bf16>, grid, dim3(256), 0, stream, p);
    return llmp_check_launch("kv8_gather");
}

// ---- copying pages -------------------------------------------------------------------------------------------------------
// Page src[i] to page dst[i] in every one of a few caches; no destination is a source or another destination (the caller
// checks), so the copies are independent. The list travels in the launch's parameters: nothing to upload, nothing that has to
// outlive the launch. A block copies 16 KB with all its reads ahead of its writes: 1,500 pages of 64 KB in 4 caches 127 us, 6.2 TB/s read and written.
#define COPY_TENSORS 48
#define COPY_PAIRS 384
struct CopyParams {
    unsigned char* base[COPY_TENSORS];
    int src[COPY_PAIRS], dst[COPY_PAIRS];
    long page_bytes;
    int wide;
};
#define COPY_BLOCK_BYTES 16384

__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CopyParams p) {
    unsigned char* base = p.base[blockIdx.z];
    const unsigned char* src = base + (size_t)p.src[blockIdx.y] * p.page_bytes;
    unsigned char* dst = base + (size_t)p.dst[blockIdx.y] * p.page_bytes;
    const long at = (long)blockIdx.x * COPY_BLOCK_BYTES;
    const int bytes = (int)(p.page_bytes - at < COPY_BLOCK_BYTES ? p.page_bytes - at : COPY_BLOCK_BYTES);
    pdl_trigger();
    pdl_wait();
    if (p.wide) {
        uint4 v[COPY_BLOCK_BYTES / 4096];
#pragma unroll
        for (int i = 0; i < COPY_BLOCK_BYTES / 4096; ++i) {
            const int o = (i * 256 + threadIdx.x) * 16;
            if (o < bytes) v[i] = *reinterpret_cast<const uint4*>(src + at + o);
        }
#pragma unroll
        for (int i = 0; i < COPY_BLOCK_BYTES / 4096; ++i) {
            const int o = (i * 256 + threadIdx.x) * 16;
            if (o < bytes) *reinterpret_cast<uint4*>(dst + at + o) = v[i];
        }
    } else {
        for (int o = threadIdx.x; o < bytes; o += 256) dst[at + o] = src[at + o];
    }
}

LLMP_API int llmp_copy_pages_max_tensors() { return COPY_TENSORS; }
LLMP_API int llmp_copy_pages_max_pairs() { return COPY_PAIRS; }

// bases: host array of `tensors` device pointers; src, dst: host arrays of `pairs` page numbers.
LLMP_API int llmp_copy_pages(const void* const* bases, int tensors, long page_bytes, const int* src, const int* dst, int pairs,
                             cudaStream_t stream) {
    if (tensors <= 0 || pairs <= 0 || page_bytes <= 0) return 0;
    LLMP_REQUIRE(tensors <= COPY_TENSORS && pairs <= COPY_PAIRS, "copy_pages: %d caches and %d pages are more than a launch takes", tensors, pairs);
    CopyParams p;
    bool wide = page_bytes % 16 == 0;
    for (int i = 0; i < tensors; ++i) {
        p.base[i] = (unsigned char*)const_cast<void*>(bases[i]);
        wide = wide && ((size_t)bases[i] % 16) == 0;
    }
    for (int i = 0; i < pairs; ++i) {
        p.src[i] = src[i];
        p.dst[i] = dst[i];
    }
    p.page_bytes = page_bytes;
    p.wide = wide;
    const long chunks = (page_bytes + COPY_BLOCK_BYTES - 1) / COPY_BLOCK_BYTES;
    LLMP_REQUIRE(chunks < (1L << 31), "copy_pages: a page is too large");
    const dim3 grid((unsigned)chunks, pairs, tensors);
    llmp_launch_dependent(copy_pages_kernel, grid, dim3(256), 0, stream, p);
    return llmp_check_launch("copy_pages");
}
