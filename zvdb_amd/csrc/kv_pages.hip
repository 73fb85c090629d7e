// kv_pages.hip -- the 4-bit key/value cache's pages: planning (block tables, slot map), writing rows, reading them back.
//
// All three are bound by latency when a decode step calls them (3.9, 2.7 and 2.7 us on the device for 64 tokens) and by HBM when a prompt
// does; none has arithmetic worth counting.
#include "kv_cache.h"

#include <algorithm>

namespace zvdb {

int kv_check_layout(const zvdb_hip_kv_layout *l, KvGeom *g) {
    KV_ARG(l, "null layout");
    KV_ARG(l->abi_version == ZVDB_HIP_ABI_VERSION, "kv layout: ABI version %u, library %u", l->abi_version, (unsigned)ZVDB_HIP_ABI_VERSION);
    KV_ARG(l->head_dim >= 8 && l->head_dim <= 256 && l->head_dim % 8 == 0, "kv layout: head_dim %u (a multiple of 8 up to 256)", l->head_dim);
    KV_ARG(l->kv_heads >= 1 && l->kv_heads <= 1024, "kv layout: kv_heads %u (1 .. 1024)", l->kv_heads);
    KV_ARG(l->page_size >= 16 && l->page_size <= 256 && (l->page_size & (l->page_size - 1)) == 0, "kv layout: page_size %u (16, 32, 64, 128 or 256)", l->page_size);
    KV_ARG(l->pages >= 1 && l->pages < 0x7FFFFFFFu, "kv layout: %llu pages (1 .. 2^31 - 2)", (unsigned long long)l->pages);
    g->head_bytes = (uint32_t)kv_head_bytes(l);
    g->page_bytes = (uint64_t)g->head_bytes * l->kv_heads;
    g->pages = (uint32_t)l->pages;
    g->heads = l->kv_heads;
    g->dim = l->head_dim;
    g->page_size = l->page_size;
    g->page_shift = (uint32_t)__builtin_ctz(l->page_size);
    return ZVDB_OK;
}

int KvDevice::enter(const void *p, hipStream_t s) {
    int n = 0;
    if (hipGetDeviceCount(&n) != hipSuccess || n == 0) {
        (void)hipGetLastError();
        set_error("no HIP device");
        return ZVDB_ERR_NO_DEVICE;
    }
    hipPointerAttribute_t at;
    if (hipPointerGetAttributes(&at, p) != hipSuccess || (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged) || at.device < 0 || at.device >= n) {
        (void)hipGetLastError();
        set_error("a kv call needs device memory");
        return ZVDB_ERR_INVALID;
    }
    if (s) {
        hipDevice_t d = 0;
        ZV_HIP(hipStreamGetDevice(s, &d));
        KV_ARG(d == at.device, "the stream is of device %d, the memory of device %d", (int)d, at.device);
    }
    int cur = 0;
    ZV_HIP(hipGetDevice(&cur));
    if (cur != at.device) {
        ZV_HIP(hipSetDevice(at.device));
        prev_ = cur;
    }
    ZV_HIP(hipDeviceGetAttribute(&cus_, hipDeviceAttributeMultiprocessorCount, at.device));
    return ZVDB_OK;
}

// ---- plan ---------------------------------------------------------------------------------------------------------------

struct KvPlanArgs {
    const uint32_t *lengths, *fresh, *ring;
    const uint64_t *cursor;
    uint32_t *tables, *starts, *out_lengths, *status;
    uint64_t *slots, *out_cursor;
    uint64_t slot_cap;
    uint32_t n, ring_size, table_stride, pages, page_shift;
};

constexpr uint32_t kPlanMax = 16384;  // requests of a call: 16 to a thread

// last i with first[i] <= x, in first[0 .. n] (first[0] = 0 <= x < first[n])
__device__ inline uint32_t kv_owner(const uint32_t *first, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n;  // first[lo] <= x < first[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (first[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Sums of counts that stop at 2^31 - 1, which no call may reach: they saturate, so the order of the additions does not matter
constexpr uint32_t kPlanFull = 0x7FFFFFFF;
__device__ inline uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, kPlanFull); }

// Inclusive sums over 16 lanes (a DPP row), and from there over 64: no LDS
template <int CTRL, int ROWS>
__device__ inline uint32_t dpp_or_zero(uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, false); }
__device__ inline uint32_t sum_upto_16(uint32_t x) {
    x = sat_add(x, dpp_or_zero<0x111, 0xF>(x));  // row_shr:1
    x = sat_add(x, dpp_or_zero<0x112, 0xF>(x));  // row_shr:2
    x = sat_add(x, dpp_or_zero<0x114, 0xF>(x));  // row_shr:4
    return sat_add(x, dpp_or_zero<0x118, 0xF>(x));  // row_shr:8
}
__device__ inline uint32_t sum_upto_64(uint32_t x) {
    x = sum_upto_16(x);
    x = sat_add(x, dpp_or_zero<0x142, 0xA>(x));  // row_bcast:15 into rows 1 and 3
    return sat_add(x, dpp_or_zero<0x143, 0xC>(x));  // row_bcast:31 into rows 2 and 3
}

// Every block sums the whole batch (8 n bytes that stay in L2): one launch, no block waits for another, and nothing that a block
// reads is written by one (a partly filled page's table entry is an older call's; new pages are read from the ring).  The unit of
// work behind the sums is a RUN, the new tokens of one page: 16 lanes find its request -- a search over the threads' sums in LDS, then
// a scan of that thread's at most 16 requests -- look its page up once and write its slots side by side.  Bound by latency: the sums
// and one run are some ten dependent reads (2,048 prompts, 1.05M tokens: 10.0 us; 16.1 with a search for each token, 13.0 with sums in
// 64 bits through LDS).
__global__ __launch_bounds__(1024) void k_kv_plan(const KvPlanArgs a) {
    __shared__ uint32_t tok[1025], pag[1025], run[1025];  // sums before each thread's requests
    __shared__ uint32_t wave_sum[3][16], bad;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nt = blockDim.x;
    const uint32_t per = (a.n + nt - 1) / nt, i0 = min(tid * per, a.n), i1 = min(i0 + per, a.n);
    const uint32_t mask = (1u << a.page_shift) - 1;
    if (tid == 0) bad = 0;
    __syncthreads();
    uint32_t st = 0, sp = 0, sr = 0;
    for (uint32_t i = i0; i < i1; ++i) {
        const uint32_t c = a.lengths[i], f = a.fresh[i];
        const uint64_t e = (uint64_t)c + f, want = (e + mask) >> a.page_shift;
        if (want > a.table_stride || e > kPlanFull) {
            bad = 1;  // (every writer writes the same)
            st = sat_add(st, min(f, kPlanFull));
            sp = sat_add(sp, (uint32_t)(want - (((uint64_t)c + mask) >> a.page_shift)));
        } else {
            st = sat_add(st, f);
            sp = sat_add(sp, (uint32_t)want - ((c + mask) >> a.page_shift));
            sr += f ? (uint32_t)want - (c >> a.page_shift) : 0;
        }
    }
    uint32_t it = sum_upto_64(st), ip = sum_upto_64(sp), ir = sum_upto_64(sr);  // over the block's threads
    if (lane == 63) { wave_sum[0][wave] = it; wave_sum[1][wave] = ip; wave_sum[2][wave] = ir; }
    __syncthreads();
    uint32_t tt = 0, tp = 0, tr = 0;
    {
        const bool there = lane < nt / 64;
        const uint32_t x = sum_upto_16(there ? wave_sum[0][lane & 15] : 0), y = sum_upto_16(there ? wave_sum[1][lane & 15] : 0), z = sum_upto_16(there ? wave_sum[2][lane & 15] : 0);
        tt = __builtin_amdgcn_readlane(x, 15);
        tp = __builtin_amdgcn_readlane(y, 15);
        tr = __builtin_amdgcn_readlane(z, 15);
        if (wave) {
            const uint32_t w = __builtin_amdgcn_readfirstlane(wave) - 1;
            it = sat_add(it, __builtin_amdgcn_readlane(x, w));
            ip = sat_add(ip, __builtin_amdgcn_readlane(y, w));
            ir = sat_add(ir, __builtin_amdgcn_readlane(z, w));
        }
    }
    const uint64_t taken = a.cursor[0], given = a.cursor[1];
    const uint64_t left = given > taken ? min(given - taken, (uint64_t)a.ring_size) : 0;
    const uint32_t code = bad ? ZVDB_KV_TABLE_TOO_SHORT : tt > a.slot_cap ? ZVDB_KV_SLOTS_TOO_FEW : tp > left ? ZVDB_KV_OUT_OF_PAGES : ZVDB_KV_PLANNED;
    const bool ok = code == ZVDB_KV_PLANNED;  // then no sum is full: slot_cap and the ring are below that
    tok[tid] = it - st;
    pag[tid] = ip - sp;
    run[tid] = ir - sr;
    if (tid == 0) run[nt] = tr;
    if (blockIdx.x == 0) {
        uint32_t x = it - st;
        for (uint32_t i = i0; i < i1; ++i) {
            const uint32_t c = a.lengths[i], f = a.fresh[i];
            a.starts[i] = ok ? x : 0;
            a.out_lengths[i] = c + (ok ? f : 0);
            x += f;
        }
        if (tid == 0) {
            a.starts[a.n] = ok ? tt : 0;
            a.out_cursor[0] = taken + (ok ? tp : 0);
            a.out_cursor[1] = given;
            a.status[0] = code;
            a.status[1] = tp;
            a.status[2] = tt;
            a.status[3] = 0;
        }
    }
    __syncthreads();
    const uint64_t at = (uint64_t)blockIdx.x * nt + tid, step = (uint64_t)gridDim.x * nt;
    for (uint64_t t = (ok ? tt : 0) + at; t < a.slot_cap; t += step) a.slots[t] = ~0ull;
    if (!ok) return;
    const uint32_t base = (uint32_t)(taken % a.ring_size), l16 = tid & 15, group = lane & ~15u;
    for (uint64_t x = at / 16; x < tr; x += step / 16) {
        const uint32_t c = kv_owner(run, nt, (uint32_t)x);
        const uint32_t i = c * per + l16;
        const bool mine = l16 < per && i < a.n;
        const uint32_t len = mine ? a.lengths[i] : 0, add = mine ? a.fresh[i] : 0;
        const uint32_t want = (len + add + mask) >> a.page_shift, news = want - ((len + mask) >> a.page_shift), runs = add ? want - (len >> a.page_shift) : 0;
        const uint32_t xt = sum_upto_16(add), xp = sum_upto_16(news), xr = sum_upto_16(runs);  // over the thread's requests
        const uint32_t r = (uint32_t)x - run[c];
        const uint64_t hit = __ballot(r >= xr - runs && r < xr) >> group & 0xFFFF;  // one lane's request holds the run
        const int src = __ffsll((unsigned long long)hit) - 1;
        const uint32_t o_len = __shfl(len, src, 16), o_add = __shfl(add, src, 16), o_tok = tok[c] + __shfl(xt - add, src, 16), o_pag = pag[c] + __shfl(xp - news, src, 16),
                       o_run = __shfl(xr - runs, src, 16);
        const uint64_t row = (uint64_t)(c * per + src) * a.table_stride;
        const uint32_t p = (o_len >> a.page_shift) + r - o_run, have = (o_len + mask) >> a.page_shift;
        uint32_t page;
        if (p < have) {
            page = a.tables[row + p];
        } else {
            const uint64_t from = (uint64_t)base + o_pag + p - have;  // below twice the ring
            page = a.ring[from >= a.ring_size ? from - a.ring_size : from];
            if (l16 == 0) a.tables[row + p] = page;
        }
        const uint32_t lo = max(o_len, p << a.page_shift), hi = min(o_len + o_add, (p + 1) << a.page_shift);
        for (uint32_t pos = lo + l16; pos < hi; pos += 16)
            a.slots[o_tok + (pos - o_len)] = page < a.pages ? ((uint64_t)page << a.page_shift) | (pos & mask) : ~0ull;
    }
}

// ---- append -------------------------------------------------------------------------------------------------------------

template <class T>
__device__ inline void kv_load8(const T *p, float *x) {
    if constexpr (sizeof(T) == 2) {
        const uint4 u = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    } else {
        const float4 u = *reinterpret_cast<const float4 *>(p), v = *reinterpret_cast<const float4 *>(p + 4);
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
        x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
    }
}

// One lane takes 8 elements of a row, four lanes a block of 32.  The block's scale is the power of two at or under its largest
// magnitude over E2M1's 4 -- the next one from 7/4 of it on, where 6 would be nearer than 8 and the largest element would lose an
// eighth and more of itself.  A power of two divides exactly, so the code is the nearest of x / scale, ties to even (bf16 rows
// meet ties often: 8 significant bits over a grid of 3), saturating at 6.  Lanes of one wave hold consecutive tokens of ONE head:
// the four tokens of a V group are written by neighbouring lanes into the same 16 pieces.  A lane takes two heads of its token, so that
// more of what it reads is in flight and in one place (65,537 rows of 8 x 128 bf16, keys and values, buffers in turn: one head a lane 89 us,
// two 72, four 71, eight 76; 40,000 of 5 x 64 fp32: 23.4, 23.4, 27.3, 25.1).  Bound by HBM: 340 MB in 72 us, 4.7 TB/s; 32,771 rows of 8 x 96
// fp32: 237 MB in 46 us, 5.2 TB/s.  Loads that pass the caches by: 70.7 and 48.4 us, 8,192 rows 11.2 for 9.9; not taken.
constexpr int kAppendHeads = 2;

template <class T, int NB>
__global__ __launch_bounds__(256) void k_kv_append(uint8_t *cache, const KvGeom g, const T *k, uint64_t k_stride, const T *v, uint64_t v_stride,
                                                   const uint64_t *slots, uint32_t n) {
    constexpr uint32_t L = 4 * NB;  // lanes of a row
    const uint32_t c8 = threadIdx.x % L, groups = (g.heads + kAppendHeads - 1) / kAppendHeads, head0 = kv_block() % groups * kAppendHeads;
    const uint64_t i = (uint64_t)(kv_block() / groups) * (256 / L) + threadIdx.x / L;
    if (i >= n) return;  // (whole rows leave: the four lanes of a block stay together)
    const uint64_t slot = slots[i];
    if (slot >= (uint64_t)g.pages << g.page_shift) return;
    const bool value = blockIdx.z;
    const T *src = (value ? v + i * v_stride : k + i * k_stride) + (uint64_t)head0 * g.dim + c8 * 8;
    float x[kAppendHeads][8] = {};
#pragma unroll
    for (int h = 0; h < kAppendHeads; ++h)
        if (head0 + h < g.heads && c8 * 8 < g.dim) kv_load8(src + (uint64_t)h * g.dim, x[h]);
    const uint32_t t = (uint32_t)slot & (g.page_size - 1), half = g.page_size * 16 * NB;
    uint8_t *at = cache + (slot >> g.page_shift) * g.page_bytes + (uint64_t)head0 * g.head_bytes;
#pragma unroll
    for (int h = 0; h < kAppendHeads; ++h, at += g.head_bytes) {
        if (head0 + h >= g.heads) break;
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[h][j]) & 0x7FFFFFFFu);
        top = max(top, (uint32_t)__shfl_xor((int)top, 1));
        top = max(top, (uint32_t)__shfl_xor((int)top, 2));
        const int e = (int)((top + 0x200000u) >> 23) - 2;
        uint32_t b = (uint32_t)min(max(e, (int)kKvScaleMin), (int)kKvScaleMax), code = 0;
        if (top >= 0x7F800000u) {
            b = kKvScaleNaN;
        } else {
            const float s = __uint_as_float(b << 23);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[h][0], x[h][1], s, 0);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[h][2], x[h][3], s, 1);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[h][4], x[h][5], s, 2);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[h][6], x[h][7], s, 3);
        }
        uint8_t *const scales = at + 2 * half;
        if (!value) {
            *reinterpret_cast<uint32_t *>(at + t * (16 * NB) + c8 * 4) = code;
            if (c8 % 4 == 0) scales[t * NB + c8 / 4] = (uint8_t)b;
        } else {
            uint8_t *const w = at + half;
            if constexpr (NB == 2) {
                *reinterpret_cast<uint16_t *>(w + kv_v_offset<NB>(t, 2 * c8)) = (uint16_t)code;
                *reinterpret_cast<uint16_t *>(w + kv_v_offset<NB>(t, 2 * c8 + 1)) = (uint16_t)(code >> 16);
            } else if constexpr (NB == 4) {
                *reinterpret_cast<uint32_t *>(w + kv_v_offset<NB>(t, c8)) = code;
            } else {
                *reinterpret_cast<uint32_t *>(w + kv_v_offset<NB>(t, c8 / 2) + (c8 % 2) * 4) = code;
            }
            if (c8 % 4 == 0) scales[g.page_size * NB + (t >> 2) * (4 * NB) + c8 + (t & 3)] = (uint8_t)b;
        }
    }
}

// ---- read ---------------------------------------------------------------------------------------------------------------

// Rows read back are not read again here: their stores pass the caches by (65,537 rows of 8 x 128 bf16: 51 us, 68 without).
template <class T>
__device__ inline void kv_store16(T *p, const float *x) {
    if constexpr (sizeof(T) == 2) {  // a code times a power of two is a bf16 number: nothing is rounded
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (__float_as_uint(x[2 * i]) >> 16) | (__float_as_uint(x[2 * i + 1]) & 0xFFFF0000u);
        __builtin_nontemporal_store(u32x4{w[0], w[1], w[2], w[3]}, reinterpret_cast<u32x4 *>(p));
    } else {
        __builtin_nontemporal_store(f32x4{x[0], x[1], x[2], x[3]}, reinterpret_cast<f32x4 *>(p));
    }
}

// The append the other way round; a slot that is not in the cache reads as zeros.  A lane makes 16 bytes of a row, so that every store
// fills whole lines (8 fp32 elements to a lane, two stores of half a line each: 102 us where this takes 71, append included), and takes
// four heads of its token: what a block writes lies together, and four loads are on their way at once (heads 1 / 2 / 4 / 8 a lane: 92 / 69 / 62 /
// 65 us).  Bound by HBM: 65,537 rows of 8 x 128 to bf16, keys and values: 340 MB in 51 us into one pair of buffers, in 62 into four in
// turn, 5.5 TB/s.
constexpr int kReadHeads = 4;

template <class T, int NB>
__global__ __launch_bounds__(256) void k_kv_read(const uint8_t *cache, const KvGeom g, const uint64_t *slots, uint32_t n, T *k, T *v) {
    constexpr uint32_t E = 16 / sizeof(T), L = 32 * NB / E;  // elements of a lane, lanes of a row
    const uint32_t col = threadIdx.x % L * E, groups = (g.heads + kReadHeads - 1) / kReadHeads, head0 = kv_block() % groups * kReadHeads;
    const uint64_t i = (uint64_t)(kv_block() / groups) * (256 / L) + threadIdx.x / L;
    const bool value = k == nullptr || blockIdx.z;
    T *const dst = value ? v : k;
    if (i >= n || col >= g.dim) return;
    const uint64_t slot = slots[i];
    uint32_t code[kReadHeads] = {}, b[kReadHeads] = {};
    if (slot < (uint64_t)g.pages << g.page_shift) {
        const uint32_t t = (uint32_t)slot & (g.page_size - 1), half = g.page_size * 16 * NB;
        const uint8_t *const first = cache + (slot >> g.page_shift) * g.page_bytes + (uint64_t)head0 * g.head_bytes;
#pragma unroll
        for (int h = 0; h < kReadHeads; ++h) {
            if (head0 + h >= g.heads) break;
            const uint8_t *const at = first + (uint64_t)h * g.head_bytes, *const scales = at + 2 * half;
            const uint8_t *const w = value ? at + half + kv_v_offset<NB>(t, col / (2 * NB)) + col % (2 * NB) / 2 : at + t * (16 * NB) + col / 2;
            if constexpr (E == 4) code[h] = *reinterpret_cast<const uint16_t *>(w);
            else if constexpr (NB == 2)
                code[h] = *reinterpret_cast<const uint16_t *>(w) |
                          (uint32_t)*reinterpret_cast<const uint16_t *>(value ? at + half + kv_v_offset<NB>(t, col / 4 + 1) : w + 2) << 16;
            else code[h] = *reinterpret_cast<const uint32_t *>(w);
            b[h] = value ? scales[g.page_size * NB + (t >> 2) * (4 * NB) + (col / 32) * 4 + (t & 3)] : scales[t * NB + col / 32];
        }
    }
    T *const out = dst + (i * g.heads + head0) * g.dim + col;
#pragma unroll
    for (int h = 0; h < kReadHeads; ++h) {
        if (head0 + h >= g.heads) break;
        const float s = __uint_as_float(b[h] << 23);
        bf16x2 y[4] = {};
        y[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code[h], s, 0);
        y[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code[h], s, 1);
        if constexpr (E == 8) {
            y[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code[h], s, 2);
            y[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code[h], s, 3);
        }
        float x[E];
#pragma unroll
        for (uint32_t j = 0; j < E; ++j) x[j] = b[h] == kKvScaleNaN ? __uint_as_float(0x7FC00000u) : (float)y[j / 2][j % 2];
        kv_store16(out + (uint64_t)h * g.dim, x);
    }
}

template <class T>
static void launch_append(uint8_t *cache, const KvGeom &g, const void *k, uint64_t ks, const void *v, uint64_t vs, const uint64_t *slots, uint32_t n, hipStream_t s) {
    const T *kk = static_cast<const T *>(k), *vv = static_cast<const T *>(v);
    const uint32_t w = kv_width(g.dim), rows = 256 / (w / 8);
    const dim3 grid = kv_grid(((uint64_t)n + rows - 1) / rows * ((g.heads + kAppendHeads - 1) / kAppendHeads), 2);
    if (w == 64) hipLaunchKernelGGL((k_kv_append<T, 2>), grid, dim3(256), 0, s, cache, g, kk, ks, vv, vs, slots, n);
    else if (w == 128) hipLaunchKernelGGL((k_kv_append<T, 4>), grid, dim3(256), 0, s, cache, g, kk, ks, vv, vs, slots, n);
    else hipLaunchKernelGGL((k_kv_append<T, 8>), grid, dim3(256), 0, s, cache, g, kk, ks, vv, vs, slots, n);
}

template <class T>
static void launch_read(const uint8_t *cache, const KvGeom &g, const uint64_t *slots, uint32_t n, void *k, void *v, hipStream_t s) {
    T *kk = static_cast<T *>(k), *vv = static_cast<T *>(v);
    const uint32_t w = kv_width(g.dim), rows = 256 * 16 / sizeof(T) / w, groups = (g.heads + kReadHeads - 1) / kReadHeads;
    const dim3 grid = kv_grid(((uint64_t)n + rows - 1) / rows * groups, k && v ? 2 : 1);
    if (w == 64) hipLaunchKernelGGL((k_kv_read<T, 2>), grid, dim3(256), 0, s, cache, g, slots, n, kk, vv);
    else if (w == 128) hipLaunchKernelGGL((k_kv_read<T, 4>), grid, dim3(256), 0, s, cache, g, slots, n, kk, vv);
    else hipLaunchKernelGGL((k_kv_read<T, 8>), grid, dim3(256), 0, s, cache, g, slots, n, kk, vv);
}

}  // namespace zvdb

using namespace zvdb;

extern "C" {

int zvdb_hip_kv_page_bytes(const zvdb_hip_kv_layout *layout, uint64_t *out_bytes) {
    KvGeom g;
    ZV_CHECK(kv_check_layout(layout, &g));
    KV_ARG(out_bytes, "null argument");
    *out_bytes = g.page_bytes;
    return ZVDB_OK;
}

int zvdb_hip_kv_plan_dev(const zvdb_hip_kv_layout *layout, const void *d_lengths, const void *d_new, uint32_t n, const void *d_ring,
                         uint32_t ring_size, const void *d_cursor, void *d_tables, uint32_t table_stride, void *d_starts, void *d_slots,
                         uint64_t slot_cap, void *d_out_lengths, void *d_out_cursor, void *d_status, void *stream) {
    KvGeom g;
    ZV_CHECK(kv_check_layout(layout, &g));
    KV_ARG(d_cursor && d_ring && d_starts && d_out_cursor && d_status, "null argument");
    KV_ARG(n == 0 || (d_lengths && d_new && d_tables && d_out_lengths), "null argument");
    KV_ARG(slot_cap == 0 || d_slots, "null argument");
    KV_ARG(n <= kPlanMax, "kv_plan: %u requests (at most %u)", n, kPlanMax);
    KV_ARG(ring_size >= 1 && ring_size < 0x7FFFFFFFu, "kv_plan: a ring of %u pages", ring_size);
    KV_ARG(table_stride >= 1 && table_stride < 0x7FFFFFFFu, "kv_plan: table_stride %u", table_stride);
    KV_ARG(slot_cap < 0x7FFFFFFFu, "kv_plan: %llu slots (below 2^31 - 1)", (unsigned long long)slot_cap);
    KV_ARG(kv_aligned(d_cursor, 8) && kv_aligned(d_out_cursor, 8) && kv_aligned(d_slots, 8), "kv_plan: a 64-bit array is not 8-byte aligned");
    KV_ARG(d_out_cursor != d_cursor && (n == 0 || (d_out_lengths != d_lengths && d_out_lengths != d_new)), "kv_plan: an output is an input (every block reads the inputs)");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    KvDevice dev;
    ZV_CHECK(dev.enter(d_status, s));
    KvPlanArgs a;
    a.lengths = static_cast<const uint32_t *>(d_lengths);
    a.fresh = static_cast<const uint32_t *>(d_new);
    a.ring = static_cast<const uint32_t *>(d_ring);
    a.cursor = static_cast<const uint64_t *>(d_cursor);
    a.tables = static_cast<uint32_t *>(d_tables);
    a.starts = static_cast<uint32_t *>(d_starts);
    a.out_lengths = static_cast<uint32_t *>(d_out_lengths);
    a.status = static_cast<uint32_t *>(d_status);
    a.slots = static_cast<uint64_t *>(d_slots);
    a.out_cursor = static_cast<uint64_t *>(d_out_cursor);
    a.slot_cap = slot_cap;
    a.n = n; a.ring_size = ring_size; a.table_stride = table_stride; a.pages = g.pages; a.page_shift = g.page_shift;
    // 16 lanes for a run: a run for each page's worth of slots and, with few tokens each, for each request
    const uint32_t threads = n > 256 || slot_cap > 4096 ? 1024 : 256;
    const uint64_t runs = slot_cap / g.page_size + std::min<uint64_t>(n, slot_cap) + 1;
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((runs * 16 + threads - 1) / threads, 2 * (uint64_t)dev.cus());
    hipLaunchKernelGGL(k_kv_plan, dim3(blocks), dim3(threads), 0, s, a);
    ZV_HIP(hipGetLastError());
    return ZVDB_OK;
}

int zvdb_hip_kv_append_dev(const zvdb_hip_kv_layout *layout, void *d_cache, const void *d_k, uint64_t k_stride, const void *d_v, uint64_t v_stride,
                           uint32_t type, uint32_t n, const void *d_slots, void *stream) {
    KvGeom g;
    ZV_CHECK(kv_check_layout(layout, &g));
    KV_ARG(type == ZVDB_KV_F32 || type == ZVDB_KV_BF16, "kv_append: type %u", type);
    if (n == 0) return ZVDB_OK;
    KV_ARG(d_cache && d_k && d_v && d_slots, "null argument");
    KV_ARG((uint64_t)n * g.heads < 0x7FFFFFFFull, "kv_append: the call is too large (%u tokens)", n);
    KV_ARG(kv_aligned(d_cache, 16) && kv_aligned(d_k, 16) && kv_aligned(d_v, 16) && kv_aligned(d_slots, 8), "kv_append: cache, k and v need 16-byte alignment, slots 8");
    const uint64_t row = (uint64_t)g.heads * g.dim;
    KV_ARG(kv_stride_ok(k_stride, row) && kv_stride_ok(v_stride, row), "kv_append: a token's stride is at least kv_heads * head_dim = %llu, below 2^40 and a multiple of 8", (unsigned long long)row);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    KvDevice dev;
    ZV_CHECK(dev.enter(d_cache, s));
    uint8_t *c = static_cast<uint8_t *>(d_cache);
    const uint64_t *slots = static_cast<const uint64_t *>(d_slots);
    if (type == ZVDB_KV_F32) launch_append<float>(c, g, d_k, k_stride, d_v, v_stride, slots, n, s);
    else launch_append<uint16_t>(c, g, d_k, k_stride, d_v, v_stride, slots, n, s);
    ZV_HIP(hipGetLastError());
    return ZVDB_OK;
}

int zvdb_hip_kv_read_dev(const zvdb_hip_kv_layout *layout, const void *d_cache, const void *d_slots, uint32_t n, void *d_k, void *d_v, uint32_t type, void *stream) {
    KvGeom g;
    ZV_CHECK(kv_check_layout(layout, &g));
    KV_ARG(type == ZVDB_KV_F32 || type == ZVDB_KV_BF16, "kv_read: type %u", type);
    if (n == 0 || (!d_k && !d_v)) return ZVDB_OK;
    KV_ARG(d_cache && d_slots, "null argument");
    KV_ARG((uint64_t)n * g.heads < 0x7FFFFFFFull, "kv_read: the call is too large (%u tokens)", n);
    KV_ARG(kv_aligned(d_cache, 16) && kv_aligned(d_k, 16) && kv_aligned(d_v, 16) && kv_aligned(d_slots, 8), "kv_read: cache, k and v need 16-byte alignment, slots 8");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    KvDevice dev;
    ZV_CHECK(dev.enter(d_cache, s));
    const uint8_t *c = static_cast<const uint8_t *>(d_cache);
    const uint64_t *slots = static_cast<const uint64_t *>(d_slots);
    if (type == ZVDB_KV_F32) launch_read<float>(c, g, slots, n, d_k, d_v, s);
    else launch_read<uint16_t>(c, g, slots, n, d_k, d_v, s);
    ZV_HIP(hipGetLastError());
    return ZVDB_OK;
}

}  // extern "C"
