// kv_attend.hip -- attention over the 4-bit key/value cache (kv_cache.h): o = softmax(scale q K^T) V with one pass over K and V.
//
// Mathematics.  Rows are (token j, head g) pairs of one request and key/value head, 16 to a tile.  A wave takes 32 tokens at a
// time and forms both products TRANSPOSED with v_mfma_f32_16x16x32_bf16: S^T = K Q^T (A = 16 tokens x 32 elements of K) and
// O^T += V^T P^T (A = 16 columns x 32 tokens of V).  The accumulator of S^T then holds, in lane (row r = lane % 16, g = lane / 16),
// the scores of tokens 4 g .. 4 g + 3 of a tile, which is what the second product wants as its B operand -- its 32 tokens may stand
// in any order as long as both operands agree, so P goes from registers to registers and no LDS is touched in the loop.  Both the
// running maximum and the rescaling of O^T stay inside a lane's own row.
//
// Layout.  One 16-byte load (width 128) gives a lane 32 consecutive elements of one key: a whole scale block, in the element order
// that both operands of S^T agree on (group g of lanes owns the g-th quarter of the row).  One 16-byte load gives it 8 columns of
// four tokens of V, a 4-byte load their four scales.  v_cvt_scalef32_pk_bf16_fp4 applies the block's scale while it widens: a code
// times a power of two is a bf16 number, so K and V lose nothing on the way into the matrix instructions.
//
// Rounding.  bf16 queries: products and sums are fp32; P is rounded to bf16 (2^-9 relative, signs at random, below the rounding of
// the bf16 output), the sum of P is of the unrounded values.  fp32 queries: q and P are split into three bf16 terms each (24 bits,
// exact for q) and every product runs three times.
//
// The maximum is lazy: m moves only when a score exceeds it by more than 2^kSlack (a wave-wide vote, no exchange between lanes);
// exp2 arguments stay below kSlack, so sums of 2^31 tokens stay far inside fp32.
#include "kv_cache.h"

#include <algorithm>
#include <cfloat>

namespace zvdb {

struct KvAttendArgs {
    KvGeom g;
    const uint8_t *cache;
    const void *q;
    void *out;
    float *lse;
    const uint32_t *starts, *lengths, *tables;
    float *part;  // [rows][q heads][splits][dim + 2]: O (not divided), m, l
    const uint64_t *ids;
    const uint32_t *counts;
    uint64_t q_stride;
    float scale_log2;  // scale * log2(e)
    uint32_t table_stride, group, n, rows, max_new, max_length, split_tokens, splits, tiles, k;
    bool causal;
};

// Row tiles of a wave when a prompt gives every wave its own: as many as its registers hold beside two chunks of raw rows, with two waves on a SIMD
constexpr int wide_tiles(int nb, int terms) { return terms == 1 && nb <= 4 ? 3 : 1; }
constexpr float kSlack = 8.0f;
constexpr float kNone = -FLT_MAX;  // maximum of a row that has seen nothing: exp2(-inf - kNone) = 0, never NaN
constexpr float kLn2 = 0.693147180559945309f;

// one wave's 32 tokens, as loaded
template <int NB>
struct KvRaw {
    uint32_t k[2][NB], v[2][NB], ks[2], vs[2];
};

template <int N>
__device__ inline void load_words(uint32_t *dst, const uint8_t *p) {
    if constexpr (N == 2) {
        const uint2 u = *reinterpret_cast<const uint2 *>(p);
        dst[0] = u.x; dst[1] = u.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 u = *reinterpret_cast<const uint4 *>(p + 4 * i);
            dst[i] = u.x; dst[i + 1] = u.y; dst[i + 2] = u.z; dst[i + 3] = u.w;
        }
    }
}

// the scale bytes of the blocks that lane group g's part of a key row lies in: one byte, two at width 256
template <int NB>
__device__ inline uint32_t load_key_scales(const uint8_t *p, uint32_t g) {
    if constexpr (NB == 8) return *reinterpret_cast<const uint16_t *>(p + 2 * g);
    else return p[NB == 4 ? g : g / 2];
}

__device__ inline float pow2_of(uint32_t word, int byte) { return __uint_as_float(((word >> (8 * byte)) & 0xFFu) << 23); }

__device__ inline float max_over_row(float x) {  // over the four lanes of a row (lane, lane ^ 16, lane ^ 32, lane ^ 48)
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ inline float sum_over_row(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

template <int N>
__device__ inline void split_bf16(const float *x, bf16x8 *t) {  // x[8] = t[0] + t[1] + t[2] (N = 3), or rounded to t[0]
    float r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = x[j];
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            t[n][j] = (__bf16)r[j];
            if (n + 1 < N) r[j] -= (float)t[n][j];
        }
    }
}

// The state of NT tiles of 16 rows in a wave
template <int NB, int NT, int TERMS>
struct KvRows {
    bf16x8 q[NT][TERMS][NB];
    f32x4 o[NT][2 * NB];
    float m[NT], l[NT];
    uint32_t nan_at;  // smallest index of a token whose V block of this lane's columns is NaN

    __device__ void clear() {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int i = 0; i < 2 * NB; ++i) o[t][i] = f32x4{0, 0, 0, 0};
            m[t] = kNone;
            l[t] = 0;
        }
        nan_at = ~0u;
    }

    // row pointer of this lane's row of tile t (nullptr: no row): element j of step s is q[g * 8 NB + 8 s + j]
    __device__ void load_q(int t, const void *row, uint32_t dim) {
        const uint32_t g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int s = 0; s < NB; ++s) {
            const uint32_t d = (g * NB + s) * 8;
            const bool live = row && d < dim;
            if constexpr (TERMS == 1) {
                uint4 u = make_uint4(0, 0, 0, 0);
                if (live) u = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(row) + d);
                q[t][0][s] = __builtin_bit_cast(bf16x8, u);
            } else {
                float x[8] = {};
                if (live) {
                    const float4 a = *reinterpret_cast<const float4 *>(static_cast<const float *>(row) + d), b = *reinterpret_cast<const float4 *>(static_cast<const float *>(row) + d + 4);
                    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
                }
                bf16x8 y[TERMS];
                split_bf16<TERMS>(x, y);
#pragma unroll
                for (int n = 0; n < TERMS; ++n) q[t][n][s] = y[n];
            }
        }
    }

    // `seen(t, i, j)`: whether this lane's row of row tile t sees token 4 g + j of token tile i; asked only where `mask` (uniform).
    // `token(i, j)`: the index that nan_at counts of that token.
    template <class Seen, class Token>
    __device__ void step(const KvRaw<NB> &raw, float scale_log2, bool mask, Seen seen, Token token) {
        // V's scales; a NaN block counts as 0 here and is entered in nan_at, so that rows that do not see its token stay whole
        float vs[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) vs[j] = pow2_of(raw.vs[j / 4], j % 4);
        float top = vs[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, vs[j]);
        if (__any(top == INFINITY)) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (vs[j] == INFINITY) { vs[j] = 0.0f; nan_at = min(nan_at, token(j / 4, j % 4)); }
        }
        f32x4 s[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float ks = pow2_of(raw.ks[i], NB == 8 ? b / 4 : 0);
                const bf16x2 c0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(raw.k[i][b], ks, 0), c1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(raw.k[i][b], ks, 1),
                             c2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(raw.k[i][b], ks, 2), c3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(raw.k[i][b], ks, 3);
                const bf16x8 a = {c0[0], c0[1], c1[0], c1[1], c2[0], c2[1], c3[0], c3[1]};
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int n = TERMS - 1; n >= 0; --n) s[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q[t][n][b], s[t][i], 0, 0, 0);
            }
        bf16x8 p[NT][TERMS];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (mask) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!seen(t, j / 4, j % 4)) s[t][j / 4][j % 4] = -INFINITY;
            }
            float mx = s[t][0][0];
#pragma unroll
            for (int j = 1; j < 8; ++j) mx = fmaxf(mx, s[t][j / 4][j % 4]);
            mx *= scale_log2;
            if (__any(mx > m[t] + kSlack)) {
                const float to = fmaxf(m[t], max_over_row(mx)), by = __builtin_amdgcn_exp2f(m[t] - to);
                m[t] = to;
                l[t] *= by;
#pragma unroll
                for (int i = 0; i < 2 * NB; ++i) o[t][i] *= by;
            }
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = __builtin_amdgcn_exp2f(fmaf(s[t][j / 4][j % 4], scale_log2, -m[t]));
                l[t] += x[j];
            }
            split_bf16<TERMS>(x, p[t]);
        }
        // byte b of a piece holds columns 2 b and 2 b + 1 of one token: widen 8 tokens, then sort the pairs by column
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int byte = (j % 4) * NB + b;
                const uint32_t src = raw.v[j / 4][byte / 4];
                bf16x2 c;
                switch (byte % 4) {
                    case 0: c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(src, vs[j], 0); break;
                    case 1: c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(src, vs[j], 1); break;
                    case 2: c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(src, vs[j], 2); break;
                    default: c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(src, vs[j], 3); break;
                }
                w[j] = __builtin_bit_cast(uint32_t, c);
            }
            uint4 lo, hi;
            lo.x = __builtin_amdgcn_perm(w[1], w[0], 0x05040100u); hi.x = __builtin_amdgcn_perm(w[1], w[0], 0x07060302u);
            lo.y = __builtin_amdgcn_perm(w[3], w[2], 0x05040100u); hi.y = __builtin_amdgcn_perm(w[3], w[2], 0x07060302u);
            lo.z = __builtin_amdgcn_perm(w[5], w[4], 0x05040100u); hi.z = __builtin_amdgcn_perm(w[5], w[4], 0x07060302u);
            lo.w = __builtin_amdgcn_perm(w[7], w[6], 0x05040100u); hi.w = __builtin_amdgcn_perm(w[7], w[6], 0x07060302u);
            const bf16x8 a0 = __builtin_bit_cast(bf16x8, lo), a1 = __builtin_bit_cast(bf16x8, hi);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int n = TERMS - 1; n >= 0; --n) {
                    o[t][2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, p[t][n], o[t][2 * b], 0, 0, 0);
                    o[t][2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, p[t][n], o[t][2 * b + 1], 0, 0, 0);
                }
        }
    }

    __device__ void close() {  // sums of a row's four lanes
#pragma unroll
        for (int t = 0; t < NT; ++t) l[t] = sum_over_row(l[t]);
    }
};

// Column block of V that lane `row` c of the A operand loads (its 2 NB columns lie in one block of 32), and the block of accumulator
// element i of lane group g: columns (4 g + i) 2 NB ...
template <int NB>
__device__ inline uint32_t v_block(uint32_t c) { return c * NB / 16; }

// Smallest nan_at over all lanes that loaded block v_block(4 g + i), for each i (all 64 lanes call this)
template <int NB>
__device__ inline void nan_blocks(uint32_t nan_at, uint32_t *first) {
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4;
    if (!__any(nan_at != ~0u)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) first[i] = ~0u;
        return;
    }
    uint32_t x = nan_at;  // over the lane groups (other tokens, same columns)
    x = min(x, (uint32_t)__shfl_xor((int)x, 16));
    x = min(x, (uint32_t)__shfl_xor((int)x, 32));
    // (lanes of one block hold the same bytes: one of them speaks for all)
#pragma unroll
    for (int i = 0; i < 4; ++i) first[i] = (uint32_t)__shfl((int)x, (int)(4 * g + i));
}

// Stores one row's 2 NB columns from d on (a multiple of 4 elements, head_dim of 8)
template <int NB, int TERMS>
__device__ inline void store_columns(void *row, uint32_t d, uint32_t dim, const float *x) {
    constexpr int N = 2 * NB, STEP = N < 8 ? N : 8;
#pragma unroll
    for (int e = 0; e < N; e += STEP) {
        if (d + e >= dim) break;
        if constexpr (TERMS == 1) {
            uint32_t w[STEP / 2];
#pragma unroll
            for (int j = 0; j < STEP / 2; ++j) {
                const bf16x2 y = {(__bf16)x[e + 2 * j], (__bf16)x[e + 2 * j + 1]};
                w[j] = __builtin_bit_cast(uint32_t, y);
            }
            uint16_t *p = static_cast<uint16_t *>(row) + d + e;
            if constexpr (STEP == 4) *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            float *p = static_cast<float *>(row) + d + e;
#pragma unroll
            for (int j = 0; j < STEP; j += 4) *reinterpret_cast<float4 *>(p + j) = make_float4(x[e + j], x[e + j + 1], x[e + j + 2], x[e + j + 3]);
        }
    }
}

__device__ inline float lse_of(float m, float l) { return (m + __log2f(l)) * kLn2; }

// Joins the four waves of a block, each with its own tokens, in wave 0 (all 256 threads call this).  Sums in a fixed order.
template <int NB, int TERMS>
__device__ inline void join_waves(KvRows<NB, 1, TERMS> &r) {
    __shared__ float ml[4][2][16];
    __shared__ f32x4 buf[2][2 * NB][64];
    __shared__ uint32_t nan[4][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane < 16) { ml[wave][0][lane] = r.m[0]; ml[wave][1][lane] = r.l[0]; }
    nan[wave][lane] = r.nan_at;
    __syncthreads();
    const uint32_t row = lane & 15;
    const float m = fmaxf(fmaxf(ml[0][0][row], ml[1][0][row]), fmaxf(ml[2][0][row], ml[3][0][row]));
    float l = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) l += ml[w][1][row] * __builtin_amdgcn_exp2f(ml[w][0][row] - m);
    const float by = __builtin_amdgcn_exp2f(r.m[0] - m);
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) r.o[0][i] *= by;
    if (wave >= 2)
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) buf[wave - 2][i][lane] = r.o[0][i];
    __syncthreads();
    if (wave < 2)
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) r.o[0][i] += buf[wave][i][lane];
    __syncthreads();
    if (wave == 1)
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) buf[0][i][lane] = r.o[0][i];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) r.o[0][i] += buf[0][i][lane];
        r.m[0] = m;
        r.l[0] = l;
        r.nan_at = min(min(nan[0][lane], nan[1][lane]), min(nan[2][lane], nan[3][lane]));
    }
}

// ---- attention over whole requests --------------------------------------------------------------------------------------

// A block takes row tile(s) x one key/value head x one split of the tokens of a request.  WIDE = false (few rows: decode): its four
// waves share 16 rows and divide the split's tokens, joined in LDS.  WIDE = true (prompts): each wave has NT tiles of its own and
// walks the same tokens.  Blocks are numbered head first, so that (with 8 heads) an XCD's L2 keeps the pages of its own heads,
// and row tiles last to first, so that the causal ones with most tokens start first.  The requests turn by one from one tile or split to
// the next: blocks are dealt to the shader engines in order, and without it one of them gets all of a long request (4 prompts: 465 us, a
// third of the wave slots empty).
template <int NB, int NT, int TERMS, bool WIDE>
__global__ __launch_bounds__(256, NB == 8 && TERMS == 3 ? 1 : WIDE || NB == 8 || TERMS == 3 ? 2 : 4) void k_kv_attend(const KvAttendArgs a) {
    static_assert(WIDE || NT == 1, "waves that share rows hold one tile");
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    uint32_t b = blockIdx.x;
    const uint32_t head = b % a.g.heads;
    b /= a.g.heads;
    const uint32_t turn = b / a.n, i = (b + turn) % a.n, split = turn % a.splits, tile = a.tiles - 1 - turn / a.splits;

    // the request: rows [first, first + count) of q, `length` tokens, of which those up to `end` are reachable
    const uint32_t first = min(a.starts[i], a.rows), next = min(a.starts[i + 1], a.rows), count = next > first ? next - first : 0;
    const uint32_t length = a.lengths[i];
    const uint32_t reach = (uint32_t)min((uint64_t)min(length, a.max_length), (uint64_t)a.table_stride << a.g.page_shift);
    const uint32_t rows = min(count, a.max_new) * a.group;
    constexpr uint32_t kWaveRows = 16 * NT;
    const uint32_t block_row = tile * (WIDE ? 4 * kWaveRows : 16);
    if (block_row >= rows) return;
    const uint32_t wave_row = block_row + (WIDE ? wave * kWaveRows : 0);
    // a row's limit: the tokens it sees are [0, limit)
    auto limit_of = [&](uint32_t row) {
        if (!a.causal) return reach;
        const int64_t x = (int64_t)length - count + row / a.group + 1;
        return (uint32_t)min(max(x, (int64_t)0), (int64_t)reach);
    };
    const uint32_t block_end = limit_of(min(block_row + (WIDE ? 4 * kWaveRows : 16), rows) - 1);
    uint32_t t0 = split * a.split_tokens;
    if (a.splits > 1 && t0 >= block_end) return;  // (no row of the block sees a token of this split: k_kv_join knows)
    uint32_t t1 = a.splits > 1 ? min(t0 + a.split_tokens, block_end) : block_end;
    if (WIDE) {
        if (wave_row >= rows) return;
        t1 = min(t1, limit_of(min(wave_row + kWaveRows, rows) - 1));
    } else {  // this wave's quarter, in whole chunks
        const uint32_t part = ((t1 - t0 + 127) >> 7) << 5;
        t0 = min(t0 + wave * part, t1);
        t1 = min(t0 + part, t1);
    }

    KvRows<NB, NT, TERMS> r;
    r.clear();
    uint32_t limit[NT];
    const uint32_t qheads = a.g.heads * a.group;
    constexpr uint32_t kSize = TERMS == 1 ? 2 : 4;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const uint32_t row = wave_row + t * 16 + (lane & 15);
        limit[t] = row < rows ? limit_of(row) : 0;
        const uint8_t *p = static_cast<const uint8_t *>(a.q) + ((uint64_t)(first + row / a.group) * a.q_stride + (uint64_t)(head * a.group + row % a.group) * a.g.dim) * kSize;
        r.load_q(t, row < rows ? p : nullptr, a.g.dim);
    }
    const uint32_t all_see = __builtin_amdgcn_readfirstlane(limit_of(min(wave_row, rows - 1)));  // rows behind the last one do not count: they are not stored
    uint32_t seen_from = ~0u;  // first token of the first page that is there

    if (t0 < t1) {
        const uint32_t *table = a.tables + (uint64_t)i * a.table_stride;
        const uint32_t last_page = (t1 - 1) >> a.g.page_shift, half = a.g.page_size * 16 * NB, mask = a.g.page_size - 1;
        const uint8_t *heads = a.cache + (uint64_t)head * a.g.head_bytes;
        const uint32_t chunks = (t1 - t0 + 31) >> 5;
        auto page_of = [&](uint32_t t) { return table[min(t >> a.g.page_shift, last_page)]; };
        // what a lane adds to a tile's place: the rest of an address is uniform
        const uint32_t key_at = (lane & 15) * (16 * NB) + g * (4 * NB), key_scale_at = (lane & 15) * NB, val_at = g * (64 * NB) + (lane & 15) * (4 * NB),
                       val_scale_at = g * (4 * NB) + v_block<NB>(lane & 15) * 4;
        auto load = [&](KvRaw<NB> &raw, uint32_t t, const uint32_t *page) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint8_t *p = heads + (uint64_t)(page[x] < a.g.pages ? page[x] : 0) * a.g.page_bytes;
                const uint32_t in = (t + 16 * x) & mask;
                const uint8_t *keys = p + in * (16 * NB), *vals = keys + half, *scales = p + 2 * half + in * NB;
                load_words<NB>(raw.k[x], keys + key_at);
                raw.ks[x] = load_key_scales<NB>(scales + key_scale_at, g);
                load_words<NB>(raw.v[x], vals + val_at);
                raw.vs[x] = *reinterpret_cast<const uint32_t *>(scales + a.g.page_size * NB + val_scale_at);
            }
        };
        auto work = [&](KvRaw<NB> &raw, uint32_t t, const uint32_t *page) {
            const bool there[2] = {page[0] < a.g.pages, page[1] < a.g.pages};
            const bool part = !(there[0] && there[1] && t + 32 <= t1);  // some token is none
            if (there[0]) seen_from = min(seen_from, t);
            else if (there[1]) seen_from = min(seen_from, t + 16);
            if (part) {
                // scales of tokens that are not there (or not in this part): whatever lies in the page must not turn 0 into NaN
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const uint32_t at = t + 16 * x + 4 * g, live = !there[x] || at >= t1 ? 0 : min(t1 - at, 4u);
                    if (live < 4) raw.vs[x] &= (1u << (8 * live)) - 1;
                }
            }
            r.step(raw, a.scale_log2, part || t + 32 > all_see,
                   [&](int row_tile, int x, int j) { const uint32_t at = t + 16 * x + 4 * g + j; return there[x] && at < limit[row_tile] && at < t1; },
                   [&](int x, int j) { return t + 16 * x + 4 * g + j; });
        };
        KvRaw<NB> cur, nxt;
        uint32_t page[2] = {page_of(t0), page_of(t0 + 16)};
        load(cur, t0, page);
        for (uint32_t c = 0; c < chunks; ++c) {
            const uint32_t t = t0 + c * 32, tn = min(t + 32, t0 + (chunks - 1) * 32);
            const uint32_t pn[2] = {page_of(tn), page_of(tn + 16)};
            load(nxt, tn, pn);
            work(cur, t, page);
            cur = nxt;
            page[0] = pn[0];
            page[1] = pn[1];
        }
    }
    r.close();
    if constexpr (!WIDE) {
        __shared__ uint32_t from[4];
        if (lane == 0) from[wave] = seen_from;
        join_waves<NB, TERMS>(r);
        if (wave != 0) return;
        seen_from = min(min(from[0], from[1]), min(from[2], from[3]));
    }
    uint32_t nan_first[4];
    nan_blocks<NB>(r.nan_at, nan_first);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const uint32_t row = wave_row + t * 16 + (lane & 15);
        if (row >= rows) continue;
        const uint64_t out_row = (uint64_t)(first + row / a.group) * qheads + head * a.group + row % a.group;
        const bool some = seen_from < limit[t];
        const bool whole = a.splits == 1;
        const float by = whole ? (some ? 1.0f / r.l[t] : 0.0f) : 1.0f;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            float y[2 * NB];
#pragma unroll
            for (int e = 0; e < 2 * NB; ++e) y[e] = nan_first[x] < limit[t] ? __uint_as_float(0x7FC00000u) : r.o[t][e][x] * by;
            const uint32_t d = (4 * g + x) * 2 * NB;
            if (whole) store_columns<NB, TERMS>(static_cast<uint8_t *>(a.out) + out_row * a.g.dim * kSize, d, a.g.dim, y);
            else store_columns<NB, 3>(a.part + (out_row * a.splits + split) * (a.g.dim + 4), d, a.g.dim, y);
        }
        if (g == 0) {
            if (!whole) {
                float *p = a.part + (out_row * a.splits + split) * (a.g.dim + 4) + a.g.dim;
                p[0] = some ? r.m[t] : -INFINITY;  // -inf: this split saw nothing
                p[1] = r.l[t];
            } else if (a.lse) {
                a.lse[out_row] = some ? lse_of(r.m[t], r.l[t]) : -INFINITY;
            }
        }
    }
}

// Joins the splits (at most 256) of a row, one block for a (row, head): a thread for each split's maximum and sum, then four columns and
// every (1024 / W)-th split to a thread.  The order of the sums depends on the sizes alone.  Latency of three dependent reads: the first
// parts are on their way before the weights are known.
template <int W, int TERMS>
__global__ __launch_bounds__(256) void k_kv_join(const KvAttendArgs a) {
    constexpr uint32_t COLS = W / 4, LANES = 256 / COLS, AHEAD = 2;
    __shared__ float weight[256], red[2][4];
    __shared__ float4 sum[LANES][COLS];
    const uint32_t tid = threadIdx.x, qheads = a.g.heads * a.group, head = blockIdx.x % qheads, i = blockIdx.x / qheads % a.n, j = blockIdx.x / qheads / a.n;
    const uint32_t first = min(a.starts[i], a.rows), next = min(a.starts[i + 1], a.rows), count = next > first ? next - first : 0;
    if (j >= count) return;
    const uint32_t length = a.lengths[i];
    const uint32_t reach = (uint32_t)min((uint64_t)min(length, a.max_length), (uint64_t)a.table_stride << a.g.page_shift);
    uint32_t limit = reach;
    if (a.causal) limit = (uint32_t)min(max((int64_t)length - count + (int64_t)j + 1, (int64_t)0), (int64_t)reach);
    const uint64_t row = (uint64_t)(first + j) * qheads + head;
    const uint32_t live = min((limit + a.split_tokens - 1) / a.split_tokens, a.splits), step = a.g.dim + 4;
    const float *part = a.part + row * a.splits * step;
    const uint32_t lane = tid / COLS, d = tid % COLS * 4;
    const bool mine = d < a.g.dim;
    float4 ahead[AHEAD] = {};
#pragma unroll
    for (uint32_t u = 0; u < AHEAD; ++u)
        if (mine && lane + u * LANES < live) ahead[u] = *reinterpret_cast<const float4 *>(part + (lane + u * LANES) * step + d);
    const float ms = tid < live ? part[tid * step + a.g.dim] : -INFINITY, ls = tid < live ? part[tid * step + a.g.dim + 1] : 0.0f;
    float m = ms;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
    if ((tid & 63) == 0) red[0][tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float w = ms == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms - m);  // (-inf: the split saw nothing and left nothing)
    weight[tid] = w;
    float l = ms == -INFINITY ? 0.0f : ls * w;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) l += __shfl_xor(l, x);
    if ((tid & 63) == 0) red[1][tid >> 6] = l;
    __syncthreads();
    float4 o = make_float4(0, 0, 0, 0);
    auto add = [&](const float4 &x, uint32_t s) {
        const float by = weight[s];
        if (by != 0.0f) { o.x += x.x * by; o.y += x.y * by; o.z += x.z * by; o.w += x.w * by; }
    };
    if (mine) {
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; ++u)
            if (lane + u * LANES < live) add(ahead[u], lane + u * LANES);
#pragma unroll 4
        for (uint32_t s = lane + AHEAD * LANES; s < live; s += LANES) add(*reinterpret_cast<const float4 *>(part + s * step + d), s);
    }
    sum[lane][tid % COLS] = o;
    __syncthreads();
    if (lane != 0) return;
#pragma unroll
    for (uint32_t u = 1; u < LANES; ++u) {
        const float4 x = sum[u][tid % COLS];
        o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
    }
    l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    const bool some = m != -INFINITY;
    const float by = some ? 1.0f / l : 0.0f;
    const float y[4] = {o.x * by, o.y * by, o.z * by, o.w * by};
    constexpr uint32_t kSize = TERMS == 1 ? 2 : 4;
    if (mine) store_columns<2, TERMS>(static_cast<uint8_t *>(a.out) + row * a.g.dim * kSize, d, a.g.dim, y);
    if (tid == 0 && a.lse) a.lse[row] = some ? lse_of(m, l) : -INFINITY;
}

// ---- attention over selected rows ---------------------------------------------------------------------------------------

// A block takes one request and key/value head: its list of ids is resolved to rows of the cache in LDS (a search's ids and counts
// as zvdb_hip_search_*_dev writes them), then its four waves take 32 entries at a time.
constexpr uint32_t kSelPass = 1024;  // entries resolved at a time

template <int NB, int TERMS>
__global__ __launch_bounds__(256) void k_kv_attend_selected(const KvAttendArgs a) {
    __shared__ uint64_t rows_at[kSelPass];  // page << 8 | token in it; ~0: not there
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    const uint32_t head = blockIdx.x % a.g.heads, b = blockIdx.x / a.g.heads, i = b % a.n, tile = b / a.n;
    const uint32_t qheads = a.g.heads * a.group, length = a.lengths[i];
    const uint32_t reach = (uint32_t)min((uint64_t)length, (uint64_t)a.table_stride << a.g.page_shift);
    const uint64_t list = (uint64_t)head * a.n + i;
    const uint32_t entries = min(a.counts ? a.counts[list] : a.k, a.k);
    constexpr uint32_t kSize = TERMS == 1 ? 2 : 4;
    const uint32_t row = tile * 16 + (lane & 15);
    KvRows<NB, 1, TERMS> r;
    r.clear();
    r.load_q(0, row < a.group ? static_cast<const uint8_t *>(a.q) + ((uint64_t)i * a.q_stride + (uint64_t)(head * a.group + row) * a.g.dim) * kSize : nullptr, a.g.dim);
    const uint32_t half = a.g.page_size * 16 * NB, mask = a.g.page_size - 1;
    const uint8_t *heads = a.cache + (uint64_t)head * a.g.head_bytes;
    bool any = false;
    for (uint32_t e0 = 0; e0 < entries; e0 += kSelPass) {
        const uint32_t m = min(entries - e0, kSelPass);
        if (e0) __syncthreads();
        for (uint32_t e = threadIdx.x; e < kSelPass && e < ((m + 31) & ~31u); e += 256) {
            uint64_t at = ~0ull;
            const uint64_t id = e < m ? a.ids[list * a.k + e0 + e] : ~0ull;
            if (id < reach) {
                const uint32_t page = a.tables[(uint64_t)i * a.table_stride + (uint32_t)(id >> a.g.page_shift)];
                if (page < a.g.pages) at = (uint64_t)page << 8 | (id & mask);
            }
            rows_at[e] = at;
        }
        __syncthreads();
        for (uint32_t e = wave * 32; e < m; e += 128) {
            KvRaw<NB> raw;
            bool seen[8];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint64_t key = rows_at[e + 16 * x + (lane & 15)];
                const uint32_t tok = (uint32_t)key & 0xFF;
                const uint8_t *p = heads + (key == ~0ull ? 0 : (key >> 8) * a.g.page_bytes);
                const uint32_t kt = key == ~0ull ? 0 : tok;
                load_words<NB>(raw.k[x], p + kt * (16 * NB) + g * (4 * NB));
                raw.ks[x] = load_key_scales<NB>(p + 2 * half + kt * NB, g);
                raw.vs[x] = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint64_t val = rows_at[e + 16 * x + 4 * g + j];
                    seen[4 * x + j] = val != ~0ull;
                    const uint32_t vt = val == ~0ull ? 0 : (uint32_t)val & 0xFF;
                    const uint8_t *w = heads + (val == ~0ull ? 0 : (val >> 8) * a.g.page_bytes);
                    const uint8_t *piece = w + half + kv_v_offset<NB>(vt, lane & 15);
                    if constexpr (NB == 2) {
                        const uint32_t u = *reinterpret_cast<const uint16_t *>(piece);
                        if (j % 2 == 0) raw.v[x][j / 2] = u;
                        else raw.v[x][j / 2] |= u << 16;
                    } else if constexpr (NB == 4) {
                        raw.v[x][j] = *reinterpret_cast<const uint32_t *>(piece);
                    } else {
                        load_words<2>(raw.v[x] + 2 * j, piece);
                    }
                    const uint32_t s = w[2 * half + a.g.page_size * NB + (vt >> 2) * (4 * NB) + v_block<NB>(lane & 15) * 4 + (vt & 3)];
                    raw.vs[x] |= (val == ~0ull ? 0u : s) << (8 * j);
                    any |= seen[4 * x + j];
                }
            }
            r.step(raw, a.scale_log2, true, [&](int, int x, int j) { return seen[4 * x + j]; }, [](int, int) { return 0u; });
        }
    }
    r.close();
    const bool some = __syncthreads_or(any);
    join_waves<NB, TERMS>(r);
    if (wave != 0) return;
    uint32_t nan_first[4];
    nan_blocks<NB>(r.nan_at, nan_first);
    if (row >= a.group) return;
    const uint64_t out_row = (uint64_t)i * qheads + head * a.group + row;
    const float by = some ? 1.0f / r.l[0] : 0.0f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        float y[2 * NB];
#pragma unroll
        for (int e = 0; e < 2 * NB; ++e) y[e] = nan_first[x] == 0 ? __uint_as_float(0x7FC00000u) : r.o[0][e][x] * by;
        store_columns<NB, TERMS>(static_cast<uint8_t *>(a.out) + out_row * a.g.dim * kSize, (4 * g + x) * 2 * NB, a.g.dim, y);
    }
    if (g == 0 && a.lse) a.lse[out_row] = some ? lse_of(r.m[0], r.l[0]) : -INFINITY;
}

// ---- launches -----------------------------------------------------------------------------------------------------------

// How a call is cut.  Rows of one (request, head) that fit 64 are few: blocks of 16 whose waves divide the tokens; more of them give
// each wave its own tiles.  The tokens are split until the card has work for all its units, in parts of whole chunks.
struct KvCut {
    bool wide;
    uint32_t nt, tiles, splits, split_tokens;
    uint64_t blocks;
};

static KvCut kv_cut(const KvGeom &g, uint32_t type, uint32_t group, uint32_t n, uint32_t max_new, uint32_t max_length, int cus) {
    KvCut c;
    const uint64_t rows = (uint64_t)max_new * group;
    const uint32_t w = kv_width(g.dim);
    c.wide = rows > 64;
    c.nt = c.wide ? wide_tiles(w / 32, type == ZVDB_KV_F32 ? 3 : 1) : 1;
    const uint32_t block_rows = c.wide ? 64 * c.nt : 16;
    c.tiles = (uint32_t)((rows + block_rows - 1) / block_rows);
    const uint64_t base = (uint64_t)g.heads * n * c.tiles;
    const uint64_t want = (uint64_t)cus * (c.wide ? 4 : 8);  // blocks the card should have
    uint64_t splits = base ? (want + base - 1) / base : 1;
    const uint32_t least = c.wide ? 256 : 128;
    splits = std::min<uint64_t>(splits, ((uint64_t)max_length + least - 1) / least);
    splits = std::max<uint64_t>(std::min<uint64_t>(splits, 256), 1);
    c.split_tokens = (uint32_t)std::max<uint64_t>((((uint64_t)max_length + splits - 1) / splits + 127) / 128 * 128, 128);
    c.splits = (uint32_t)std::max<uint64_t>(((uint64_t)max_length + c.split_tokens - 1) / c.split_tokens, 1);
    c.blocks = base * c.splits;
    return c;
}

template <int NB>
static void launch_attend(const KvAttendArgs &a, const KvCut &c, uint32_t type, hipStream_t s) {
    const dim3 grid((uint32_t)c.blocks), block(256);
    if (type == ZVDB_KV_F32) {
        if (c.wide) hipLaunchKernelGGL((k_kv_attend<NB, wide_tiles(NB, 3), 3, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((k_kv_attend<NB, 1, 3, false>), grid, block, 0, s, a);
    } else {
        if (c.wide) hipLaunchKernelGGL((k_kv_attend<NB, wide_tiles(NB, 1), 1, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((k_kv_attend<NB, 1, 1, false>), grid, block, 0, s, a);
    }
}

template <int W>
static void launch_join(const KvAttendArgs &a, uint32_t blocks, uint32_t type, hipStream_t s) {
    if (type == ZVDB_KV_F32) hipLaunchKernelGGL((k_kv_join<W, 3>), dim3(blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_kv_join<W, 1>), dim3(blocks), dim3(256), 0, s, a);
}

template <int NB>
static void launch_selected(const KvAttendArgs &a, uint32_t blocks, uint32_t type, hipStream_t s) {
    if (type == ZVDB_KV_F32) hipLaunchKernelGGL((k_kv_attend_selected<NB, 3>), dim3(blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_kv_attend_selected<NB, 1>), dim3(blocks), dim3(256), 0, s, a);
}

static int check_queries(const KvGeom &g, const void *q, uint64_t q_stride, uint32_t type, uint32_t q_heads, float scale, const void *out, const void *cache) {
    KV_ARG(q && out && cache, "null argument");
    KV_ARG(kv_aligned(q, 16) && kv_aligned(out, 16) && kv_aligned(cache, 16), "kv_attend: cache, q and out need 16-byte alignment");
    KV_ARG(q_stride >= (uint64_t)q_heads * g.dim && q_stride % 8 == 0, "kv_attend: a token's stride is at least q_heads * head_dim and a multiple of 8");
    KV_ARG(scale > 0.0f && scale <= FLT_MAX, "kv_attend: scale %g (positive and finite)", (double)scale);
    (void)type;
    return ZVDB_OK;
}

static int check_heads(const KvGeom &g, uint32_t type, uint32_t q_heads) {
    KV_ARG(type == ZVDB_KV_F32 || type == ZVDB_KV_BF16, "kv_attend: type %u", type);
    KV_ARG(q_heads >= g.heads && q_heads <= 65536 && q_heads % g.heads == 0, "kv_attend: %u query heads over %u key/value heads", q_heads, g.heads);
    return ZVDB_OK;
}

static int attend_shape(const KvGeom &g, uint32_t type, uint32_t q_heads, uint32_t n, uint32_t rows, uint32_t max_new, uint32_t max_length) {
    ZV_CHECK(check_heads(g, type, q_heads));
    KV_ARG(n < (1u << 24) && rows < 0x7FFFFFFFu && max_new < 0x7FFFFFFFu && max_length < 0x7FFFFFFFu, "kv_attend: a size is out of range");
    return ZVDB_OK;
}

static int device_cus(int *out) {
    int dev = 0, n = 0;
    if (hipGetDeviceCount(&n) != hipSuccess || n == 0) {
        (void)hipGetLastError();
        set_error("no HIP device");
        return ZVDB_ERR_NO_DEVICE;
    }
    ZV_HIP(hipGetDevice(&dev));
    ZV_HIP(hipDeviceGetAttribute(out, hipDeviceAttributeMultiprocessorCount, dev));
    return ZVDB_OK;
}

}  // namespace zvdb

using namespace zvdb;

extern "C" {

int zvdb_hip_kv_attend_workspace(const zvdb_hip_kv_layout *layout, uint32_t type, uint32_t q_heads, uint32_t n, uint32_t rows, uint32_t max_new, uint32_t max_length,
                                 uint64_t *out_bytes) {
    KvGeom g;
    ZV_CHECK(kv_check_layout(layout, &g));
    KV_ARG(out_bytes, "null argument");
    ZV_CHECK(attend_shape(g, type, q_heads, n, rows, max_new, max_length));
    int cus = 0;
    ZV_CHECK(device_cus(&cus));
    const KvCut c = kv_cut(g, type, q_heads / g.heads, n, std::min(max_new, rows), max_length, cus);
    *out_bytes = c.splits > 1 ? (uint64_t)rows * q_heads * c.splits * (g.dim + 4) * 4 : 0;
    return ZVDB_OK;
}

int zvdb_hip_kv_attend_dev(const zvdb_hip_kv_layout *layout, const void *d_cache, const void *d_q, uint64_t q_stride, uint32_t type, uint32_t q_heads, uint32_t n,
                           const void *d_starts, uint32_t rows, uint32_t max_new, const void *d_lengths, const void *d_tables, uint32_t table_stride,
                           uint32_t max_length, float scale, uint32_t causal, void *d_workspace, uint64_t workspace_bytes, void *d_out, void *d_lse, void *stream) {
    KvAttendArgs a = {};
    ZV_CHECK(kv_check_layout(layout, &a.g));
    ZV_CHECK(attend_shape(a.g, type, q_heads, n, rows, max_new, max_length));
    max_new = std::min(max_new, rows);
    if (n == 0 || max_new == 0) return ZVDB_OK;
    ZV_CHECK(check_queries(a.g, d_q, q_stride, type, q_heads, scale, d_out, d_cache));
    KV_ARG(d_starts && d_lengths && d_tables, "null argument");
    KV_ARG(table_stride >= 1 && table_stride < 0x7FFFFFFFu, "kv_attend: table_stride %u", table_stride);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    KvDevice dev;
    ZV_CHECK(dev.enter(d_cache, s));
    const KvCut c = kv_cut(a.g, type, q_heads / a.g.heads, n, max_new, max_length, dev.cus());
    KV_ARG(c.blocks < 0x7FFFFFFFull, "kv_attend: the call is too large (%llu blocks)", (unsigned long long)c.blocks);
    const uint64_t need = c.splits > 1 ? (uint64_t)rows * q_heads * c.splits * (a.g.dim + 4) * 4 : 0;
    KV_ARG(workspace_bytes >= need && (need == 0 || (d_workspace && kv_aligned(d_workspace, 16))), "kv_attend: workspace %llu bytes, need %llu, 16-byte aligned",
           (unsigned long long)workspace_bytes, (unsigned long long)need);
    a.cache = static_cast<const uint8_t *>(d_cache);
    a.q = d_q;
    a.out = d_out;
    a.lse = static_cast<float *>(d_lse);
    a.starts = static_cast<const uint32_t *>(d_starts);
    a.lengths = static_cast<const uint32_t *>(d_lengths);
    a.tables = static_cast<const uint32_t *>(d_tables);
    a.part = static_cast<float *>(d_workspace);
    a.q_stride = q_stride;
    a.scale_log2 = scale * 1.44269504088896341f;
    a.table_stride = table_stride;
    a.group = q_heads / a.g.heads;
    a.n = n; a.rows = rows; a.max_new = max_new; a.max_length = max_length;
    a.split_tokens = c.split_tokens; a.splits = c.splits; a.tiles = c.tiles;
    a.causal = causal != 0;
    const uint32_t w = kv_width(a.g.dim);
    if (w == 64) launch_attend<2>(a, c, type, s);
    else if (w == 128) launch_attend<4>(a, c, type, s);
    else launch_attend<8>(a, c, type, s);
    ZV_HIP(hipGetLastError());
    if (c.splits > 1) {
        const uint64_t blocks = (uint64_t)q_heads * n * max_new;
        KV_ARG(blocks < 0x7FFFFFFFull, "kv_attend: the call is too large (%llu rows)", (unsigned long long)blocks);
        if (w == 64) launch_join<64>(a, (uint32_t)blocks, type, s);
        else if (w == 128) launch_join<128>(a, (uint32_t)blocks, type, s);
        else launch_join<256>(a, (uint32_t)blocks, type, s);
        ZV_HIP(hipGetLastError());
    }
    return ZVDB_OK;
}

int zvdb_hip_kv_attend_selected_dev(const zvdb_hip_kv_layout *layout, const void *d_cache, const void *d_q, uint64_t q_stride, uint32_t type, uint32_t q_heads,
                                    uint32_t n, const void *d_ids, const void *d_count, uint32_t k, const void *d_lengths, const void *d_tables,
                                    uint32_t table_stride, float scale, void *d_out, void *d_lse, void *stream) {
    KvAttendArgs a = {};
    ZV_CHECK(kv_check_layout(layout, &a.g));
    ZV_CHECK(attend_shape(a.g, type, q_heads, n, n, 1, 1));
    if (n == 0) return ZVDB_OK;
    ZV_CHECK(check_queries(a.g, d_q, q_stride, type, q_heads, scale, d_out, d_cache));
    KV_ARG(d_lengths && d_tables && (k == 0 || d_ids), "null argument");
    KV_ARG(kv_aligned(d_ids, 8), "kv_attend_selected: ids are not 8-byte aligned");
    KV_ARG(k < 0x7FFFFFFFu, "kv_attend_selected: k %u", k);
    KV_ARG(table_stride >= 1 && table_stride < 0x7FFFFFFFu, "kv_attend_selected: table_stride %u", table_stride);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    KvDevice dev;
    ZV_CHECK(dev.enter(d_cache, s));
    a.cache = static_cast<const uint8_t *>(d_cache);
    a.q = d_q;
    a.out = d_out;
    a.lse = static_cast<float *>(d_lse);
    a.lengths = static_cast<const uint32_t *>(d_lengths);
    a.tables = static_cast<const uint32_t *>(d_tables);
    a.ids = static_cast<const uint64_t *>(d_ids);
    a.counts = static_cast<const uint32_t *>(d_count);
    a.q_stride = q_stride;
    a.scale_log2 = scale * 1.44269504088896341f;
    a.table_stride = table_stride;
    a.group = q_heads / a.g.heads;
    a.n = n; a.k = k;
    const uint64_t blocks = (uint64_t)a.g.heads * n * ((a.group + 15) / 16);
    KV_ARG(blocks < 0x7FFFFFFFull, "kv_attend_selected: the call is too large (%llu blocks)", (unsigned long long)blocks);
    const uint32_t w = kv_width(a.g.dim);
    if (w == 64) launch_selected<2>(a, (uint32_t)blocks, type, s);
    else if (w == 128) launch_selected<4>(a, (uint32_t)blocks, type, s);
    else launch_selected<8>(a, (uint32_t)blocks, type, s);
    ZV_HIP(hipGetLastError());
    return ZVDB_OK;
}

}  // extern "C"
