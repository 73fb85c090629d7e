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
// Rounding.  bf16 queries: products and sums are fp32; P is rounded to bf16 for its product with V (at most 2^-8 of each weight, as the
// output's own rounding, and at random: 2.1e-3 off the 64-bit result in norm where rounding the exact result alone is 1.7e-3), the sum of
// P is of the unrounded values.  fp32 queries: q and P are split into three bf16 terms each (24 bits,
// exact for q) and every product runs three times.
//
// The maximum is lazy: it moves only when a score exceeds it by more than kSlack (a wave-wide vote, no exchange between lanes).  m lies
// `lift` = kSlack + log2(tokens) above it, so that no weight is over 1 / tokens and no sum of weights times values, in a wave, a split or a join, is over
// the largest of the values: they go up to 6 x 2^125.  What it costs lies at the other end: products under 2^-126 lose bits, 2^(lift - 149) of
// each in the result, which is 2^-128 over 8,192 tokens.
#include "kv_cache.h"
#include "wave_select.h"

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
    float *part;  // [rows][q heads][splits][dim + 4]: O (not divided), m, l
    const uint64_t *ids;
    const uint32_t *counts;
    uint64_t q_stride;
    float scale_log2;  // scale * log2(e)
    float lift;
    uint32_t table_stride, group, n, rows, max_new, max_length, split_tokens, splits, tiles, k;
    bool causal, by_tile;
};

constexpr float kSlack = 8.0f;
inline float kv_lift(uint32_t tokens) { return kSlack + (tokens > 1 ? 32 - __builtin_clz(tokens - 1) : 0); }
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

// the scale bytes of the blocks that a lane group's part of a key row lies in: one byte, two at width 256
template <int NB>
__device__ inline uint32_t load_key_scales(const uint8_t *p) {
    if constexpr (NB == 8) return *reinterpret_cast<const uint16_t *>(p);
    else return *p;
}
__device__ inline uint32_t key_scale_of(uint32_t g, int nb) { return nb == 8 ? 2 * g : nb == 4 ? g : g / 2; }

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

// 8 codes of a key row
__device__ inline bf16x8 widen_key(uint32_t w, float scale) {
    const bf16x2 c0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0), c1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1),
                 c2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2), c3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
    return bf16x8{c0[0], c0[1], c1[0], c1[1], c2[0], c2[1], c3[0], c3[1]};
}

// Byte b (columns 2 b and 2 b + 1) of one piece of four tokens' values v: the four tokens of each column
template <int NB>
__device__ inline void widen_values(const uint32_t *v, const float *scale, int b, uint2 &lo, uint2 &hi) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t src = v[(j * NB + b) / 4];
        bf16x2 c;
        switch ((j * NB + b) % 4) {
            case 0: c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(src, scale[j], 0); break;
            case 1: c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(src, scale[j], 1); break;
            case 2: c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(src, scale[j], 2); break;
            default: c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(src, scale[j], 3); break;
        }
        w[j] = __builtin_bit_cast(uint32_t, c);
    }
    lo.x = __builtin_amdgcn_perm(w[1], w[0], 0x05040100u); hi.x = __builtin_amdgcn_perm(w[1], w[0], 0x07060302u);
    lo.y = __builtin_amdgcn_perm(w[3], w[2], 0x05040100u); hi.y = __builtin_amdgcn_perm(w[3], w[2], 0x07060302u);
}

// Scales of 4 N tokens' value blocks.  A NaN block counts as 0, so that rows that do not see its token stay whole; the smallest index of
// such a token is returned (~0: none).  All 64 lanes call this.
template <int N, class Token>
__device__ inline uint32_t value_scales(const uint32_t *words, float *vs, Token token) {
    uint32_t nan = ~0u;
#pragma unroll
    for (int j = 0; j < 4 * N; ++j) vs[j] = pow2_of(words[j / 4], j % 4);
    float top = vs[0];
#pragma unroll
    for (int j = 1; j < 4 * N; ++j) top = fmaxf(top, vs[j]);
    if (__any(top == INFINITY)) {
#pragma unroll
        for (int j = 0; j < 4 * N; ++j)
            if (vs[j] == INFINITY) { vs[j] = 0.0f; nan = min(nan, token(j / 4, j % 4)); }
    }
    return nan;
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

    // S^T of 32 tokens: key(i, b) is the A operand of token tile i and step b
    template <class Key>
    __device__ void scores(f32x4 (*s)[2], Key key) const {
#pragma unroll
        for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 2; ++i) {  // (the two token tiles in turn: sums that do not wait for each other)
                const bf16x8 a = key(i, b);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int n = TERMS - 1; n >= 0; --n) s[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q[t][n][b], s[t][i], 0, 0, 0);
            }
    }

    // Scores to weights.  `seen(t, i, j)`: whether this lane's row of row tile t sees token 4 g + j of token tile i; asked only where
    // `mask` (uniform).
    template <class Seen>
    __device__ void weights(f32x4 (*s)[2], bf16x8 (*p)[TERMS], float scale_log2, float lift, bool mask, Seen seen) {
        if (mask) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!seen(t, j / 4, j % 4)) s[t][j / 4][j % 4] = -INFINITY;
        }
        float mx[NT];
        bool over = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            mx[t] = s[t][0][0];
#pragma unroll
            for (int j = 1; j < 8; ++j) mx[t] = fmaxf(mx[t], s[t][j / 4][j % 4]);
            mx[t] *= scale_log2;
            over |= mx[t] > m[t] + (kSlack - lift);
        }
        if (__any(over)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float to = fmaxf(m[t], max_over_row(mx[t]) + lift), by = __builtin_amdgcn_exp2f(m[t] - to);
                m[t] = to;
                l[t] = fmaf(l[t], by, to - to);  // (NaN where a score is over all of fp32: exp2 makes 0 of a finite one minus infinity)
#pragma unroll
                for (int i = 0; i < 2 * NB; ++i) o[t][i] *= by;
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = __builtin_amdgcn_exp2f(fmaf(s[t][j / 4][j % 4], scale_log2, -m[t]));
                l[t] += x[j];
            }
            split_bf16<TERMS>(x, p[t]);
        }
    }

    // O^T += V^T P^T: value(b, a) gives the A operands of columns 2 b and 2 b + 1 of the pieces
    template <class Value>
    __device__ void products(const bf16x8 (*p)[TERMS], Value value) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            bf16x8 a[2];
            value(b, a);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int n = TERMS - 1; n >= 0; --n) {
                    o[t][2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], p[t][n], o[t][2 * b], 0, 0, 0);
                    o[t][2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[1], p[t][n], o[t][2 * b + 1], 0, 0, 0);
                }
        }
    }

    // 32 tokens that this wave widens for itself; `token(i, j)`: the index that nan_at counts of token 4 g + j of token tile i
    template <class Seen, class Token>
    __device__ void step(const KvRaw<NB> &raw, float scale_log2, float lift, bool mask, Seen seen, Token token) {
        float vs[8];
        nan_at = min(nan_at, value_scales<2>(raw.vs, vs, token));
        f32x4 s[NT][2];
        scores(s, [&](int i, int b) { return widen_key(raw.k[i][b], pow2_of(raw.ks[i], NB == 8 ? b / 4 : 0)); });
        bf16x8 p[NT][TERMS];
        weights(s, p, scale_log2, lift, mask, seen);
        products(p, [&](int b, bf16x8 *a) {
            uint2 lo[2], hi[2];
            widen_values<NB>(raw.v[0], vs, b, lo[0], hi[0]);
            widen_values<NB>(raw.v[1], vs + 4, b, lo[1], hi[1]);
            a[0] = __builtin_bit_cast(bf16x8, make_uint4(lo[0].x, lo[0].y, lo[1].x, lo[1].y));
            a[1] = __builtin_bit_cast(bf16x8, make_uint4(hi[0].x, hi[0].y, hi[1].x, hi[1].y));
        });
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

// The scale bytes of the four tokens from `at` on that are there (before t1, in a page): whatever lies in the place of the others must not
// turn 0 into NaN
__device__ inline uint32_t live_scales(bool there, uint32_t at, uint32_t t1) {
    const uint32_t live = !there || at >= t1 ? 0 : min(t1 - at, 4u);
    return live == 4 ? ~0u : (1u << (8 * live)) - 1;
}

// 1 / l; 0 where nothing is seen, or no score above -inf
__device__ inline float over_sum(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }
__device__ inline float lse_of(float m, float l) { return (m + __log2f(l)) * kLn2; }

// Where the waves of a block that share 16 rows and have tokens of their own are joined: every wave leaves what it has, and after one
// barrier all threads sum it, four columns each, in the waves' order.  (Rows are padded by four words against bank conflicts.)
template <int NB, int WAVES>
struct KvJoin {
    float o[WAVES][16][32 * NB + 4], m[WAVES][16], l[WAVES][16];

    // `rows` of the 16 and the first `waves` waves count (uniform); a NaN token below `limit` (this lane's row's) spoils its columns.  All
    // threads call this.
    template <int TERMS>
    __device__ void leave(const KvRows<NB, 1, TERMS> &r, uint32_t rows, uint32_t waves, uint32_t limit) {
        const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, g = lane >> 4;
        uint32_t nan_first[4];
        nan_blocks<NB>(r.nan_at, nan_first);
        if (wave < waves && row < rows) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int e = 0; e < 2 * NB; e += 4) {
                    float4 y = make_float4(r.o[0][e][x], r.o[0][e + 1][x], r.o[0][e + 2][x], r.o[0][e + 3][x]);
                    if (nan_first[x] < limit) y.x = y.y = y.z = y.w = __uint_as_float(0x7FC00000u);
                    *reinterpret_cast<float4 *>(&o[wave][row][(4 * g + x) * 2 * NB + e]) = y;
                }
            if (g == 0) { m[wave][row] = r.m[0]; l[wave][row] = r.l[0]; }
        }
        __syncthreads();
    }

    // emit(row, d, y[4], m, l) for four columns of every row
    template <class Emit>
    __device__ void take(uint32_t rows, uint32_t waves, uint32_t dim, Emit emit) const {
        for (uint32_t item = threadIdx.x; item < rows * (8 * NB); item += 64 * WAVES) {
            const uint32_t row = item / (8 * NB), d = item % (8 * NB) * 4;
            if (d >= dim) continue;
            float top = m[0][row], sum = 0, y[4] = {};
#pragma unroll
            for (int w = 1; w < WAVES; ++w) top = w < waves ? fmaxf(top, m[w][row]) : top;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                if (w >= waves) break;
                const float by = __builtin_amdgcn_exp2f(m[w][row] - top);
                const float4 x = *reinterpret_cast<const float4 *>(&o[w][row][d]);
                sum += l[w][row] * by;
                y[0] += x.x * by; y[1] += x.y * by; y[2] += x.z * by; y[3] += x.w * by;
            }
            emit(row, d, y, top, sum);
        }
    }
};

// ---- attention over whole requests --------------------------------------------------------------------------------------

// What a block of k_kv_attend / k_kv_attend_wide works on: row tile x one key/value head x one split of the tokens of a request.  Blocks are
// numbered head first, so that (with 8 heads) an XCD's L2 keeps the pages of its own heads, and row tiles last to first, so that the
// causal ones with most tokens start first.  The requests turn by one from one tile or split to the next: blocks are dealt to the shader
// engines in order, and without it one of them gets all of a long request (4 prompts, in the kernel's first form: 465 -> 331 us).
struct KvWhere {  // what the block's number says: known before anything is read
    uint32_t head, i, split, tile;
    __device__ explicit KvWhere(const KvAttendArgs &a) {
        const uint32_t b = kv_block() / a.g.heads, turn = b / a.n;
        head = kv_block() % a.g.heads;
        i = (b + turn) % a.n;
        split = turn % a.splits;
        tile = a.tiles - 1 - turn / a.splits;  // (from tiles on, wrapped: a block behind the last one)
    }
    __device__ bool there(const KvAttendArgs &a) const { return tile < a.tiles; }
};

// The same for up to 64 requests where blocks are more than units: the blocks of tiles that no request has come last instead of first, where
// they held the units for some us before the others began.  False: there is no such tile.  (All 64 lanes call this.)
//
// Split tiles are numbered in the order of the requests, split by split (2 prompts of 1,329 x 4 rows, not causal: 29 us, 47 in turns; 313 x
// 3 rows over 4,300 tokens: 25.6, 29.2; no difference where all requests have as many).
//
// Whole tiles go by length: block b takes the b-th longest of all requests, so that the last blocks to start are the shortest.  Each lane
// counts the tiles of one request that end behind some token, and the token is searched for behind which no more than b of them end: some
// 2 us at a block's start, worth it where units get blocks one after the other (4 prompts, 1,376 blocks: 248 us, 277 in turns; 2 requests of
// 197 x 16 rows at width 256, fp32, 400 blocks: 54, 85; 16 short prompts: 17.4, 16.7).
template <uint32_t ROWS>
__device__ inline bool find_tile(const KvAttendArgs &a, KvWhere &where) {
    const uint32_t lane = threadIdx.x & 63, rank = kv_block() / a.g.heads;
    uint32_t tiles = 0, seeing = 0, reach = 0;  // row tiles, tokens whose rows these are, tokens that can be read
    int64_t base = 0;
    if (lane < a.n) {
        const uint32_t first = min(a.starts[lane], a.rows), next = min(a.starts[lane + 1], a.rows), count = next > first ? next - first : 0, length = a.lengths[lane];
        seeing = min(count, a.max_new);
        tiles = (seeing * a.group + ROWS - 1) / ROWS;
        reach = (uint32_t)min((uint64_t)min(length, a.max_length), (uint64_t)a.table_stride << a.g.page_shift);
        base = (int64_t)length - count;
    }
    if (a.splits > 1) {
        const uint32_t upto = wave_incl_scan(tiles, (int)lane), total = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
        if (rank >= (uint64_t)total * a.splits) return false;
        const uint32_t nth = rank % total, at = (uint32_t)__builtin_ctzll(__ballot(upto > nth));
        where.i = at;
        where.split = rank / total;
        where.tile = (uint32_t)__builtin_amdgcn_readlane((int)(nth - (upto - tiles)), at);
        return true;
    }
    auto wave_sum = [&](uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)wave_incl_scan(x, (int)lane), 63); };
    auto behind = [&](int32_t end) -> uint32_t {
        if (end < 0) return tiles;
        if ((uint32_t)end >= reach) return 0;
        const int64_t x = end - base;  // the row of this token sees end + 1 of them, and is the first that does
        if (!a.causal || x < 0) return tiles;
        return x >= seeing ? 0 : tiles - (uint32_t)x * a.group / ROWS;
    };
    int32_t low = -1, high = (int32_t)a.max_length;
    if (rank >= wave_sum(tiles)) return false;
    while (high - low > 1) {
        const int32_t mid = low + (high - low) / 2;
        if (wave_sum(behind(mid)) > rank) low = mid;
        else high = mid;
    }
    // of the tiles that end at `high`, in the order of the requests
    const uint32_t longer = behind(high), here = behind(low) - longer;
    const uint32_t upto = wave_incl_scan(here, (int)lane), skip = rank - wave_sum(longer), at = (uint32_t)__builtin_ctzll(__ballot(upto > skip));
    where.i = at;
    where.split = 0;
    where.tile = (uint32_t)__builtin_amdgcn_readlane((int)(tiles - 1 - longer - (skip - (upto - here))), at);
    return true;
}

struct KvBlock : KvWhere {
    uint32_t first, count, length, reach, rows, row0, end;

    __device__ KvBlock(const KvAttendArgs &a, const KvWhere &where, uint32_t block_rows) : KvWhere(where) {
        row0 = tile * block_rows;
        // rows [first, first + count) of q, `length` tokens, of which those below `reach` can be read
        first = min(a.starts[i], a.rows);
        const uint32_t next = min(a.starts[i + 1], a.rows);
        count = next > first ? next - first : 0;
        length = a.lengths[i];
        reach = (uint32_t)min((uint64_t)min(length, a.max_length), (uint64_t)a.table_stride << a.g.page_shift);
        rows = min(count, a.max_new) * a.group;
        end = row0 < rows ? limit(a, min(row0 + block_rows, rows) - 1) : 0;  // no row of the block sees more
    }
    __device__ uint32_t limit(const KvAttendArgs &a, uint32_t row) const {  // the tokens a row sees are [0, limit)
        if (!a.causal) return reach;
        const int64_t x = (int64_t)length - count + row / a.group + 1;
        return (uint32_t)min(max(x, (int64_t)0), (int64_t)reach);
    }
    __device__ const void *query(const KvAttendArgs &a, uint32_t row, uint32_t size) const {
        if (row >= rows) return nullptr;
        return static_cast<const uint8_t *>(a.q) + ((uint64_t)(first + row / a.group) * a.q_stride + (uint64_t)(head * a.group + row % a.group) * a.g.dim) * size;
    }
    // place of a row in out (times head_dim) and lse
    __device__ uint64_t place(const KvAttendArgs &a, uint32_t row) const { return (uint64_t)(first + row / a.group) * (a.g.heads * a.group) + head * a.group + row % a.group; }
};

// The pages of a wave's tiles (16 tokens), gone through in order: where 64 of them start lies in registers, one to a lane, and the next 64
// are on their way, so that no load of a page waits for its number or for a multiplication.  The wave takes STEP tokens of every STRIDE
// from `t0` on.  Entries behind the request's own are read too, and are nothing to anybody: their tokens are not seen.  (All 64 lanes
// call these.)
template <uint32_t STEP, uint32_t STRIDE>
struct KvPages {
    const uint32_t *table;
    uint64_t page_bytes;
    uint32_t t0, last, shift, pages, base, next, low, high;
    uint64_t are;

    __device__ KvPages(const KvAttendArgs &a, uint32_t request, uint32_t from)
        : table(a.tables + (uint64_t)request * a.table_stride), page_bytes(a.g.page_bytes), t0(from), last(a.table_stride - 1), shift(a.g.page_shift), pages(a.g.pages), base(0) {
        next = read(0);
    }
    __device__ uint32_t read(uint32_t tile) const {
        const uint32_t at = tile + (threadIdx.x & 63);
        return table[min((t0 + at / (STEP / 16) * STRIDE + at % (STEP / 16) * 16) >> shift, last)];
    }
    __device__ void take() {  // once before the first tile is asked for
        are = __ballot(next < pages);
        const uint64_t at = (next < pages ? next : 0) * page_bytes;
        low = (uint32_t)at;
        high = (uint32_t)(at >> 32);
        next = read(base + 64);
    }
    __device__ void reach(uint32_t tile) {  // before anything is asked about the tiles from `tile` (uniform) to the next multiple of 64
        if (tile >= base + 64) {
            base += 64;
            take();
        }
    }
    // where the tile's page starts in the cache (the first page's place if it has none)
    __device__ uint64_t start(uint32_t tile) const { return (uint64_t)(uint32_t)__builtin_amdgcn_readlane(high, tile - base) << 32 | (uint32_t)__builtin_amdgcn_readlane(low, tile - base); }
    __device__ uint32_t there(uint32_t tile) const { return (uint32_t)(are >> (tile - base)); }  // bit 0: the tile has a page; bit 1: the next; ...
};

// What a lane adds to the place of a tile in its page: the parts that a tile's tokens (16 NB or NB bytes each) move are uniform
template <int NB>
struct KvLane {
    uint32_t key, key_scale, value, value_scale;
    __device__ KvLane(uint32_t half, uint32_t page_size) {
        const uint32_t c = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
        key = c * (16 * NB) + g * (4 * NB);
        key_scale = 2 * half + c * NB + key_scale_of(g, NB);
        value = half + g * (64 * NB) + c * (4 * NB);
        value_scale = 2 * half + page_size * NB + g * (4 * NB) + v_block<NB>(c) * 4;
    }
};

// Writes a wave's rows: the result, or (several splits) the part that the join reads
template <int NB, int NT, int TERMS>
__device__ inline void store_rows(const KvAttendArgs &a, const KvBlock &blk, const KvRows<NB, NT, TERMS> &r, const uint32_t *limit, uint32_t wave_row, uint32_t seen_from) {
    constexpr uint32_t kSize = TERMS == 1 ? 2 : 4;
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4;
    uint32_t nan_first[4];
    nan_blocks<NB>(r.nan_at, nan_first);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const uint32_t row = wave_row + t * 16 + (lane & 15);
        if (row >= blk.rows) continue;
        const uint64_t at = blk.place(a, row);
        const bool some = seen_from < limit[t], whole = a.splits == 1;
        const float by = whole ? over_sum(r.l[t]) : 1.0f;
        float *part = a.part + (at * a.splits + blk.split) * (a.g.dim + 4);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            float y[2 * NB];
#pragma unroll
            for (int e = 0; e < 2 * NB; ++e) y[e] = nan_first[x] < limit[t] ? __uint_as_float(0x7FC00000u) : r.o[t][e][x] * by;
            const uint32_t d = (4 * g + x) * 2 * NB;
            if (whole) store_columns<NB, TERMS>(static_cast<uint8_t *>(a.out) + at * a.g.dim * kSize, d, a.g.dim, y);
            else store_columns<NB, 3>(part, d, a.g.dim, y);
        }
        if (g == 0) {
            if (!whole) {
                part[a.g.dim] = some ? r.m[t] : -INFINITY;  // -inf: this split saw nothing
                part[a.g.dim + 1] = r.l[t];
            } else if (a.lse) {
                a.lse[at] = some ? lse_of(r.m[t], r.l[t]) : -INFINITY;
            }
        }
    }
}

// Few rows (decode): 16 of them to a block, whose waves take the chunks of the split's tokens in turn and are joined in LDS.  Each wave
// widens what it loads, one chunk of 32 tokens ahead: 4.3 KB at width 128, three waves on a SIMD.  Bound by HBM: 48 requests to 8,192
// tokens, 8 x 128, bf16: 223 MB in 53 us with the join, as long with the loads alone and no arithmetic; with fp32 queries, whose products run
// three times, by the instructions around them (3 requests to 131,072 tokens, 4 x 64: 88 MB in 35 us, 30 with the loads alone).  One
// masked step serves whole and cut chunks: two copies of it took 232 registers for 128 and one wave less.
template <int NB, int TERMS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, NB == 8 && TERMS == 3 ? 1 : NB == 8 || TERMS == 3 || WAVES == 8 ? 2 : NB == 4 ? 3 : 4) void k_kv_attend(const KvAttendArgs a) {
    constexpr uint32_t STRIDE = 32 * WAVES;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    const KvWhere where(a);
    if (!where.there(a)) return;
    const uint32_t from = where.split * a.split_tokens, t0 = from + 32 * wave;  // the chunks of 32 go round the waves
    KvPages<32, STRIDE> pages(a, where.i, t0);                                     // (on their way together with the lengths)
    const KvBlock blk(a, where, 16);
    if (blk.row0 >= blk.rows) return;
    if (a.splits > 1 && from >= blk.end) return;  // (no row of the block sees a token of this split: joined_row knows)
    const uint32_t t1 = a.splits > 1 ? min(from + a.split_tokens, blk.end) : blk.end;

    KvRows<NB, 1, TERMS> r;
    r.clear();
    const uint32_t row = blk.row0 + (lane & 15), limit = row < blk.rows ? blk.limit(a, row) : 0;
    r.load_q(0, blk.query(a, row, TERMS == 1 ? 2 : 4), a.g.dim);
    const uint32_t all_see = __builtin_amdgcn_readfirstlane(blk.limit(a, blk.row0));  // rows behind the last one do not count: they are not stored
    uint32_t seen_from = ~0u;  // first token of the first page that is there

    if (t0 < t1) {
        const uint32_t half = a.g.page_size * 16 * NB, mask = a.g.page_size - 1;
        const uint8_t *heads = a.cache + (uint64_t)blk.head * a.g.head_bytes;
        const uint32_t chunks = (t1 - t0 + STRIDE - 1) / STRIDE;
        pages.take();
        const KvLane<NB> at(half, a.g.page_size);
        auto load = [&](KvRaw<NB> &raw, uint32_t c) -> uint32_t {
            pages.reach(2 * c);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint8_t *p = heads + pages.start(2 * c + x);
                const uint32_t in = (t0 + STRIDE * c + 16 * x) & mask;
                load_words<NB>(raw.k[x], p + (at.key + in * (16 * NB)));
                raw.ks[x] = load_key_scales<NB>(p + (at.key_scale + in * NB));
                load_words<NB>(raw.v[x], p + (at.value + in * (16 * NB)));
                raw.vs[x] = *reinterpret_cast<const uint32_t *>(p + (at.value_scale + in * NB));
            }
            return pages.there(2 * c) & 3;
        };
        auto work = [&](KvRaw<NB> &raw, uint32_t t, uint32_t there) {
            const bool part = there != 3 || t + 32 > t1;  // some token is none
            if (there) seen_from = min(seen_from, t + (there & 1 ? 0 : 16));
            if (part) {
#pragma unroll
                for (int x = 0; x < 2; ++x) raw.vs[x] &= live_scales(there >> x & 1, t + 16 * x + 4 * g, t1);
            }
            r.step(raw, a.scale_log2, a.lift, part || t + 32 > all_see,
                   [&](int, int x, int j) { const uint32_t at = t + 16 * x + 4 * g + j; return (there >> x & 1) && at < limit && at < t1; },
                   [&](int x, int j) { return t + 16 * x + 4 * g + j; });
        };
        KvRaw<NB> cur, nxt;
        uint32_t there = load(cur, 0);
        for (uint32_t c = 0; c < chunks; ++c) {
            const uint32_t there_next = load(nxt, min(c + 1, chunks - 1));
            work(cur, t0 + c * STRIDE, there);
            cur = nxt;
            there = there_next;
        }
    }
    r.close();
    __shared__ KvJoin<NB, WAVES> join;
    __shared__ uint32_t seen[WAVES];
    if (lane == 0) seen[wave] = seen_from;
    const uint32_t rows = min(blk.rows - blk.row0, 16u);
    const uint32_t waves = t1 > from ? min((t1 - from + 31) / 32, (uint32_t)WAVES) : 1;  // that have tokens
    join.leave(r, rows, waves, limit);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) seen_from = min(seen_from, seen[w]);
    const bool whole = a.splits == 1;
    join.take(rows, waves, a.g.dim, [&](uint32_t row, uint32_t d, float *y, float m, float l) {
        const uint64_t at = blk.place(a, blk.row0 + row);
        const bool some = seen_from < blk.limit(a, blk.row0 + row);
        if (whole) {
            const float by = over_sum(l);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] *= by;
            store_columns<2, TERMS>(static_cast<uint8_t *>(a.out) + at * a.g.dim * (TERMS == 1 ? 2 : 4), d, a.g.dim, y);
            if (d == 0 && a.lse) a.lse[at] = some ? lse_of(m, l) : -INFINITY;
        } else {
            float *to = a.part + (at * a.splits + blk.split) * (a.g.dim + 4);
            store_columns<2, 3>(to, d, a.g.dim, y);
            if (d == 0) {
                to[a.g.dim] = some ? m : -INFINITY;  // -inf: this split saw nothing
                to[a.g.dim + 1] = l;
            }
        }
    });
}

// Row tiles of a wave of k_kv_attend_wide, at most: what 256 registers hold, and at width 64 two, which leave room for more waves on a SIMD
// (8 prompts of up to 1,000 tokens, 32 heads x 64: 32 us, 36 with three; fp32, 3 of up to 1,469: 91, 83 with three, but 4 of 2,048: 151, 185)
constexpr int wide_tiles(int nb, int terms) { return nb == 8 ? 1 : nb == 4 && terms == 1 ? 3 : 2; }

// Many rows (prompts): each of a block's four waves has NT tiles of its own and all walk the same tokens.  A wave's tile of 16 tokens (at
// width 256 its keys or its values) is widened once for the block into LDS, in the order in which the matrix instructions take it: 64
// tokens (32) at a time into one of two buffers while the other is read, one barrier for each.  A wave's next raw rows are requested as
// soon as it has widened the last, a whole chunk ahead.
//
// Bound by instruction issue: 32 tokens x 48 rows are 48 matrix instructions (768 cycles of the unit) and some 180 others (1,020), of
// which the weights are two thirds; a SIMD's two waves overlap them by half at best, and what is lost to waits is as much.  4 prompts of
// 1,500 to 2,048 tokens, 32 heads, causal: 245 us, 1.02 PFLOP/s, where a library product of 8192^3 reaches 1.21.  Taken and measured
// (before the longest blocks came first, 275 us): every wave widening for itself 331 us; 32 or 64 rows a wave 297 / 666 (registers); three
// waves of 32 rows on a SIMD 291; eight waves sharing a widened tile 300; raised priority around the matrix instructions 308.  At width
// 256 a wave has 16 rows and the start and end of a block weigh as much as its 20 chunks (33 rows of 8 heads over 4,100 tokens: 49 us; two
// tiles a wave at one wave a SIMD 78; keys widened by every wave 86).
template <int NB, int NT, int TERMS>
__global__ __launch_bounds__(256, NB == 8 && TERMS == 3 ? 1 : 2) void k_kv_attend_wide(const KvAttendArgs a) {
    constexpr uint32_t TILES = NB == 8 ? 2 : 4, T = 16 * TILES;
    constexpr bool BOTH = NB < 8;  // a wave widens keys and values of its tile
    __shared__ uint4 keys[2][TILES][NB][64], vals[2][TILES / 2][2 * NB][64];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    KvWhere where(a);
    if (a.by_tile ? !find_tile<64 * NT>(a, where) : !where.there(a)) return;
    const uint32_t t0 = where.split * a.split_tokens;
    KvPages<T, T> pages(a, where.i, t0);
    const KvBlock blk(a, where, 64 * NT);
    if (blk.row0 >= blk.rows) return;
    if (a.splits > 1 && t0 >= blk.end) return;
    const uint32_t t1 = a.splits > 1 ? min(t0 + a.split_tokens, blk.end) : blk.end;
    const uint32_t wave_row = blk.row0 + wave * (16 * NT);

    KvRows<NB, NT, TERMS> r;
    r.clear();
    uint32_t limit[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const uint32_t row = wave_row + t * 16 + (lane & 15);
        limit[t] = row < blk.rows ? blk.limit(a, row) : 0;
        r.load_q(t, blk.query(a, row, TERMS == 1 ? 2 : 4), a.g.dim);
    }
    const bool rows_here = wave_row < blk.rows;
    const uint32_t all_see = rows_here ? __builtin_amdgcn_readfirstlane(blk.limit(a, wave_row)) : 0;
    const uint32_t wave_end = rows_here ? min(t1, __builtin_amdgcn_readfirstlane(blk.limit(a, min(wave_row + 16 * NT, blk.rows) - 1))) : 0;
    uint32_t seen_from = ~0u;

    if (t0 < t1) {
        const uint32_t half = a.g.page_size * 16 * NB, mask = a.g.page_size - 1;
        const uint8_t *heads = a.cache + (uint64_t)blk.head * a.g.head_bytes;
        pages.take();
        const uint32_t chunks = (t1 - t0 + T - 1) / T, tile = BOTH ? wave : wave & 1;
        const bool does_keys = BOTH || wave < 2, does_vals = BOTH || wave >= 2;
        const KvLane<NB> place(half, a.g.page_size);
        uint32_t k[NB], v[BOTH ? NB : 1], ks = 0, vs = 0;  // raw rows of the chunk after the one that is read (v shares k at width 256)
        uint32_t *const vv = BOTH ? v : k;
        // bit x: page of the chunk's tile x is there
        auto fetch = [&](uint32_t c) -> uint32_t {
            c = min(c, chunks - 1);
            pages.reach(c * TILES);
            const uint32_t in = (t0 + c * T + 16 * tile) & mask;
            const uint8_t *p = heads + pages.start(c * TILES + tile);
            if (does_keys) {
                load_words<NB>(k, p + (place.key + in * (16 * NB)));
                ks = load_key_scales<NB>(p + (place.key_scale + in * NB));
            }
            if (does_vals) {
                load_words<NB>(vv, p + (place.value + in * (16 * NB)));
                vs = *reinterpret_cast<const uint32_t *>(p + (place.value_scale + in * NB));
            }
            return pages.there(c * TILES) & ((1u << TILES) - 1);
        };
        auto widen = [&](uint32_t c, uint32_t there) {
            const uint32_t buf = c & 1, at = t0 + c * T + 16 * tile + 4 * g;
            if (does_keys) {
#pragma unroll
                for (int b = 0; b < NB; ++b) keys[buf][tile][b][lane] = __builtin_bit_cast(uint4, widen_key(k[b], pow2_of(ks, NB == 8 ? b / 4 : 0)));
            }
            if (does_vals) {
                uint32_t word = vs & live_scales(there >> tile & 1, at, t1);
                float scale[4];
                r.nan_at = min(r.nan_at, value_scales<1>(&word, scale, [&](int, int j) { return at + j; }));
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    uint2 lo, hi;
                    widen_values<NB>(vv, scale, b, lo, hi);
                    reinterpret_cast<uint2 *>(&vals[buf][tile / 2][2 * b][lane])[tile & 1] = lo;
                    reinterpret_cast<uint2 *>(&vals[buf][tile / 2][2 * b + 1][lane])[tile & 1] = hi;
                }
            }
        };
        uint32_t there = fetch(0);
        widen(0, there);
        uint32_t there_next = fetch(1);
        for (uint32_t c = 0; c < chunks; ++c) {
            __syncthreads();  // chunk c is whole; the buffer of chunk c + 1 has been read
            const uint32_t t = t0 + c * T, buf = c & 1;
            if (there) seen_from = min(seen_from, t + 16 * (uint32_t)__builtin_ctz(there));
#pragma unroll
            for (uint32_t h = 0; h < TILES / 2; ++h) {
                const uint32_t th = t + 32 * h;
                if (th >= wave_end) break;
                const bool here[2] = {(there >> (2 * h) & 1) != 0, (there >> (2 * h + 1) & 1) != 0};
                f32x4 s[NT][2];
                r.scores(s, [&](int x, int b) { return __builtin_bit_cast(bf16x8, keys[buf][2 * h + x][b][lane]); });
                bf16x8 p[NT][TERMS];
                r.weights(s, p, a.scale_log2, a.lift, !(here[0] && here[1]) || th + 32 > all_see || th + 32 > t1,
                          [&](int row_tile, int x, int j) { const uint32_t at = th + 16 * x + 4 * g + j; return here[x] && at < limit[row_tile] && at < t1; });
                r.products(p, [&](int b, bf16x8 *v2) {
                    v2[0] = __builtin_bit_cast(bf16x8, vals[buf][h][2 * b][lane]);
                    v2[1] = __builtin_bit_cast(bf16x8, vals[buf][h][2 * b + 1][lane]);
                });
            }
            there = there_next;
            if (c + 1 < chunks) {
                widen(c + 1, there);
                there_next = fetch(c + 2);
            }
        }
    }
    r.close();
    // each wave knows the NaN blocks that it widened: the smallest index over the four
    __syncthreads();
    uint32_t *const nan = reinterpret_cast<uint32_t *>(&keys[0][0][0][0]);
    nan[wave * 64 + lane] = r.nan_at;
    __syncthreads();
    if (!rows_here) return;
    r.nan_at = min(min(nan[lane], nan[64 + lane]), min(nan[128 + lane], nan[192 + lane]));
    store_rows(a, blk, r, limit, wave_row, seen_from);
}

// The at-th (row, head) of a join: where it is in q and out, and how many splits any of its tokens lie in.  False where a request has no
// such row.
__device__ inline bool joined_row(const KvAttendArgs &a, uint32_t at, uint64_t &row, uint32_t &live) {
    const uint32_t qheads = a.g.heads * a.group, head = at % qheads, i = at / qheads % a.n, j = at / qheads / a.n;
    const uint32_t first = min(a.starts[i], a.rows), next = min(a.starts[i + 1], a.rows), count = next > first ? next - first : 0;
    if (j >= count) return false;
    const uint32_t length = a.lengths[i];
    const uint32_t reach = (uint32_t)min((uint64_t)min(length, a.max_length), (uint64_t)a.table_stride << a.g.page_shift);
    uint32_t limit = reach;
    if (a.causal) limit = (uint32_t)min(max((int64_t)length - count + (int64_t)j + 1, (int64_t)0), (int64_t)reach);
    row = (uint64_t)(first + j) * qheads + head;
    live = min((limit + a.split_tokens - 1) / a.split_tokens, a.splits);
    return true;
}

// Joins up to kFewSplits splits of a row: four columns to a thread, which reads every split's maximum and sum for itself.  All that it
// reads is asked for at once and nothing is waited for twice, where k_kv_join has three barriers for a row (4,864 rows of 256 in seven
// splits: 8.4 us, 2.4 less than with k_kv_join; 1,536 of 128 in three: 4.9, 0.8 less).
constexpr uint32_t kFewSplits = 8;

template <int W, int TERMS>
__global__ __launch_bounds__(256) void k_kv_join_few(const KvAttendArgs a, uint32_t count) {
    constexpr uint32_t COLS = W / 4;
    const uint32_t at = blockIdx.x * (256 / COLS) + threadIdx.x / COLS, d = threadIdx.x % COLS * 4, step = a.g.dim + 4;
    if (at >= count || d >= a.g.dim) return;
    uint64_t row;
    uint32_t live;
    if (!joined_row(a, at, row, live)) return;
    const float *part = a.part + row * a.splits * step;
    float4 x[kFewSplits];
    float2 ml[kFewSplits];
#pragma unroll
    for (uint32_t u = 0; u < kFewSplits; ++u) {
        if (u >= a.splits) break;
        if (u < live) {
            x[u] = *reinterpret_cast<const float4 *>(part + u * step + d);
            ml[u] = *reinterpret_cast<const float2 *>(part + u * step + a.g.dim);
        } else {
            x[u] = make_float4(0, 0, 0, 0);
            ml[u] = make_float2(-INFINITY, 0.0f);
        }
    }
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (uint32_t u = 0; u < kFewSplits; ++u) {
        if (u >= a.splits) break;
        m = fmaxf(m, ml[u].x);
    }
    float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
    for (uint32_t u = 0; u < kFewSplits; ++u) {
        if (u >= a.splits) break;
        if (ml[u].x == -INFINITY) continue;  // (the split saw nothing and left nothing)
        const float by = __builtin_amdgcn_exp2f(ml[u].x - m);  // 0 spares nothing: a NaN that the split holds stays one
        l += ml[u].y * by;
        o.x += x[u].x * by; o.y += x[u].y * by; o.z += x[u].z * by; o.w += x[u].w * by;
    }
    const bool some = m != -INFINITY;
    const float by = over_sum(l);
    const float y[4] = {o.x * by, o.y * by, o.z * by, o.w * by};
    constexpr uint32_t kSize = TERMS == 1 ? 2 : 4;
    store_columns<2, TERMS>(static_cast<uint8_t *>(a.out) + row * a.g.dim * kSize, d, a.g.dim, y);
    if (d == 0 && a.lse) a.lse[row] = some ? lse_of(m, l) : -INFINITY;
}

// Joins more splits (at most 256) of a row, one block for a (row, head): a thread for each split's maximum and sum, then four columns and
// every (1024 / W)-th split to a thread.  The order of the sums depends on the sizes alone.  Latency of three dependent reads: the first
// parts are on their way before the weights are known.
template <int W, int TERMS>
__global__ __launch_bounds__(256) void k_kv_join(const KvAttendArgs a) {
    constexpr uint32_t COLS = W / 4, LANES = 256 / COLS, AHEAD = 2;
    __shared__ float weight[256], red[2][4];
    __shared__ float4 sum[LANES][COLS];
    const uint32_t tid = threadIdx.x, step = a.g.dim + 4;
    uint64_t row;
    uint32_t live;
    if (!joined_row(a, blockIdx.x, row, live)) return;
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
    const float w = ms == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms - m);  // (-inf: the split saw nothing and left zeros)
    weight[tid] = w;
    float l = ms == -INFINITY ? 0.0f : ls * w;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) l += __shfl_xor(l, x);
    if ((tid & 63) == 0) red[1][tid >> 6] = l;
    __syncthreads();
    float4 o = make_float4(0, 0, 0, 0);
    auto add = [&](const float4 &x, uint32_t s) {
        const float by = weight[s];  // 0 spares nothing: a NaN that the split holds stays one
        o.x += x.x * by; o.y += x.y * by; o.z += x.z * by; o.w += x.w * by;
    };
    if (mine) {
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; ++u)
            if (lane + u * LANES < live) add(ahead[u], lane + u * LANES);
#pragma unroll 8
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
    const float by = over_sum(l);
    const float y[4] = {o.x * by, o.y * by, o.z * by, o.w * by};
    constexpr uint32_t kSize = TERMS == 1 ? 2 : 4;
    if (mine) store_columns<2, TERMS>(static_cast<uint8_t *>(a.out) + row * a.g.dim * kSize, d, a.g.dim, y);
    if (tid == 0 && a.lse) a.lse[row] = some ? lse_of(m, l) : -INFINITY;
}

// ---- attention over selected rows ---------------------------------------------------------------------------------------

// A block takes one request and key/value head: its list of ids is resolved to places in the cache in LDS (a search's ids and counts
// as zvdb_hip_search_*_dev writes them), then its four waves take 32 entries at a time.  A list of 100 is three dependent reads (ids,
// pages, rows) and one chunk to a wave, so what counts is how many blocks a unit holds; a token's V lies in 16 pieces of four tokens
// each, of which the other three are read for nothing.  256 requests x 8 heads x 100 rows of 65,536, 4 x 128: 16.5 us; the 128-byte lines
// that it touches are 131 MB (640 bytes for a row's 136), 7.9 TB/s of them out of the caches.
constexpr uint32_t kSelPass = 1024;  // entries resolved at a time

template <int NB, int TERMS>
__global__ __launch_bounds__(256, NB == 8 && TERMS == 3 ? 1 : NB == 8 || TERMS == 3 ? 2 : 4) void k_kv_attend_selected(const KvAttendArgs a) {
    constexpr uint64_t kNo = ~0ull;
    __shared__ union {
        uint64_t places[kSelPass];  // bytes from the cache's start to the page | token in the page << 48; kNo: not there
        KvJoin<NB, 4> join;
    } lds;
    uint64_t *const places = lds.places;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    const uint32_t head = kv_block() % a.g.heads, b = kv_block() / a.g.heads, i = b % a.n, tile = b / a.n;
    if (tile * 16 >= a.group) return;
    const uint64_t list = (uint64_t)head * a.n + i;
    const uint64_t *ids = a.ids + list * a.k;
    constexpr uint32_t AHEAD = kSelPass / 256;
    uint64_t id[AHEAD];  // the first pass's, asked for before the count is known
#pragma unroll
    for (uint32_t x = 0; x < AHEAD; ++x) id[x] = threadIdx.x + 256 * x < a.k ? ids[threadIdx.x + 256 * x] : kNo;
    const uint32_t entries = min(a.counts ? a.counts[list] : a.k, a.k), length = a.lengths[i];
    const uint32_t reach = (uint32_t)min((uint64_t)length, (uint64_t)a.table_stride << a.g.page_shift);
    const uint32_t qheads = a.g.heads * a.group, row = tile * 16 + (lane & 15);
    constexpr uint32_t kSize = TERMS == 1 ? 2 : 4;
    KvRows<NB, 1, TERMS> r;
    r.clear();
    const uint32_t half = a.g.page_size * 16 * NB, mask = a.g.page_size - 1;
    const uint8_t *cache = a.cache + (uint64_t)head * a.g.head_bytes;
    bool any = false;
    for (uint32_t e0 = 0; e0 < entries; e0 += kSelPass) {
        const uint32_t m = min(entries - e0, kSelPass);
        if (e0) {
            __syncthreads();
#pragma unroll
            for (uint32_t x = 0; x < AHEAD; ++x) id[x] = e0 + threadIdx.x + 256 * x < a.k ? ids[e0 + threadIdx.x + 256 * x] : kNo;
        }
#pragma unroll
        for (uint32_t x = 0; x < AHEAD; ++x) {
            const uint32_t e = threadIdx.x + 256 * x;
            uint64_t at = kNo;
            if (e < m && id[x] < reach) {
                const uint32_t page = a.tables[(uint64_t)i * a.table_stride + (uint32_t)(id[x] >> a.g.page_shift)];
                if (page < a.g.pages) at = page * a.g.page_bytes | (id[x] & mask) << 48;
            }
            places[e] = at;
        }
        if (e0 == 0) r.load_q(0, row < a.group ? static_cast<const uint8_t *>(a.q) + ((uint64_t)i * a.q_stride + (uint64_t)(head * a.group + row) * a.g.dim) * kSize : nullptr, a.g.dim);
        __syncthreads();
        for (uint32_t e = wave * 32; e < m; e += 128) {
            KvRaw<NB> raw;
            uint32_t seen = 0;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint64_t key = places[e + 16 * x + (lane & 15)] == kNo ? 0 : places[e + 16 * x + (lane & 15)];
                const uint8_t *p = cache + (key & 0xFFFFFFFFFFFFull);
                const uint32_t kt = (uint32_t)(key >> 48);
                load_words<NB>(raw.k[x], p + kt * (16 * NB) + g * (4 * NB));
                raw.ks[x] = load_key_scales<NB>(p + 2 * half + kt * NB + key_scale_of(g, NB));
                raw.vs[x] = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint64_t there = places[e + 16 * x + 4 * g + j], val = there == kNo ? 0 : there;
                    const uint32_t vt = (uint32_t)(val >> 48);
                    const uint8_t *w = cache + (val & 0xFFFFFFFFFFFFull);
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
                    raw.vs[x] |= (there == kNo ? 0u : s) << (8 * j);
                    seen |= there == kNo ? 0u : 1u << (4 * x + j);
                }
            }
            any |= seen != 0;
            r.step(raw, a.scale_log2, a.lift, true, [&](int, int x, int j) { return seen >> (4 * x + j) & 1; }, [](int, int) { return 0u; });
        }
    }
    r.close();
    const bool some = __syncthreads_or(any);  // (and the places have been read)
    const uint32_t rows = min(a.group - tile * 16, 16u), waves = min((entries + 31) / 32, 4u);
    lds.join.leave(r, rows, waves ? waves : 1, 1);
    lds.join.take(rows, waves ? waves : 1, a.g.dim, [&](uint32_t at, uint32_t d, float *y, float m, float l) {
        const uint64_t out_row = (uint64_t)i * qheads + head * a.group + tile * 16 + at;
        const float by = over_sum(l);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] *= by;
        store_columns<2, TERMS>(static_cast<uint8_t *>(a.out) + out_row * a.g.dim * kSize, d, a.g.dim, y);
        if (d == 0 && a.lse) a.lse[out_row] = some ? lse_of(m, l) : -INFINITY;
    });
}

// ---- launches -----------------------------------------------------------------------------------------------------------

// How a call is cut (all forms measured: profiles/kv/cuts.txt).  Rows of one (request, head) that fit 64 are few: blocks of 16 whose waves
// divide the tokens; more of them give each wave its own tiles, as many as leave three blocks with rows for two units of the card (one prompt
// of 4,000 over 4,000, 16 heads: 218 us with two tiles, 266 with one, 260 with three; 8 prompts of up to 300 x 4 rows: 34 with one, 51 with
// three; 82 new tokens of 7 heads over 2,452: 14 with one, 20 with three).  The total of the rows says how many blocks that is, where prompts are
// of many lengths.
//
// Tokens are split where blocks are fewer than the card wants.  Each part costs its start (some 5 us of dependent reads), its rows in the
// workspace and its place in the join.  Few rows: none up to 1,024 tokens (one request: 9.7 us, 12.6 in two), parts of at least 512 up to
// 32 parts (16 requests to 4,000, 32 heads x 64, fp32: 15.6 us, 17.4 with 1,024; x 128: 23.9, 22.1), of 1,024 beyond (one head over 131,072: 16.1
// us, 19.0 with 2,048, 16.6 with 512), up to four blocks for each unit unless there are two (requests differ in length, a good third of the
// splits is empty: 48 requests to 8,192 tokens: 2 / 3 / 5 splits 58.0 / 53.8 / 57.4 us; 64 of 2,048: whole 30, two splits 38); at width 256,
// where a unit holds one block or two, up to one (24 requests to 11,000, fp32: 36 us, 46 with four; 64 to 2,000: 33 whole, 49).  Many: none
// from one block a unit on (7 prompts of 1,294 tokens, 294 blocks: 33 us, with four splits 50), else to two, four at width 256 with bf16 queries,
// whose blocks are the slowest (33 rows of 8 heads over 4,100 tokens: 50 us, 65 with two, 64 with six; fp32, one block resident on a unit: 4
// prompts of 422 x 5 rows over 1,415: 37 us, 46 with four).  Few rows that leave units empty even so get eight waves to a block (one request of
// 1,024 tokens: 9.7 us, 10.1 with four waves, 12.6 with four waves and splits).
struct KvCut {
    bool wide, by_tile;
    uint32_t nt, tiles, splits, split_tokens, waves;
    uint64_t blocks;
};

static KvCut kv_cut(const KvGeom &g, uint32_t type, uint32_t group, uint32_t n, uint32_t all_rows, uint32_t max_new, uint32_t max_length, int cus) {
    KvCut c;
    const uint64_t rows = (uint64_t)max_new * group;
    const uint32_t w = kv_width(g.dim);
    c.wide = rows > 64;
    c.nt = c.wide ? wide_tiles(w / 32, type == ZVDB_KV_F32 ? 3 : 1) : 1;
    auto cut_rows = [&]() {
        const uint32_t block_rows = c.wide ? 64 * c.nt : 16;
        c.tiles = (uint32_t)((rows + block_rows - 1) / block_rows);
        return (uint64_t)g.heads * n * c.tiles;
    };
    uint64_t base = cut_rows();
    // blocks that have rows, at most: the host knows how many rows there are in all
    auto busy = [&]() { return std::min(base, (uint64_t)g.heads * ((uint64_t)all_rows * group / (64 * c.nt) + n)); };
    while (c.nt > 1 && busy() < 3 * (uint64_t)cus / 2) {
        --c.nt;
        base = cut_rows();
    }
    const uint64_t want = (uint64_t)cus * (c.wide ? (w < 256 || type == ZVDB_KV_F32 ? 2 : 4) : w < 256 ? 4 : 1);
    uint64_t splits = base && base < (c.wide || w == 256 ? 1 : 2) * (uint64_t)cus ? (want + base - 1) / base : 1;
    auto parts_of = [&](uint64_t tokens) { return (max_length + tokens - 1) / tokens; };
    splits = std::min<uint64_t>(splits, c.wide ? parts_of(256) : max_length <= 1024 ? 1 : std::max<uint64_t>(std::min<uint64_t>(parts_of(512), 32), parts_of(1024)));
    splits = std::max<uint64_t>(std::min<uint64_t>(splits, 256), 1);
    c.split_tokens = (uint32_t)std::max<uint64_t>((((uint64_t)max_length + splits - 1) / splits + 127) / 128 * 128, 128);
    c.splits = (uint32_t)std::max<uint64_t>(((uint64_t)max_length + c.split_tokens - 1) / c.split_tokens, 1);
    c.blocks = base * c.splits;
    c.by_tile = c.wide && n > 1 && n <= 64 && c.blocks > (uint64_t)cus;
    c.waves = !c.wide && c.blocks <= (uint64_t)cus && w <= 128 && c.split_tokens > 256 ? 8 : 4;
    return c;
}

template <int NB, int TERMS>
static void launch_attend_as(const KvAttendArgs &a, const KvCut &c, hipStream_t s) {
    const dim3 grid = kv_grid(c.blocks), block(64 * c.waves);
    if (c.wide && c.nt == 3) hipLaunchKernelGGL((k_kv_attend_wide<NB, wide_tiles(NB, TERMS), TERMS>), grid, block, 0, s, a);
    else if (c.wide && c.nt == 2) hipLaunchKernelGGL((k_kv_attend_wide<NB, NB == 8 ? 1 : 2, TERMS>), grid, block, 0, s, a);
    else if (c.wide) hipLaunchKernelGGL((k_kv_attend_wide<NB, 1, TERMS>), grid, block, 0, s, a);
    else if (c.waves == 8) hipLaunchKernelGGL((k_kv_attend<NB < 8 ? NB : 4, TERMS, 8>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_kv_attend<NB, TERMS, 4>), grid, block, 0, s, a);
}

template <int NB>
static void launch_attend(const KvAttendArgs &a, const KvCut &c, uint32_t type, hipStream_t s) {
    if (type == ZVDB_KV_F32) launch_attend_as<NB, 3>(a, c, s);
    else launch_attend_as<NB, 1>(a, c, s);
}

template <int W>
static void launch_join(const KvAttendArgs &a, uint32_t blocks, uint32_t type, hipStream_t s) {
    if (a.splits <= kFewSplits) {
        const dim3 few((uint32_t)(((uint64_t)blocks * W + 1023) / 1024));
        if (type == ZVDB_KV_F32) hipLaunchKernelGGL((k_kv_join_few<W, 3>), few, dim3(256), 0, s, a, blocks);
        else hipLaunchKernelGGL((k_kv_join_few<W, 1>), few, dim3(256), 0, s, a, blocks);
    } else if (type == ZVDB_KV_F32) hipLaunchKernelGGL((k_kv_join<W, 3>), dim3(blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_kv_join<W, 1>), dim3(blocks), dim3(256), 0, s, a);
}

template <int NB>
static void launch_selected(const KvAttendArgs &a, uint32_t blocks, uint32_t type, hipStream_t s) {
    if (type == ZVDB_KV_F32) hipLaunchKernelGGL((k_kv_attend_selected<NB, 3>), kv_grid(blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_kv_attend_selected<NB, 1>), kv_grid(blocks), dim3(256), 0, s, a);
}

static int check_queries(const KvGeom &g, const void *q, uint64_t q_stride, uint32_t type, uint32_t q_heads, float scale, const void *out, const void *cache) {
    KV_ARG(q && out && cache, "null argument");
    KV_ARG(kv_aligned(q, 16) && kv_aligned(out, 16) && kv_aligned(cache, 16), "kv_attend: cache, q and out need 16-byte alignment");
    KV_ARG(kv_stride_ok(q_stride, (uint64_t)q_heads * g.dim), "kv_attend: a token's stride is at least q_heads * head_dim, below 2^40 and a multiple of 8");
    KV_ARG(scale > 0.0f && scale <= 1e38f, "kv_attend: scale %g (positive, at most 1e38)", (double)scale);
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
    KV_ARG((uint64_t)std::min(max_new, rows) * (q_heads / g.heads) < 0x7FFFFFFFu, "kv_attend: %u rows of %u heads each are too many for one request", std::min(max_new, rows),
           q_heads / g.heads);
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
    const KvCut c = kv_cut(g, type, q_heads / g.heads, n, rows, std::min(max_new, rows), max_length, cus);
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
    const KvCut c = kv_cut(a.g, type, q_heads / a.g.heads, n, rows, max_new, max_length, dev.cus());
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
    a.lift = kv_lift(max_length);
    a.n = n; a.rows = rows; a.max_new = max_new; a.max_length = max_length;
    a.split_tokens = c.split_tokens; a.splits = c.splits; a.tiles = c.tiles;
    a.causal = causal != 0; a.by_tile = c.by_tile;
    const uint32_t w = kv_width(a.g.dim);
    if (w == 64) launch_attend<2>(a, c, type, s);
    else if (w == 128) launch_attend<4>(a, c, type, s);
    else launch_attend<8>(a, c, type, s);
    ZV_HIP(hipGetLastError());
    if (c.splits > 1) {
        const uint32_t blocks = q_heads * n * max_new;  // (a call in splits has fewer than two tiles of rows for each unit)
        if (w == 64) launch_join<64>(a, blocks, type, s);
        else if (w == 128) launch_join<128>(a, blocks, type, s);
        else launch_join<256>(a, blocks, type, s);
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
    a.lift = kv_lift(k);
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
