// kv_cache.h -- the 4-bit key/value cache: its layout (include/zvdb_hip.h: "4-bit key/value cache") as the kernels use it, and what
// every zvdb_hip_kv_* entry point checks before it launches.
#pragma once

#include "common.h"

namespace zvdb {

// A stored row is kv_width(head_dim) elements wide (zero behind head_dim): three widths, so that the kernels know how many bytes a
// lane loads.  One head's part of a page, P tokens, D = 32 NB elements:
//   K codes [P][D/2] | V codes [P/4][16][4][NB] | K scales [P][NB] | V scales [P/4][NB][4]      = P (D + 2 NB) bytes
inline uint32_t kv_width(uint32_t head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }
inline uint64_t kv_head_bytes(const zvdb_hip_kv_layout *l) { return (uint64_t)l->page_size * (kv_width(l->head_dim) + kv_width(l->head_dim) / 16); }

// the layout as kernels take it
struct KvGeom {
    uint64_t page_bytes;  // all heads of one page
    uint32_t head_bytes, pages, heads, dim;
    uint32_t page_size, page_shift;
};

// Smallest and largest scale exponent a block gets: 2^-125 x 0.5 is the smallest normal bf16, 2^125 x 6 is finite in bf16, so a
// dequantised value is always a normal number that the matrix instructions take as it is.  255 marks a block that held a NaN or
// an infinity: all of it reads back as NaN.
constexpr uint32_t kKvScaleMin = 2, kKvScaleMax = 252, kKvScaleNaN = 255;

int kv_check_layout(const zvdb_hip_kv_layout *l, KvGeom *g);

// Puts the calling thread on the device that owns `p` (and must own the stream) for the length of a call.
class KvDevice {
  public:
    KvDevice() = default;
    ~KvDevice() { if (prev_ >= 0) (void)hipSetDevice(prev_); }
    KvDevice(const KvDevice &) = delete;
    KvDevice &operator=(const KvDevice &) = delete;
    int enter(const void *p, hipStream_t s);
    int cus() const { return cus_; }

  private:
    int prev_ = -1, cus_ = 0;
};

#define KV_ARG(cond, ...)                 \
    do {                                  \
        if (!(cond)) {                    \
            zvdb::set_error(__VA_ARGS__); \
            return ZVDB_ERR_INVALID;      \
        }                                 \
    } while (0)

// Elements from one token's row to the next.  Far above any memory, far below where a row's offset wraps (a negative stride is refused)
constexpr uint64_t kKvStrideEnd = 1ull << 40;
inline bool kv_stride_ok(uint64_t stride, uint64_t row) { return stride >= row && stride < kKvStrideEnd && stride % 8 == 0; }

// A launch has fewer than 2^32 threads in a direction: blocks from 2^kGridShift on go on in y, and kv_block() counts them all.  The last
// row of y is launched whole, so that a kernel meets blocks behind its last one.
constexpr uint32_t kGridShift = 22;
inline dim3 kv_grid(uint64_t blocks, uint32_t z = 1) {
    return blocks <= 1u << kGridShift ? dim3((uint32_t)blocks, 1, z) : dim3(1u << kGridShift, (uint32_t)((blocks - 1) >> kGridShift) + 1, z);
}

inline bool kv_aligned(const void *p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

#if defined(__HIPCC__)
__device__ inline uint32_t kv_block() { return blockIdx.y << kGridShift | blockIdx.x; }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Offset of element `piece` of token t's V codes within a head's V region: 16 pieces of 2 NB elements, four tokens side by side
template <int NB>
__device__ inline uint32_t kv_v_offset(uint32_t t, uint32_t piece) {
    return (t >> 2) * (64 * NB) + piece * (4 * NB) + (t & 3) * NB;
}
#endif

}  // namespace zvdb
