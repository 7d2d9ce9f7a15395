// Internal interface between the entry points of the microscaled 4-bit calls
// (mx4_capi.hip) and their kernels (mx4.hip, mx4_cache.hip, mx4_matmul.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fufft {
namespace mx4 {

// element types, as the public FUFFT_F32, FUFFT_BF16, FUFFT_F16
enum { T_F32 = 0, T_BF16 = 1, T_F16 = 2 };
inline int64_t type_bytes(int type) { return type == T_F32 ? 4 : 2; }
inline int64_t padded(int64_t k) { return (k + 127) / 128 * 128; }

// Lanes that one launch may have in x: the runtime counts them in 32 bits, and starts a grid
// of more without an error but with the count's low bits.
constexpr int64_t kMostLanes = 0xffffffff;
inline bool grid_ok(int64_t blocks, int64_t lanes) { return blocks <= kMostLanes / lanes; }

// what the launches below return for sizes that they cannot hold, before anything is launched
constexpr hipError_t kTooLarge = hipErrorNotSupported;

struct QuantizeParams {
   const void*    x;         // rows x k, leading dimension ld (elements)
   const uint8_t* rand;      // a byte per value, rows x k, or NULL: nearest
   uint8_t*       codes;     // rows x kp / 2 (NULL: not wanted)
   uint8_t*       scales;    // rows x kp / 32
   uint8_t*       codes_t;   // k x rowsp / 2 (NULL: not wanted)
   uint8_t*       scales_t;  // k x rowsp / 32
   const int64_t* slots;     // row r goes to row slots[r] of codes and scales (NULL: r)
   int64_t        slot_count;// rows of codes and scales; a slot outside is skipped
   int64_t        ld, rows, k;
   int            type;
   int            fit;
};
hipError_t launch_quantize(const QuantizeParams& p, hipStream_t s);

struct DequantizeParams {
   const uint8_t* codes;
   const uint8_t* scales;
   void*          out;       // rows x k, leading dimension ld (elements)
   int64_t        ld, rows, k;
   int            type;
};
hipError_t launch_dequantize(const DequantizeParams& p, hipStream_t s);

// A paged cache: token t of sequence b is row table[b * width + t / page] * page + t % page
// of codes and scales; pages outside [0, pages) read as zeros.
struct CacheParams {
   const uint8_t* codes;
   const uint8_t* scales;
   const int32_t* table;
   const int32_t* lens;
   int64_t        pages, channels, width, batch;
   int            page_log;
};
hipError_t launch_cache_read(const CacheParams& c, void* out, int type, int64_t length, bool channels_first,
                             hipStream_t s);
hipError_t launch_cache_conv(const CacheParams& c, const void* taps, int tap_type, int64_t tap_count, void* out,
                             int out_type, float* work, int64_t splits, hipStream_t s);

struct MatmulParams {
   const void*    x;         // mx4 codes (m x kp / 2), or rows of x_type with leading dimension ldx
   const uint8_t* x_scales;  // m x kp / 32 (mx4 only)
   const uint8_t* w;         // n x kp / 2
   const uint8_t* w_scales;  // n x kp / 32
   const float*   bias;      // n, or NULL
   void*          out;       // m x n, leading dimension ld
   int64_t        ldx, ld, m, n, k;
   int            x_type;    // linear only
   int            type;
};
hipError_t launch_matmul(const MatmulParams& p, hipStream_t s);
hipError_t launch_linear(const MatmulParams& p, hipStream_t s);

}  // namespace mx4
}  // namespace fufft
