// Copies of arrays whose rows begin anywhere, for kernels whose operands the copy engine fetches: it wants rows that begin on multiples of
// 16 bytes.
#ifndef MOPS_B200_PACK_HPP
#define MOPS_B200_PACK_HPP

#include "arrays.hpp"

namespace mops_b200 {

// For the length of a call: the arrays that need it are copied into scratch memory, rows a multiple of 16 bytes apart, all in one launch.
class Packing {
  public:
    explicit Packing(const Call& call) : call_(call) {}
    ~Packing() {
        try {
            release();
        } catch (...) { // (there is an exception already)
        }
    }
    Packing(const Packing&) = delete;
    Packing& operator=(const Packing&) = delete;

    // Replaces the array (of 2 dimensions, or of 3 of which either of the last two has a stride of 1) where it has to be copied.
    void add(Array& a);
    void run();     // the copies, on the call's stream
    void release(); // the scratch memory, once what reads the copies is launched

    struct Job {
        const void* from;
        void* to;
        int64_t outer, outer_stride, slice_stride, slices; // strides of `from`, in values
        int64_t inner, packs;                              // values of a row, and 16-byte pieces of a row of `to`
        const unsigned char *begin, *end;                  // the bytes that `from` reaches over
    };
    static constexpr int kMost = 3;

  private:
    const Call& call_;
    Job jobs_[kMost];
    int n_ = 0;
    int32_t type_ = 0;
};

#ifdef __CUDACC__
// n values (8 of 16 bits, 4 of 32; zeros behind them where n is less) from wherever p is: of 16-bit values from the two vectors that they lie in, where both are inside of [begin, end), else value by value.
template <typename T>
__device__ __forceinline__ uint4 load_anywhere(const T* p, int64_t n, const unsigned char* begin, const unsigned char* end) {
    constexpr int kValues = kPack<T>;
    uint32_t w[8] = {};
    const uint32_t shift = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15;
    const unsigned char* from = reinterpret_cast<const unsigned char*>(p) - shift;
    if (sizeof(T) == 2 && n >= kValues && from >= begin && from + 32 <= end) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(from)), v = __ldg(reinterpret_cast<const uint4*>(from) + 1);
        w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w, w[4] = v.x, w[5] = v.y, w[6] = v.z, w[7] = v.w;
        // down by 8, 4 and 2 bytes as needed
        if (shift & 8) {
#pragma unroll
            for (int i = 0; i < 6; i++) w[i] = w[i + 2];
        }
        if (shift & 4) {
#pragma unroll
            for (int i = 0; i < 5; i++) w[i] = w[i + 1];
        }
        if (shift & 2) {
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kValues; i++) {
            if (i >= n) continue;
            if constexpr (sizeof(T) == 2) w[i / 2] |= static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(p) + i)) << (16 * (i & 1));
            else w[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
#endif

} // namespace mops_b200

#endif
