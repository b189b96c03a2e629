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

} // namespace mops_b200

#endif
