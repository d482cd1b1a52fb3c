// mx4_read_plan.h -- how k_mx4_read divides its work (plain C++: the kernel, its launch and a CPU test share it).
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define MX4_BOTH __host__ __device__
#else
#define MX4_BOTH
#endif

namespace vsg {

// A row of dim elements is per_row pieces of eight; a workgroup takes `rows` whole rows: thread t's piece belongs to its row t / per_row.
MX4_BOTH inline uint32_t mx4_read_pieces(uint32_t dim) { return (dim + 7) / 8; }   // 1 .. 8192

// about 1024 pieces a workgroup, fewer when there are not enough rows to fill the chip; rows * per_row stays below 2^16
inline uint32_t mx4_read_rows(uint64_t m, uint32_t per_row, uint32_t cus) {
    const auto least = [](uint64_t a, uint64_t b) { return a < b ? a : b; };
    const auto most = [](uint64_t a, uint64_t b) { return a > b ? a : b; };
    const uint64_t rows = most(1, 1024 / per_row);
    return (uint32_t)most(least(rows, m / ((uint64_t)cus * 8)), most(1, least(256 / per_row, m)));
}

// t / per_row as one multiplication: with r = ceil(2^31 / per_row) the upper half of 2 t r is floor(t / per_row) while
// t (r per_row - 2^31) < 2^31, and that is at most 2^16 2^13.  (2^31 and not 2^32: the reciprocal of 1 has to fit 32 bits.)
MX4_BOTH inline uint32_t mx4_reciprocal(uint32_t per_row) { return (0x80000000u + per_row - 1) / per_row; }
MX4_BOTH inline uint32_t mx4_quotient(uint32_t t, uint32_t reciprocal) { return (uint32_t)(((uint64_t)(2 * t) * reciprocal) >> 32); }

}  // namespace vsg
