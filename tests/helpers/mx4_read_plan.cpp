// mx4_read_plan.cpp -- the division of k_mx4_read's work (csrc/mx4_read_plan.h) against ordinary division, for tests/test_mx4.py
#include "mx4_read_plan.h"

using namespace vsg;

// pieces t < end whose row differs from t / per_row
extern "C" long wrong_rows(uint32_t per_row, uint32_t end) {
    const uint32_t r = mx4_reciprocal(per_row);
    long wrong = 0;
    for (uint32_t t = 0; t < end; t++) wrong += mx4_quotient(t, r) != t / per_row;
    return wrong;
}
extern "C" uint32_t pieces(uint32_t dim) { return mx4_read_pieces(dim); }
extern "C" uint32_t rows(uint64_t m, uint32_t per_row, uint32_t cus) { return mx4_read_rows(m, per_row, cus); }
