// vsgpu_mx4_scan4.hip -- the table passes of mx4_scan_kernels.hpp for queries of 4 bits (a translation unit of its own: compile time)
#include "mx4_scan_launch.hpp"

int vsg::mx4_scan4(hipStream_t s, int mode, const Mx4Scan &P, const Mx4ScanShape &shape) { return mx4_scan<4>(s, mode, P, shape); }
