// mx4_scan_launch.hpp -- which instance of k_mx4_scan runs, and on how many workgroups.
#pragma once
#include "vsgpu_internal.hpp"
#include "mx4_host.hpp"
#include "mx4_scan_kernels.hpp"

namespace vsg {

template <int BITS, int QT, int MODE, int NB, int SRC> static int launch_scan(hipStream_t s, const Mx4Scan &P, const Mx4ScanShape &shape) {
    const uint32_t waves = SRC == MX4_REGS ? (P.groups == 3 ? 3 : 4) : 4, abreast = waves / P.groups;
    const size_t lds = (SRC == MX4_SHARED ? (size_t)QT * P.qtile_bytes : 0) + P.groups * QT * 256 + (MODE == MX4_FILTER ? 4 * MX4_QUEUE * 16 : 0);
    if (lds > 64 * 1024)
        (void)hipFuncSetAttribute(reinterpret_cast<const void *>(k_mx4_scan<BITS, QT, MODE, NB, SRC>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    // as many workgroups as stay resident; few panels: fewer, so that a wave's start is not most of its work
    const uint64_t fit = std::max<uint64_t>(1, std::min<uint64_t>(mx4_scan_waves(BITS, QT, MODE, NB, SRC), (160 * 1024) / (lds + 512)));
    const uint64_t gx = std::max<uint64_t>(1, std::min<uint64_t>((P.n_take + abreast - 1) / abreast, (uint64_t)shape.cus * fit / shape.y));
    hipLaunchKernelGGL((k_mx4_scan<BITS, QT, MODE, NB, SRC>), dim3((unsigned)gx, shape.y), dim3(64 * waves), lds, s, P);
    HIPCHK(hipGetLastError());
    return VSGPU_OK;
}
template <int BITS, int MODE> static int launch_mode(hipStream_t s, const Mx4Scan &P, const Mx4ScanShape &shape) {
    if (shape.src == MX4_GLOBAL) return launch_scan<BITS, 1, MODE, 4, MX4_GLOBAL>(s, P, shape);
    if (shape.src == MX4_REGS) {
        switch (P.rows.kg) {
        case 1: return launch_scan<BITS, 2, MODE, 1, MX4_REGS>(s, P, shape);
        case 2: return launch_scan<BITS, 2, MODE, 2, MX4_REGS>(s, P, shape);
        case 3: return launch_scan<BITS, 2, MODE, 3, MX4_REGS>(s, P, shape);
        default: return launch_scan<BITS, 2, MODE, 4, MX4_REGS>(s, P, shape);
        }
    }
    if (P.rows.kg == 1) return shape.qt == 1 ? launch_scan<BITS, 1, MODE, 1, MX4_SHARED>(s, P, shape) : launch_scan<BITS, 2, MODE, 1, MX4_SHARED>(s, P, shape);
    return shape.qt == 1 ? launch_scan<BITS, 1, MODE, 4, MX4_SHARED>(s, P, shape) : launch_scan<BITS, 2, MODE, 4, MX4_SHARED>(s, P, shape);
}
template <int BITS> static int mx4_scan(hipStream_t s, int mode, const Mx4Scan &P, const Mx4ScanShape &shape) {
    switch (mode) {
    case MX4_PROBE: return launch_mode<BITS, MX4_PROBE>(s, P, shape);
    case MX4_PROBE_ROWS: return launch_mode<BITS, MX4_PROBE_ROWS>(s, P, shape);
    case MX4_FILTER: return launch_mode<BITS, MX4_FILTER>(s, P, shape);
    default: return launch_mode<BITS, MX4_DENSE>(s, P, shape);
    }
}

}  // namespace vsg
