// mx4_scan_launch.hpp -- which instance of k_mx4_scan runs, and on how many workgroups.
#pragma once
#include "vsgpu_internal.hpp"
#include "mx4_host.hpp"
#include "mx4_scan_kernels.hpp"

namespace vsg {

template <int BITS, int QT, int MODE, int NB, int SRC> static int launch_scan(hipStream_t s, const Mx4Scan &P, const Mx4ScanShape &shape) {
    const uint32_t waves = SRC == MX4_REGS && P.groups == 3 ? 3 : 4, groups = SRC == MX4_REGS ? P.groups : 1, abreast = waves / groups;
    const uint32_t y = SRC == MX4_REGS ? 1 : shape.y;   // (REGS: all of a batch's tiles in one workgroup)
    const size_t lds = mx4_scan_lds(SRC, QT, groups, P.qtile_bytes);
    if (lds > 64 * 1024)
        (void)hipFuncSetAttribute(reinterpret_cast<const void *>(k_mx4_scan<BITS, QT, MODE, NB, SRC>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    const uint64_t gx = MODE == MX4_FILTER ? P.segments : mx4_scan_grid(BITS, QT, MODE, NB, SRC, lds, P.n_take, P.rows.kg, abreast, shape.cus, y);
    hipLaunchKernelGGL((k_mx4_scan<BITS, QT, MODE, NB, SRC>), dim3((unsigned)gx, y), dim3(64 * waves), lds, s, P);
    HIPCHK(hipGetLastError());
    return VSGPU_OK;
}
template <int BITS, int QT, int MODE, int SRC> static int launch_chunks(hipStream_t s, const Mx4Scan &P, const Mx4ScanShape &shape) {
    switch (P.rows.kg) {
    case 1: return launch_scan<BITS, QT, MODE, 1, SRC>(s, P, shape);
    case 2: return launch_scan<BITS, QT, MODE, 2, SRC>(s, P, shape);
    case 3: return launch_scan<BITS, QT, MODE, 3, SRC>(s, P, shape);
    default: return launch_scan<BITS, QT, MODE, 4, SRC>(s, P, shape);
    }
}
template <int BITS, int QT, int MODE, int NB, int M> static int launch_ring4(hipStream_t s, const Mx4Scan &P, const Mx4ScanShape &shape) {
    const size_t lds = (size_t)mx4_ring_bytes(NB) + MX4_RING_WAVES * QT * 256;
    (void)hipFuncSetAttribute(reinterpret_cast<const void *>(k_mx4_ring<BITS, QT, MODE, NB, M>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    const uint64_t gx = MODE == MX4_FILTER ? P.segments : std::min<uint64_t>(P.n_take, (uint64_t)shape.cus);
    hipLaunchKernelGGL((k_mx4_ring<BITS, QT, MODE, NB, M>), dim3((unsigned)gx), dim3(64 * MX4_RING_WAVES), lds, s, P);
    HIPCHK(hipGetLastError());
    return VSGPU_OK;
}
template <int BITS, int QT, int MODE, int NB> static int launch_ring3(hipStream_t s, const Mx4Scan &P, const Mx4ScanShape &shape) {
    if (P.metric == MX4_L2) return launch_ring4<BITS, QT, MODE, NB, MX4_L2>(s, P, shape);
    if (P.metric == MX4_IP) return launch_ring4<BITS, QT, MODE, NB, MX4_IP>(s, P, shape);
    return launch_ring4<BITS, QT, MODE, NB, MX4_COSINE>(s, P, shape);
}
template <int BITS, int QT, int MODE> static int launch_ring(hipStream_t s, const Mx4Scan &P, const Mx4ScanShape &shape) {
    if constexpr (QT == 2)
        if (P.rows.kg == 2) return launch_ring3<BITS, QT, MODE, 2>(s, P, shape);
    return P.rows.kg == 3 ? launch_ring3<BITS, QT, MODE, 3>(s, P, shape) : launch_ring3<BITS, QT, MODE, 4>(s, P, shape);
}
template <int BITS, int MODE> static int launch_mode(hipStream_t s, const Mx4Scan &P, const Mx4ScanShape &shape) {
    if (shape.src == MX4_GLOBAL) return launch_scan<BITS, 1, MODE, 4, MX4_GLOBAL>(s, P, shape);
    if constexpr (MODE == MX4_DENSE || MODE == MX4_PROBE_ROWS) {
        if (shape.src == MX4_REGS) return launch_chunks<BITS, 2, MODE, MX4_REGS>(s, P, shape);
    } else if (shape.ring) {
        return shape.qt == 1 ? launch_ring<BITS, 1, MODE>(s, P, shape) : launch_ring<BITS, 2, MODE>(s, P, shape);
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
