// Sequence operators: parameters and launchers (defined in nsfps_embed.hip,
// nsfps_conv.hip, nsfps_scan.hip and nsfps_scan_grad.hip; called by
// nsfps_sequence.cpp).  Not part of the C ABI.
#pragma once

#include "nsfps.h"

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace nsfps {

hipError_t preload_embed_kernels();
hipError_t preload_conv_kernels();
hipError_t preload_scan_kernels();
hipError_t preload_scan_grad_kernels();

// Arguments arrive checked: sizes within the limits of the header, strides of
// at least a row, no null pointer where one is needed, no empty grid.

// embedding (nsfps_embed.hip)
hipError_t launch_embed(const nsfps_embed_args &a, hipStream_t st);
uint64_t embed_grad_bytes(const nsfps_embed_args &a);
hipError_t launch_embed_grad(const nsfps_embed_args &a, hipStream_t st);

// convolution (nsfps_conv.hip)
hipError_t launch_conv(const nsfps_conv_args &a, hipStream_t st);
uint64_t conv_grad_bytes(const nsfps_conv_args &a);
hipError_t launch_conv_grad(const nsfps_conv_args &a, const nsfps_conv_grads &g, hipStream_t st);

// scan (nsfps_scan.hip, nsfps_scan_grad.hip)
uint64_t scan_bytes(const nsfps_scan_args &a);
hipError_t launch_scan(const nsfps_scan_args &a, hipStream_t st);
uint64_t scan_grad_bytes(const nsfps_scan_args &a);
hipError_t launch_scan_grad(const nsfps_scan_args &a, const nsfps_scan_grads &g, hipStream_t st);
hipError_t launch_scan_step(const nsfps_step_args &a, hipStream_t st);

}  // namespace nsfps
