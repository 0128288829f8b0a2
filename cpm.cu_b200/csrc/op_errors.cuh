// What the kernels of the operators on the caller's streams report (a wait that ran out, a slot behind the cache).
//
// Events are counted in device memory and nothing clears the counters: a check compares them with what its stream has been told, so that it takes
// away nothing that another stream, or a later launch, reports.  Each stream has counters of its own, found by the stream's id (a handle
// may come back for another stream).  Launches that are being captured, whose graph may run on any stream, share one set, and every stream is told of those.
#pragma once
#include "common.cuh"

enum OpError : int { OP_TIMEOUT = 0, OP_KV_OVERFLOW = 1, OP_ERROR_KINDS = 2 };
typedef unsigned OpCount;   // (of 64 bits: a row's rotation 2 % slower, 3000 rows of 8 + 2 * 2 heads of 128 6.75 -> 6.9 us)

// the counters [OP_ERROR_KINDS] of a launch on s
OpCount* op_counters(cudaStream_t s);

struct OpErrors {
    int own = 0, shared = 0;   // KernelError bits of the stream's launches, and of graphs' launches on any stream
};
// Waits for s.  What has been reported since the last call for it; s must not be in a capture.
OpErrors new_op_errors(cudaStream_t s);

__device__ __forceinline__ void report(OpCount* counters, OpError what) { atomicAdd(counters + what, 1u); }
