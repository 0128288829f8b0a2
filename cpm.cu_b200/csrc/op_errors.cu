// Host side of op_errors.cuh.
#include "op_errors.cuh"

#include <mutex>
#include <type_traits>
#include <unordered_map>

namespace {

constexpr int SETS = 1024;   // set 0 is shared; streams beyond the last one use it too

struct Known {
    int set = 0;
    std::mutex checking;   // of two checks of a stream at once the later one has the later counts
    OpCount own[OP_ERROR_KINDS] = {}, shared[OP_ERROR_KINDS] = {};   // told so far
};
struct Registry {
    std::mutex lock;
    std::unordered_map<unsigned long long, Known> streams;   // by id
    int sets = 1;
};
Registry& registry() {
    static Registry r;
    return r;
}

OpCount* counters(int set) { return runtime().d_op_errors + set * OP_ERROR_KINDS; }

Known& known(Registry& r, unsigned long long id) {   // the lock is held
    const auto [at, fresh] = r.streams.try_emplace(id);
    if (fresh && r.sets < SETS) at->second.set = r.sets++;
    return at->second;
}

// Whether s is in a capture, and else its id, by the driver's own entry points: 24 ns, through the runtime's 80, on every launch that may report.  They want
// a current context, which a thread that has not called the runtime yet lacks.
struct StreamQuery {
    CUresult (*capturing)(CUstream, CUstreamCaptureStatus*) = nullptr;
    CUresult (*id)(CUstream, unsigned long long*) = nullptr;
    StreamQuery() {
        auto find = [](const char* name, auto& fn) {
            void* p = nullptr;
            cudaDriverEntryPointQueryResult found;
            if (cudaGetDriverEntryPoint(name, &p, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) p = nullptr;
            fn = reinterpret_cast<std::decay_t<decltype(fn)>>(p);
        };
        find("cuStreamIsCapturing", capturing);
        find("cuStreamGetId", id);
    }
};
bool id_outside_captures(cudaStream_t s, unsigned long long& id) {
    static const StreamQuery ask;
    CUstreamCaptureStatus state;
    if (ask.capturing != nullptr && ask.id != nullptr && ask.capturing(s, &state) == CUDA_SUCCESS) {
        if (state != CU_STREAM_CAPTURE_STATUS_NONE) return false;
        if (ask.id(s, &id) == CUDA_SUCCESS) return true;
    }
    cudaStreamCaptureStatus capture;
    if (cudaStreamIsCapturing(s, &capture) == cudaSuccess && capture == cudaStreamCaptureStatusNone && cudaStreamGetId(s, &id) == cudaSuccess) return true;
    cudaGetLastError();   // what is wrong with the stream the launch will say
    return false;
}

// While a stream is captured in CUDA's default mode, no thread may wait or copy, on any stream: it would end that capture.  What a check waits for and copies is
// no part of a capture, which the relaxed mode says.
struct BesideCaptures {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    BesideCaptures() { CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode)); }
    ~BesideCaptures() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

// KernelError bits of the counters that moved
int moved(const OpCount* now, OpCount* told) {
    constexpr int bit[OP_ERROR_KINDS] = {ERR_GEMM_TIMEOUT, ERR_KV_OVERFLOW};
    int bits = 0;
    for (int k = 0; k < OP_ERROR_KINDS; ++k) {
        if (now[k] != told[k]) bits |= bit[k];
        told[k] = now[k];
    }
    return bits;
}

}  // namespace

size_t op_errors_bytes() { return sizeof(OpCount) * SETS * OP_ERROR_KINDS; }

OpCount* op_counters(cudaStream_t s) {
    unsigned long long id;
    if (!id_outside_captures(s, id)) return counters(0);
    Registry& r = registry();
    std::lock_guard<std::mutex> hold(r.lock);
    const auto at = r.streams.find(id);
    if (at != r.streams.end()) return counters(at->second.set);
    return counters(r.sets < SETS ? known(r, id).set : 0);
}

OpErrors new_op_errors(cudaStream_t s) {
    cudaStreamCaptureStatus capture;
    CUDA_CHECK(cudaStreamIsCapturing(s, &capture));
    CPM_REQUIRE(capture == cudaStreamCaptureStatusNone, "stream_check: the stream is being captured");
    unsigned long long id;
    CUDA_CHECK(cudaStreamGetId(s, &id));
    Registry& r = registry();
    Known* k;   // stays where it is
    {
        std::lock_guard<std::mutex> hold(r.lock);
        k = &known(r, id);
    }
    std::lock_guard<std::mutex> hold(k->checking);
    const BesideCaptures beside;
    OpCount own[OP_ERROR_KINDS], shared[OP_ERROR_KINDS];
    CUDA_CHECK(cudaStreamSynchronize(s));
    CUDA_CHECK(cudaMemcpyAsync(own, counters(k->set), sizeof(own), cudaMemcpyDeviceToHost, s));
    CUDA_CHECK(cudaMemcpyAsync(shared, counters(0), sizeof(shared), cudaMemcpyDeviceToHost, s));
    CUDA_CHECK(cudaStreamSynchronize(s));
    OpErrors e;
    e.shared = moved(shared, k->shared);
    if (k->set != 0) e.own = moved(own, k->own);
    return e;
}
