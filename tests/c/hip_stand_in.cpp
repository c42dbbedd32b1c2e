// A HIP runtime on host memory, for running the library's host code without a GPU: "device" memory is malloc'ed, so that a
// sanitizer sees what the host reads and writes by way of the runtime; copies and fills on a stream are carried out as late as a
// program may rely on (when the stream or an event behind them is waited for); kernels are not run, their launches are checked.  A misuse
// (a copy outside an allocation, a source that changes or goes away under a copy, something destroyed twice, a wait for a stream that is
// being recorded) ends the program with a message.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <map>
#include <mutex>
#include <set>
#include <vector>

namespace {

struct Stream {
    std::vector<std::function<void()>> work;
    size_t done = 0;
    bool recording = false;
};
struct Event {
    Stream* stream = nullptr;
    size_t behind = 0;
};

std::recursive_mutex lock;
#define HOLD std::lock_guard<std::recursive_mutex> hold(lock)
Stream null_stream;
std::set<Stream*> streams;
std::map<const void*, size_t> device, pinned;
std::set<void*> events, graphs, execs;
long launches = 0, copies_until_failure = 0;

[[noreturn]] void misuse(const char* what) {
    std::fprintf(stderr, "HIP stand-in: %s\n", what);
    std::fflush(stderr);
    std::abort();
}
Stream* stream_of(hipStream_t s) {
    if (!s) return &null_stream;
    Stream* p = reinterpret_cast<Stream*>(s);
    if (!streams.count(p)) misuse("a stream that does not exist");
    return p;
}
void carry_out(Stream* s, size_t until) {
    while (s->done < until) {
        const std::function<void()> next = std::move(s->work[s->done++]);
        next();
    }
}
void carry_out_all() {
    carry_out(&null_stream, null_stream.work.size());
    for (Stream* s : streams) carry_out(s, s->work.size());
}
size_t bytes_from(const std::map<const void*, size_t>& memory, const void* p) {
    auto it = memory.upper_bound(p);
    if (it == memory.begin()) return 0;
    --it;
    const size_t offset = static_cast<size_t>(static_cast<const char*>(p) - static_cast<const char*>(it->first));
    return offset < it->second ? it->second - offset : 0;
}
void inside(const void* p, size_t n) {
    if (n && bytes_from(device, p) < n && bytes_from(pinned, p) < n) misuse("device memory outside every allocation");
}
void check(const void* to, const void* from, size_t n, hipMemcpyKind kind) {
    if (kind == hipMemcpyHostToDevice || kind == hipMemcpyDeviceToDevice) inside(to, n);
    if (kind == hipMemcpyDeviceToHost || kind == hipMemcpyDeviceToDevice) inside(from, n);
}
unsigned checksum(const void* p, size_t n) {
    unsigned h = 1;
    for (size_t i = 0; i < n; ++i) h = h * 31 + static_cast<const unsigned char*>(p)[i];
    return h;
}
template <typename T>
void destroy(std::set<void*>& of, T what) {
    HOLD;
    if (!of.erase(what)) misuse("something is destroyed that does not exist");
    std::free(what);
}
void* made(std::set<void*>& in) {
    HOLD;
    void* p = std::calloc(1, 64);
    in.insert(p);
    return p;
}
// (device variables are registered ahead of this file's own statics)
std::map<const void*, size_t>& variable_sizes() {
    static std::map<const void*, size_t> sizes;
    return sizes;
}
std::map<const void*, void*> variables;
thread_local struct {
    dim3 grid, block;
    size_t lds;
    hipStream_t stream;
} configuration;

}  // namespace

extern "C" {

// what the program that drives the library asks of the stand-in
long hip_stand_in_launches() { return launches; }
void hip_stand_in_fail_copy(long after) { copies_until_failure = after; }      // the after-th asynchronous copy from now fails (0: none)
size_t hip_stand_in_memory() { HOLD; return device.size() + pinned.size() + events.size() + graphs.size() + execs.size() + streams.size(); }

void** __hipRegisterFatBinary(const void*) { static void* handle; return &handle; }
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void*, char*, const char*, unsigned, void*, void*, void*, void*, int*) {}
void __hipRegisterVar(void**, void* variable, char*, char*, int, size_t size, int, int) { variable_sizes()[variable] = size; }
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, hipStream_t stream) {
    configuration = {grid, block, lds, stream};
    return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* lds, hipStream_t* stream) {
    *grid = configuration.grid;
    *block = configuration.block;
    *lds = configuration.lds;
    *stream = configuration.stream;
    return hipSuccess;
}
hipError_t hipLaunchKernel(const void*, dim3 grid, dim3 block, void**, size_t lds, hipStream_t stream) {
    HOLD;
    stream_of(stream);
    ++launches;
    const unsigned threads = block.x * block.y * block.z;
    if (!grid.x || !grid.y || !grid.z || !threads || threads > 1024 || grid.y > 65535 || grid.z > 65535 || lds > 160 * 1024 ||
        static_cast<unsigned long long>(grid.x) * block.x >= 1ull << 32)
        misuse("a launch that no GPU takes");
    return hipSuccess;
}
hipError_t hipGetSymbolAddress(void** p, const void* symbol) {
    HOLD;
    void*& v = variables[symbol];
    if (!v) {
        v = std::calloc(1, variable_sizes().at(symbol));
        device[v] = variable_sizes().at(symbol);
    }
    *p = v;
    return hipSuccess;
}
hipError_t hipFuncGetAttributes(hipFuncAttributes* a, const void*) {
    std::memset(a, 0, sizeof *a);
    a->maxThreadsPerBlock = 1024;
    a->numRegs = 64;
    return hipSuccess;
}
hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }
hipError_t hipOccupancyMaxActiveBlocksPerMultiprocessor(int* n, const void*, int, size_t) { *n = 2; return hipSuccess; }

hipError_t hipGetDeviceCount(int* n) { *n = 1; return hipSuccess; }
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipSetDevice(int d) { return d == 0 ? hipSuccess : hipErrorInvalidDevice; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
    std::memset(p, 0, sizeof *p);
    std::strcpy(p->name, "stand-in");
    std::strcpy(p->gcnArchName, "gfx950");
    p->multiProcessorCount = 256;
    p->warpSize = 64;
    p->sharedMemPerBlock = 160 << 10;
    p->totalGlobalMem = size_t(1) << 36;
    return hipSuccess;
}
const char* hipGetErrorString(hipError_t) { return "an error of the stand-in"; }
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipDeviceSynchronize() { HOLD; carry_out_all(); return hipSuccess; }

hipError_t hipMalloc(void** p, size_t n) {
    HOLD;
    *p = std::calloc(1, n);
    if (!*p) return hipErrorOutOfMemory;
    device[*p] = n;
    return hipSuccess;
}
hipError_t hipFree(void* p) {
    HOLD;
    if (!p) return hipSuccess;
    carry_out_all();                 // (it waits for the device)
    if (!device.erase(p)) misuse("freed what is no device memory");
    std::free(p);
    return hipSuccess;
}
hipError_t hipHostMalloc(void** p, size_t n, unsigned) {
    HOLD;
    *p = std::malloc(n);
    if (!*p) return hipErrorOutOfMemory;
    pinned[*p] = n;
    return hipSuccess;
}
hipError_t hipHostFree(void* p) {
    HOLD;
    if (!p) return hipSuccess;
    carry_out_all();
    if (!pinned.erase(p)) misuse("freed what is no pinned memory");
    std::free(p);
    return hipSuccess;
}

hipError_t hipStreamCreate(hipStream_t* s) {
    HOLD;
    Stream* p = new Stream;
    streams.insert(p);
    *s = reinterpret_cast<hipStream_t>(p);
    return hipSuccess;
}
hipError_t hipStreamDestroy(hipStream_t s) {
    HOLD;
    Stream* p = stream_of(s);
    carry_out(p, p->work.size());
    streams.erase(p);
    delete p;
    return hipSuccess;
}
hipError_t hipStreamSynchronize(hipStream_t s) {
    HOLD;
    Stream* p = stream_of(s);
    if (p->recording) misuse("a wait for a stream that is being recorded");
    carry_out(p, p->work.size());
    return hipSuccess;
}
hipError_t hipStreamBeginCapture(hipStream_t s, hipStreamCaptureMode) { HOLD; stream_of(s)->recording = true; return hipSuccess; }
hipError_t hipStreamEndCapture(hipStream_t s, hipGraph_t* g) {
    HOLD;
    stream_of(s)->recording = false;
    *g = static_cast<hipGraph_t>(made(graphs));
    return hipSuccess;
}
hipError_t hipStreamIsCapturing(hipStream_t s, hipStreamCaptureStatus* status) {
    HOLD;
    *status = stream_of(s)->recording ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
    return hipSuccess;
}
hipError_t hipGraphInstantiate(hipGraphExec_t* e, hipGraph_t g, hipGraphNode_t*, char*, size_t) {
    HOLD;
    if (!graphs.count(g)) misuse("a graph that does not exist");
    *e = static_cast<hipGraphExec_t>(made(execs));
    return hipSuccess;
}
hipError_t hipGraphLaunch(hipGraphExec_t e, hipStream_t s) {
    HOLD;
    if (!execs.count(e)) misuse("a recorded step that does not exist");
    stream_of(s);
    return hipSuccess;
}
hipError_t hipGraphExecDestroy(hipGraphExec_t e) { destroy(execs, e); return hipSuccess; }
hipError_t hipGraphDestroy(hipGraph_t g) { destroy(graphs, g); return hipSuccess; }

hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) {
    HOLD;
    Event* p = new (std::calloc(1, sizeof(Event))) Event;
    events.insert(p);
    *e = reinterpret_cast<hipEvent_t>(p);
    return hipSuccess;
}
hipError_t hipEventCreate(hipEvent_t* e) { return hipEventCreateWithFlags(e, 0); }
hipError_t hipEventDestroy(hipEvent_t e) { destroy(events, e); return hipSuccess; }
hipError_t hipEventElapsedTime(float* ms, hipEvent_t, hipEvent_t) { *ms = 0.01f; return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t e, hipStream_t s) {
    HOLD;
    if (!events.count(e)) misuse("an event that does not exist");
    Event* p = reinterpret_cast<Event*>(e);
    p->stream = stream_of(s);
    p->behind = p->stream->work.size();
    return hipSuccess;
}
hipError_t hipEventSynchronize(hipEvent_t e) {
    HOLD;
    if (!events.count(e)) misuse("an event that does not exist");
    Event* p = reinterpret_cast<Event*>(e);
    if (p->stream && p->stream != &null_stream && !streams.count(p->stream)) misuse("an event of a stream that is gone");
    if (p->stream) carry_out(p->stream, p->behind);
    return hipSuccess;
}

hipError_t hipMemcpy(void* to, const void* from, size_t n, hipMemcpyKind kind) {
    HOLD;
    for (Stream* s : streams)
        if (s->recording) misuse("a copy that waits while a stream is being recorded");
    carry_out_all();
    check(to, from, n, kind);
    std::memcpy(to, from, n);
    return hipSuccess;
}
hipError_t hipMemcpyAsync(void* to, const void* from, size_t n, hipMemcpyKind kind, hipStream_t s) {
    HOLD;
    if (copies_until_failure > 0 && --copies_until_failure == 0) return hipErrorUnknown;
    check(to, from, n, kind);
    Stream* p = stream_of(s);
    if (p->recording) return hipSuccess;
    const bool from_host = kind == hipMemcpyHostToDevice;
    const unsigned sum = from_host ? checksum(from, n) : 0;
    p->work.push_back([=] {
        check(to, from, n, kind);
        if (from_host && checksum(from, n) != sum) misuse("the source of a copy was written before the copy was waited for");
        std::memcpy(to, from, n);
    });
    return hipSuccess;
}
hipError_t hipMemset(void* to, int value, size_t n) {
    HOLD;
    carry_out_all();
    inside(to, n);
    std::memset(to, value, n);
    return hipSuccess;
}
hipError_t hipMemsetAsync(void* to, int value, size_t n, hipStream_t s) {
    HOLD;
    Stream* p = stream_of(s);
    if (p->recording) misuse("a fill is recorded");
    inside(to, n);
    p->work.push_back([=] {
        inside(to, n);
        std::memset(to, value, n);
    });
    return hipSuccess;
}
hipError_t hipMemcpy2DAsync(void* to, size_t to_pitch, const void* from, size_t from_pitch, size_t width, size_t height, hipMemcpyKind kind, hipStream_t s) {
    for (size_t i = 0; i < height; ++i) {
        const hipError_t e = hipMemcpyAsync(static_cast<char*>(to) + i * to_pitch, static_cast<const char*>(from) + i * from_pitch, width, kind, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
hipError_t hipMemcpy2D(void* to, size_t to_pitch, const void* from, size_t from_pitch, size_t width, size_t height, hipMemcpyKind kind) {
    for (size_t i = 0; i < height; ++i)
        hipMemcpy(static_cast<char*>(to) + i * to_pitch, static_cast<const char*>(from) + i * from_pitch, width, kind);
    return hipSuccess;
}

}  // extern "C"
