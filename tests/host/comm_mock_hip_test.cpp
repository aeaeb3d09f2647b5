// comm_mock_hip_test.cpp -- api_comm.cpp against a stand-in for the HIP runtime that only writes down what it is asked for:
// what the set-up and the end of an exchange between ranks do to memory, without a device.
// Usage: comm_mock_hip_test <case>; exit code 0 = pass.
#include <sys/wait.h>
#include <unistd.h>

#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <set>
#include <string>
#include <vector>

#include "../../tracking_sdf_amd/csrc/handle.hpp"

#define CHECK(c) do { if (!(c)) { std::fprintf(stderr, "CHECK failed: %s (%s:%d)\n", #c, __FILE__, __LINE__); return 1; } } while (0)

// ---- the stand-in runtime
static std::vector<std::string> calls;             // names, in order
static std::set<void*> uncached, freed;            // what hipExtMallocWithFlags handed out uncached / what hipFree was given
static int count(const char* name) { return (int)std::count(calls.begin(), calls.end(), std::string(name)); }
static long last(const char* name) {
    for (size_t i = calls.size(); i-- > 0;) if (calls[i] == name) return (long)i;
    return -1;
}
static long first(const char* name) {
    for (size_t i = 0; i < calls.size(); ++i) if (calls[i] == name) return (long)i;
    return -1;
}
extern "C" {
hipError_t hipMalloc(void** p, size_t n) { calls.push_back("hipMalloc"); *p = std::calloc(1, n); return hipSuccess; }
hipError_t hipExtMallocWithFlags(void** p, size_t n, unsigned flags) {
    calls.push_back("hipExtMallocWithFlags"); *p = std::calloc(1, n);
    if (flags == hipDeviceMallocUncached) uncached.insert(*p);
    return hipSuccess;
}
hipError_t hipFree(void* p) { calls.push_back("hipFree"); freed.insert(p); return hipSuccess; }      // (kept: the test compares addresses)
hipError_t hipMemsetAsync(void* p, int v, size_t n, hipStream_t) { calls.push_back("hipMemsetAsync"); std::memset(p, v, n); return hipSuccess; }
hipError_t hipMemcpy(void* d, const void* s, size_t n, hipMemcpyKind) { calls.push_back("hipMemcpy"); std::memcpy(d, s, n); return hipSuccess; }
hipError_t hipMemcpyAsync(void* d, const void* s, size_t n, hipMemcpyKind, hipStream_t) { calls.push_back("hipMemcpyAsync"); std::memcpy(d, s, n); return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { calls.push_back("hipStreamSynchronize"); return hipSuccess; }
hipError_t hipIpcGetMemHandle(hipIpcMemHandle_t* h, void* p) { calls.push_back("hipIpcGetMemHandle"); std::memset(h, 0, sizeof *h); std::memcpy(h, &p, sizeof p); return hipSuccess; }
hipError_t hipIpcOpenMemHandle(void** p, hipIpcMemHandle_t, unsigned) { calls.push_back("hipIpcOpenMemHandle"); *p = std::calloc(1, 1 << 16); return hipSuccess; }
hipError_t hipIpcCloseMemHandle(void*) { calls.push_back("hipIpcCloseMemHandle"); return hipSuccess; }
hipError_t hipHostRegister(void*, size_t, unsigned) { calls.push_back("hipHostRegister"); return hipErrorInvalidValue; }
hipError_t hipHostUnregister(void*) { calls.push_back("hipHostUnregister"); return hipSuccess; }
hipError_t hipHostGetDevicePointer(void** d, void* h, unsigned) { *d = h; return hipSuccess; }
hipError_t hipGetLastError(void) { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "stand-in"; }
}

// ---- what api_comm.cpp takes from the library's other files
namespace tsdf_api {
int fail(tsdf_handle* h, int code, const char* fmt, ...) {
    char buf[512]; va_list ap; va_start(ap, fmt); vsnprintf(buf, sizeof buf, fmt, ap); va_end(ap);
    std::fprintf(stderr, "%s\n", buf);
    if (h) h->err = buf;
    return code;
}
int check_ready(tsdf_handle* h, bool) { return h ? TSDF_OK : TSDF_E_BADARG; }
}
namespace tsdf {
void AqlQueue::destroy() {}
hipError_t launch_peer_exchange(hipStream_t, const PeerExchange&, double*, int, double*, unsigned long long) { return hipSuccess; }
}

static std::string seg_name(const char* what) { return "/tsdf_mock_" + std::to_string((long)getpid()) + "_" + what; }

// the fan-in over shared memory never page-locks the segment: memory that exists already is refused, and the error that the
// refusal leaves behind would be reported by whatever HIP call comes next
static int case_shm_registers_nothing() {
    for (bool host_fold : {true, false}) {
        tsdf_handle h;
        h.host_fold = host_fold;
        double row[tsdf::kRedWidth] = {1.0, 2.0};
        h.red_host = row;
        calls.clear();
        CHECK(tsdf_comm_init_shm(&h, 1, 0, seg_name("shm").c_str()) == TSDF_OK);
        double buf[2] = {3.0, 4.0};
        CHECK(tsdf_allreduce(&h, buf, 2) == TSDF_OK && buf[0] == 3.0 && buf[1] == 4.0);
        CHECK(tsdf_comm_finalize(&h) == TSDF_OK && !h.shm.active());
        CHECK(count("hipHostRegister") == 0 && count("hipHostUnregister") == 0);
        calls.clear();
        CHECK(tsdf_comm_init_peer(&h, 1, 0, seg_name("peer").c_str()) == TSDF_OK && h.peer.active());
        CHECK(tsdf_comm_finalize(&h) == TSDF_OK && !h.peer.active());
        CHECK(count("hipHostRegister") == 0);
    }
    return 0;
}

// uncached device memory that a kernel has read is never given back before the process ends: allocations made after such
// a free have held wrong values.  However the exchange ends -- finalized, set up again, replaced by the plain fan-in.
static int case_peer_keeps_its_buffer() {
    for (int way = 0; way < 3; ++way) {
        tsdf_handle h;
        double row[tsdf::kRedWidth] = {0.0};
        h.red_host = row;
        h.red_dev = row;
        CHECK(tsdf_comm_init_peer(&h, 1, 0, seg_name("keep").c_str()) == TSDF_OK && h.peer.active());
        char* const own = h.peer.own;
        CHECK(uncached.count(own) == 1);
        if (way == 1) { CHECK(tsdf_comm_init_peer(&h, 1, 0, seg_name("again").c_str()) == TSDF_OK && h.peer.own != own); }
        if (way == 2) { CHECK(tsdf_comm_init_shm(&h, 1, 0, seg_name("plain").c_str()) == TSDF_OK && !h.peer.active()); }
        CHECK(tsdf_comm_finalize(&h) == TSDF_OK && !h.peer.active());
        for (void* p : uncached) CHECK(freed.count(p) == 0);
        CHECK(count("hipFree") == count("hipMalloc"));          // the pointer table, ordinary memory, does go back
    }
    return 0;
}

int main(int argc, char** argv) {
    const std::string c = argc > 1 ? argv[1] : "";
    if (c == "shm_registers_nothing") return case_shm_registers_nothing();
    if (c == "peer_keeps_its_buffer") return case_peer_keeps_its_buffer();
    std::fprintf(stderr, "unknown case %s\n", c.c_str());
    return 2;
}
