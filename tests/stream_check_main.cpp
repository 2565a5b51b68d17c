// Host check of mc::stream_on_current_device (mc_types.h): the HIP calls that it makes are replaced by ones that fail on demand and keep a last error
// as the runtime does.  Prints one line per scenario; test_stream_check_cpu.py reads them.
#include <stdio.h>
#include "mc_types.h"

static hipError_t lastError = hipSuccess, onGetDevice = hipSuccess, onStreamGetDevice = hipSuccess;
static int currentDevice = 0, streamDevice = 0;

static hipError_t answer(hipError_t e) {
    if (e != hipSuccess) lastError = e;
    return e;
}
extern "C" {
hipError_t hipGetDevice(int* d) { *d = currentDevice; return answer(onGetDevice); }
hipError_t hipStreamGetDevice(hipStream_t, hipDevice_t* d) { *d = streamDevice; return answer(onStreamGetDevice); }
hipError_t hipPeekAtLastError() { return lastError; }
hipError_t hipGetLastError() { hipError_t e = lastError; lastError = hipSuccess; return e; }
const char* hipGetErrorString(hipError_t) { return "error"; }
}
namespace mc { void set_error(const char*, ...) {} }

static void scenario(const char* name, hipError_t getDevice, hipError_t streamGetDevice, int device, hipError_t before, bool stream) {
    onGetDevice = getDevice;
    onStreamGetDevice = streamGetDevice;
    streamDevice = device;
    lastError = before;
    int handle = 0;
    const bool on = mc::stream_on_current_device(stream ? (mcStream_t)&handle : nullptr);
    printf("%s %d %d\n", name, (int)on, mc::launch_status("launch"));
}

int main() {
    scenario("same", hipSuccess, hipSuccess, 0, hipSuccess, true);
    scenario("other", hipSuccess, hipSuccess, 1, hipSuccess, true);
    scenario("null", hipErrorNoDevice, hipErrorInvalidHandle, 1, hipSuccess, false);
    scenario("stream-unknown", hipSuccess, hipErrorInvalidHandle, 0, hipSuccess, true);
    scenario("device-unknown", hipErrorNoDevice, hipSuccess, 0, hipSuccess, true);
    scenario("failed-before", hipSuccess, hipErrorInvalidHandle, 0, hipErrorInvalidValue, true);
    return 0;
}
