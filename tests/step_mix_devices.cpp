// The host code of the adapters, the router and the experts (step_mix_api.cpp) over a model of the HIP calls it makes, for
// test_host_mix_devices.py: two devices; an address's device is its upper half - 1 (0: host memory), a stream's its handle / 16 - 1
// (the null stream: the current one).
#include STEP_API

#include <string>

static int current = 0, launches = 0;
static std::string message;

namespace qkv {
void set_error(const char * msg) { message = msg; }
static hipError_t launched(hipStream_t) { return launches++, hipSuccess; }
void lora_plan(LoraArgs & a) { a.rp = 16, a.chunks = a.slots = 1; }
void route_plan(RouteArgs & a) { a.chunks = 2; }
long long moe_plan(MoeArgs &, int, uint8_t *) { return 256; }
hipError_t launch_lora(const LoraArgs &, int, int, hipStream_t st) { return launched(st); }
hipError_t launch_logits(const RouteArgs &, int, int, hipStream_t st) { return launched(st); }
hipError_t launch_route(const RouteArgs &, int, int, hipStream_t st) { return launched(st); }
hipError_t launch_moe(const MoeArgs &, int, const RouteArgs *, hipStream_t st) { return launched(st); }
} // namespace qkv

extern "C" {
hipError_t hipGetDevice(int * d) { return *d = current, hipSuccess; }
hipError_t hipStreamGetDevice(hipStream_t st, hipDevice_t * d) {
    *d = st ? (int) ((uintptr_t) st / 16) - 1 : current;
    return *d < 2 ? hipSuccess : hipErrorInvalidHandle;
}
hipError_t hipPointerGetAttributes(hipPointerAttribute_t * at, const void * p) {
    at->device = (int) ((uintptr_t) p >> 32) - 1;
    at->type = hipMemoryTypeDevice;
    return at->device >= 0 ? hipSuccess : hipErrorInvalidValue;
}
const char * hipGetErrorString(hipError_t) { return "an error"; }
hipError_t hipGetLastError() { return hipSuccess; }

void model_device(int d) { current = d; }
int model_launches() { return launches; }
const char * model_message() { return message.c_str(); }
}
