// Checks of runtime.cu's host logic over fake_cudart.cpp; the argument names one.
// Exit status: 0 it holds, 1 it does not.
#include <stdio.h>
#include <string.h>

#include <thread>

#include "runtime.h"

using namespace nxv;

#define CHECK(x)                                       \
    do {                                               \
        if (!(x)) return printf("not so: %s\n", #x), 1; \
    } while (0)

// Either way of initialising gives the kernels a place for their report.
static int init_default_has_wait_flag() {
    Ctx c;
    CHECK(init_default() == OK && begin(c, {}) == OK);
    CHECK(wait_flag(c) != nullptr && *wait_flag(c) == 0);
    CHECK(!wait_ran_out(c));
    return 0;
}
static int init_devices_has_wait_flag() {
    Ctx c;
    const int ids[] = {1, 0};
    CHECK(init_devices(ids, 2) == OK && begin(c, {}) == OK && c.dev->id == 1);
    CHECK(wait_flag(c) != nullptr && *wait_flag(c) == 0);
    *wait_flag(c) = 1;
    CHECK(wait_ran_out(c));
    CHECK(!wait_ran_out(c));
    return 0;
}

// A wait that ran out on one device is no other device's report, nor taken by it.
static int wait_report_is_its_devices() {
    Ctx a, b;
    const int ids[] = {0, 1};
    CHECK(init_devices(ids, 2) == OK && begin(a, {}) == OK);
    CHECK(set_current(1) == OK && begin(b, {}) == OK);
    *wait_flag(a) = 1;
    CHECK(!wait_ran_out(b));
    CHECK(wait_ran_out(a));
    CHECK(!wait_ran_out(a) && !wait_ran_out(b));
    return 0;
}
// A thread that asks does not take the report from the other threads of the device; each is
// told once.
static int wait_report_reaches_every_thread() {
    Ctx c;
    CHECK(init_default() == OK && begin(c, {}) == OK);
    CHECK(!wait_ran_out(c));
    *wait_flag(c) = 1;
    bool first = false, second = true;
    std::thread([&] { first = wait_ran_out(c), second = wait_ran_out(c); }).join();
    CHECK(first && !second);
    CHECK(wait_ran_out(c));
    CHECK(!wait_ran_out(c));
    *wait_flag(c) = 1;
    CHECK(wait_ran_out(c));
    CHECK(!wait_ran_out(c));
    return 0;
}

// A call that fails is told so itself; the next one on the thread is not.
static int failed_scratch_is_its_call_s() {
    Ctx c;
    CHECK(init_default() == OK && begin(c, {}) == OK);
    CHECK(scratch(c, (size_t)1 << 38) == nullptr);
    CHECK(finish(c) == OK);
    CHECK(scratch(c, 1000) != nullptr && finish(c) == OK);
    return 0;
}
static int failed_call_is_its_call_s() {
    Ctx c;
    CHECK(init_default() == OK && begin(c, {}) == OK);
    auto call = [] {
        NXV_CK(cudaSetDevice(7));
        return (int)OK;
    };
    CHECK(call() == E_CUDA);
    CHECK(finish(c) == OK);
    return 0;
}

int main(int argc, char** argv) {
    const struct {
        const char* name;
        int (*run)();
    } all[] = {
        {"init_default_has_wait_flag", init_default_has_wait_flag},
        {"init_devices_has_wait_flag", init_devices_has_wait_flag},
        {"wait_report_is_its_devices", wait_report_is_its_devices},
        {"wait_report_reaches_every_thread", wait_report_reaches_every_thread},
        {"failed_scratch_is_its_call_s", failed_scratch_is_its_call_s},
        {"failed_call_is_its_call_s", failed_call_is_its_call_s},
    };
    for (auto& t : all)
        if (argc == 2 && !strcmp(argv[1], t.name)) return t.run();
    for (auto& t : all) puts(t.name);
    return argc == 1 ? 0 : 2;
}
