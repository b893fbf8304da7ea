"""The C++ host layer's calls of the request-batch operators compile, link
against the library and turn its refusals into the reference's exceptions
(no device needed: every call is refused before one is touched)."""

import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include "sam_hip.hpp"
#include <cstdio>
#include <stdexcept>
using namespace sam;
// the members exist with these signatures
static void (HipBackend::*lora)(const samhip_lora_bank&, const samhip_tensor&, const samhip_tensor&, const samhip_tensor*, const samhip_tensor&) =
    &HipBackend::lora_add;
static void (HipBackend::*attn)(const samhip_prefix_attn_desc&) = &HipBackend::prefix_attn;
static void (HipBackend::*norm)(const samhip_tensor&, const samhip_tensor&, int32_t, const float*, const float*, float, samhip_activation) =
    &HipBackend::group_norm;
template <class F> static bool refused(F f) {
    try { f(); } catch (const std::invalid_argument& e) { return std::string(e.what()).find("null context") != std::string::npos; }
    return false;
}
int main() {
    samhip_tensor t = make_tensor(SAMHIP_TYPE_F32, 64, 4, 4, 256, reinterpret_cast<void*>(0x1000));
    samhip_lora_bank bank{};
    samhip_prefix_attn_desc desc{};
    const bool ok = lora && attn && norm && refused([&] { check_status(samhip_lora_add(nullptr, &bank, &t, &t, nullptr, &t)); }) &&
                    refused([&] { check_status(samhip_prefix_attn(nullptr, &desc)); }) &&
                    refused([&] { check_status(samhip_group_norm(nullptr, &t, &t, 8, nullptr, nullptr, 1e-5f, SAMHIP_ACT_RELU)); }) &&
                    !samhip_supports_lora_add(&bank, &t, &t, nullptr, &t) && !samhip_supports_prefix_attn(&desc) &&
                    samhip_supports_group_norm(&t, &t, 8, nullptr, nullptr, 1e-5f, SAMHIP_ACT_RELU);
    std::puts(ok ? "ok" : "wrong");
    return ok ? 0 : 1;
}
"""


def test_host_layer_calls(tmp_path):
    src, exe = tmp_path / "calls.cpp", tmp_path / "calls"
    src.write_text(SOURCE)
    lib = os.path.join(ROOT, "sam.cpp_amd")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(lib, "host"), str(src), "-o",
                    str(exe), "-L", lib, "-lsamhip", "-Wl,-rpath," + lib], check=True, timeout=300)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out
