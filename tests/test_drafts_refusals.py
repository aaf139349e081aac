"""What the entry points of rotated positions and drafted trees refuse, without a GPU: every check comes before the first use of the device, so a context
that was never initialised is enough.  Addresses of host memory stand for whatever is not device memory."""
import ctypes
import os
import subprocess

import pytest

from __graft_entry__ import ROOT, load_package

pimdl = load_package()

SOURCE = r"""
#include <stdio.h>
#include <functional>
#include "pimdl_internal.h"

static pimdl_ctx* ctx;
static void say(const char* name, int rc) { printf("%s|%d|%s\n", name, rc, rc ? ctx->err.c_str() : ""); }

int main()
{
    ctx = new pimdl_ctx();
    alignas(16) static float host[256];
    static double freqs[64];
    static int32_t ints[64];
    static uint32_t words[64];
    typedef pimdl_rotary R;
    typedef pimdl_rotate_desc D;
    const R r0 = {freqs, 64, PIMDL_PAIRS_HALVES};
    const D d0 = {host, host, host, host, ints, nullptr, 1, 4, 2, 1, 64, 128, 64, 128, 64, PIMDL_F32};
    auto rotate = [&](const char* name, std::function<void(R&, D&)> f) { R r = r0; D d = d0; f(r, d); ctx->err.clear(); say(name, pimdl_rotate(ctx, &r, &d)); };
    rotate("rotate host memory", [](R&, D&) {});
    rotate("rotate nothing", [](R&, D& d) { d.heads = d.kv_heads = 0; });
    rotate("rotate no tokens", [](R&, D& d) { d.tokens = 0; });
    rotate("rotate no batch", [](R&, D& d) { d.batch = 0; });
    rotate("rotate odd dims", [](R& r, D&) { r.dims = 33; });
    rotate("rotate no dims", [](R& r, D&) { r.dims = 0; });
    rotate("rotate many dims", [](R& r, D&) { r.dims = 66; });
    rotate("rotate pairs", [](R& r, D&) { r.pairs = 2; });
    rotate("rotate dtype", [](R&, D& d) { d.dtype = 3; });
    rotate("rotate head_dim 0", [](R&, D& d) { d.head_dim = 0; });
    rotate("rotate head_dim 257", [](R&, D& d) { d.head_dim = 257; });
    rotate("rotate heads", [](R&, D& d) { d.heads = 65536; });
    rotate("rotate q_stride", [](R&, D& d) { d.q_stride = 127; });
    rotate("rotate q_out_stride", [](R&, D& d) { d.q_out_stride = 127; });
    rotate("rotate k_stride", [](R&, D& d) { d.k_stride = 63; });
    rotate("rotate k_out_stride", [](R&, D& d) { d.k_out_stride = 63; });
    rotate("rotate in place", [](R&, D& d) { d.q_stride = 200; });
    rotate("rotate tokens", [](R&, D& d) { d.tokens = 1u << 30; });
    rotate("rotate null starts", [](R&, D& d) { d.starts = nullptr; });
    say("rotate null", pimdl_rotate(ctx, &r0, nullptr));
    say("rotate null rotary", pimdl_rotate(ctx, nullptr, &d0));

    typedef pimdl_paged_cache C;
    const C c0 = {host, host, ints, ints, nullptr, 4, 16, 1, 64, 2, 4, PIMDL_F16};
    auto append = [&](const char* name, std::function<void(C&, R&)> f, uint32_t dtype = PIMDL_F32, uint32_t stride = 64, uint32_t batch = 1, uint32_t heads = 2, uint32_t q_stride = 128,
                      uint32_t q_out_stride = 128, uint32_t tokens = 4) {
        C c = c0; R r = r0; f(c, r); ctx->err.clear();
        say(name, pimdl_cache_append_rotary(ctx, &c, nullptr, ints, batch, tokens, host, host, stride, dtype, &r, nullptr, host, host, heads, q_stride, q_out_stride));
    };
    append("append host memory", [](C&, R&) {});
    append("append no tokens", [](C&, R&) {}, PIMDL_F32, 64, 1, 2, 128, 128, 0);
    append("append dims", [](C&, R& r) { r.dims = 128; });
    append("append bf16 to f16", [](C&, R&) {}, PIMDL_BF16);
    append("append stride", [](C&, R&) {}, PIMDL_F32, 63);
    append("append batch", [](C&, R&) {}, PIMDL_F32, 64, 3);
    append("append q_stride", [](C&, R&) {}, PIMDL_F32, 64, 1, 2, 127);
    append("append q_out_stride", [](C&, R&) {}, PIMDL_F32, 64, 1, 2, 128, 127);
    append("append in place", [](C&, R&) {}, PIMDL_F32, 64, 1, 2, 128, 200);
    append("append heads", [](C&, R&) {}, PIMDL_F32, 64, 1, 65536);
    append("append page_tokens", [](C& c, R&) { c.page_tokens = 24; });
    say("append null rotary", pimdl_cache_append_rotary(ctx, &c0, nullptr, ints, 1, 4, host, host, 64, 0, nullptr, nullptr, nullptr, nullptr, 0, 0, 0));

    typedef pimdl_tree T;
    const T t0 = {words, ints, 2};
    auto build = [&](const char* name, uint32_t w, uint32_t batch = 1, uint32_t tokens = 4) { ctx->err.clear(); say(name, pimdl_tree_build(ctx, ints, ints, batch, tokens, w, words, ints)); };
    build("build host memory", 2);
    build("build no words", 0);
    build("build many words", 33);
    build("build no tokens", 1, 1, 0);
    build("build no batch", 1, 0);
    build("build batch", 1, 1u << 24);
    auto attend = [&](const char* name, std::function<void(C&, T&)> f, uint32_t dtype = PIMDL_F32, uint32_t heads = 2, uint32_t batch = 1, uint32_t tokens = 4, float scale = 1.0f) {
        C c = c0; T t = t0; f(c, t); ctx->err.clear();
        say(name, pimdl_attention_tree(ctx, &c, nullptr, ints, batch, tokens, &t, host, host, heads, 128, 128, dtype, 5, 0, scale));
    };
    attend("attend host memory", [](C&, T&) {});
    attend("attend words", [](C&, T& t) { t.words = 40; });
    attend("attend no tokens", [](C&, T&) {}, PIMDL_F32, 2, 1, 0);
    attend("attend heads", [](C&, T&) {}, PIMDL_F32, 0);
    attend("attend batch", [](C&, T&) {}, PIMDL_F32, 2, 3);
    attend("attend scale", [](C&, T&) {}, PIMDL_F32, 2, 1, 4, __builtin_nanf(""));
    attend("attend type", [](C&, T&) {}, PIMDL_BF16);
    say("attend null tree", pimdl_attention_tree(ctx, &c0, nullptr, ints, 1, 4, nullptr, host, host, 2, 128, 128, 0, 5, 0, 1.0f));

    typedef pimdl_page_book B;
    void* pools[2] = {host, host};
    const B b0 = {ints, ints, ints, ints, 2, 4, 4, 16, pools, 2, 1, 2048};
    auto accept = [&](const char* name, std::function<void(B&, T&)> f, uint32_t row_bytes = 128, uint32_t batch = 1) {
        B b = b0; T t = t0; f(b, t); ctx->err.clear();
        say(name, pimdl_pages_accept(ctx, &b, nullptr, ints, batch, 4, &t, ints, row_bytes, ints));
    };
    accept("accept host memory", [](B&, T&) {});
    accept("accept no row_bytes", [](B&, T&) {}, 0);
    accept("accept row_bytes", [](B&, T&) {}, 96);
    accept("accept words", [](B&, T& t) { t.words = 0; });
    accept("accept batch", [](B&, T&) {}, 128, 3);
    accept("accept nothing", [](B& b, T&) { b.pool_count = 0; b.tables = nullptr; }, 128, 0);
    accept("accept pages", [](B& b, T&) { b.pages = 0; });
    say("accept null tree", pimdl_pages_accept(ctx, &b0, nullptr, ints, 1, 4, nullptr, ints, 128, ints));
    say("accept null book", pimdl_pages_accept(ctx, nullptr, nullptr, ints, 1, 4, &t0, ints, 128, ints));
    printf("sizes|%d|\n", (int)(sizeof(R) * 1000000 + sizeof(D) * 1000 + sizeof(T)));
    ctx->err.clear();
    printf("no context|%d|\n", pimdl_rotate(nullptr, &r0, &d0) + pimdl_tree_build(nullptr, ints, ints, 1, 1, 1, words, ints) + pimdl_pages_accept(nullptr, &b0, nullptr, ints, 1, 1, &t0, ints, 1, ints));
    return 0;
}
"""

INVALID, UNSUPPORTED = -1, -2
WANT = {
    "rotate host memory": (INVALID, "starts must be a device pointer"), "rotate nothing": (0, ""), "rotate no tokens": (0, ""), "rotate no batch": (0, ""),
    "rotate odd dims": (INVALID, "dims=33"), "rotate no dims": (INVALID, "dims=0"), "rotate many dims": (INVALID, "dims=66"), "rotate pairs": (INVALID, "pairs"),
    "rotate dtype": (INVALID, "dtype"), "rotate head_dim 0": (INVALID, "zero-sized"), "rotate head_dim 257": (UNSUPPORTED, "head_dim"), "rotate heads": (UNSUPPORTED, "heads"),
    "rotate q_stride": (INVALID, "q_stride"), "rotate q_out_stride": (INVALID, "q_out_stride"), "rotate k_stride": (INVALID, "k_stride"),
    "rotate k_out_stride": (INVALID, "k_out_stride"), "rotate in place": (INVALID, "its stride"), "rotate tokens": (UNSUPPORTED, "tokens"),
    "rotate null starts": (INVALID, "starts is null"), "rotate null": (INVALID, "null"), "rotate null rotary": (INVALID, "rotary is null"),
    "append host memory": (INVALID, "device pointer"), "append no tokens": (0, ""), "append dims": (INVALID, "dims=128"), "append bf16 to f16": (UNSUPPORTED, "own type"),
    "append stride": (INVALID, "kv_stride"), "append batch": (INVALID, "batch=3"), "append q_stride": (INVALID, "q_stride"), "append q_out_stride": (INVALID, "q_out_stride"),
    "append in place": (INVALID, "its stride"), "append heads": (UNSUPPORTED, "heads"), "append page_tokens": (UNSUPPORTED, "page_tokens=24"),
    "append null rotary": (INVALID, "rotary is null"),
    "build host memory": (INVALID, "device pointer"), "build no words": (UNSUPPORTED, "words=0"), "build many words": (UNSUPPORTED, "words=33"), "build no tokens": (0, ""),
    "build no batch": (0, ""), "build batch": (UNSUPPORTED, "batch"),
    "attend host memory": (INVALID, "device pointer"), "attend words": (UNSUPPORTED, "words=40"), "attend no tokens": (0, ""), "attend heads": (INVALID, "zero-sized"),
    "attend batch": (INVALID, "batch=3"), "attend scale": (INVALID, "scale"), "attend type": (UNSUPPORTED, "own type"), "attend null tree": (INVALID, "tree is null"),
    "accept host memory": (INVALID, "device pointer"), "accept no row_bytes": (INVALID, "no number of runs"), "accept row_bytes": (INVALID, "no number of runs"),
    "accept words": (UNSUPPORTED, "words=0"), "accept batch": (INVALID, "batch=3"), "accept nothing": (INVALID, "tables is null"), "accept pages": (UNSUPPORTED, "pages=0"),
    "accept null tree": (INVALID, "tree is null"), "accept null book": (INVALID, "book is null"), "no context": (3 * INVALID, ""),
}


def test_refusals_before_the_device_is_touched(tmp_path):
    if not os.path.exists(pimdl.LIB_PATH):
        pytest.skip("libpimdl.so not built yet (run __graft_entry__.build())")
    src, exe = tmp_path / "refusals.cpp", tmp_path / "refusals"
    src.write_text(SOURCE)
    lib = os.path.dirname(pimdl.LIB_PATH)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-w", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROOT, "include"), "-I", pimdl.CSRC, "-I", "/opt/rocm/include",
                           "-o", str(exe), str(src), pimdl.LIB_PATH, f"-Wl,-rpath,{lib}", "-L/opt/rocm/lib", "-lamdhip64", "-Wl,-rpath,/opt/rocm/lib"])
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stderr
    got = {}
    for line in out.stdout.splitlines():
        name, code, text = line.split("|", 2)
        got[name] = (int(code), text)
        if name == "sizes":  # the structures as the binding has them
            assert [int(code) // 10 ** 6, int(code) // 1000 % 1000, int(code) % 1000] == [ctypes.sizeof(t) for t in (pimdl.RotaryDesc, pimdl.RotateDesc, pimdl.TreeDesc)]
            continue
        want_code, want_text = WANT[name]
        assert int(code) == want_code and want_text in text, line
    assert set(got) - {"sizes"} == set(WANT)
