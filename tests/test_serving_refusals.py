"""What the entry points of windowed attention, the paged cache and its pages refuse, without a GPU: every check comes before the first use of the
device, so a context that was never initialised is enough.  Addresses of host memory stand for whatever is not device memory."""
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
    static int32_t ints[64];
    typedef pimdl_attention_window_desc W;
    const W w0 = {host, host, host, host, ints, 1, 4, 2, 1, 64, 128, 64, 128, 1, 1, 0, PIMDL_F32, 1.0f};
    auto window = [&](const char* name, std::function<void(W&)> f) { W w = w0; f(w); ctx->err.clear(); say(name, pimdl_attention_window(ctx, &w)); };
    window("window host memory", [](W&) {});
    window("window empty", [](W& w) { w.tokens = 0; });
    window("window no batch", [](W& w) { w.batch = 0; w.starts = nullptr; });
    window("window null starts", [](W& w) { w.starts = nullptr; });
    window("window dtype", [](W& w) { w.dtype = 3; });
    window("window heads", [](W& w) { w.heads = 3; w.kv_heads = 2; w.q_stride = w.out_stride = 192; w.kv_stride = 128; });
    window("window no heads", [](W& w) { w.heads = 0; });
    window("window no kv heads", [](W& w) { w.kv_heads = 0; });
    window("window head_dim 0", [](W& w) { w.head_dim = 0; });
    window("window head_dim 257", [](W& w) { w.head_dim = 257; w.q_stride = w.out_stride = w.kv_stride = 1024; });
    window("window q_stride", [](W& w) { w.q_stride = 127; });
    window("window out_stride", [](W& w) { w.out_stride = 127; });
    window("window kv_stride", [](W& w) { w.kv_stride = 63; });
    window("window scale inf", [](W& w) { w.scale = __builtin_inff(); });
    window("window scale nan", [](W& w) { w.scale = __builtin_nanf(""); });
    window("window tokens", [](W& w) { w.tokens = 1u << 30; });
    window("window odd starts", [](W& w) { w.starts = reinterpret_cast<const int32_t*>(reinterpret_cast<const char*>(ints) + 2); });
    say("window null", pimdl_attention_window(ctx, nullptr));

    typedef pimdl_paged_cache C;
    const C c0 = {host, host, ints, ints, nullptr, 4, 16, 1, 64, 2, 4, PIMDL_F16};
    auto paged = [&](const char* name, std::function<void(C&)> f, uint32_t dtype = PIMDL_F32, uint32_t heads = 2, uint32_t batch = 1, uint32_t tokens = 1, float scale = 1.0f, uint32_t stride = 128) {
        C c = c0; f(c); ctx->err.clear();
        say(name, pimdl_attention_paged(ctx, &c, nullptr, ints, batch, tokens, host, host, heads, stride, stride, dtype, 5, 0, scale));
    };
    auto append = [&](const char* name, std::function<void(C&)> f, uint32_t dtype = PIMDL_F32, uint32_t stride = 64, uint32_t batch = 1) {
        C c = c0; f(c); ctx->err.clear();
        say(name, pimdl_cache_append(ctx, &c, nullptr, ints, batch, 1, host, host, stride, dtype));
    };
    paged("paged host memory", [](C&) {});
    paged("paged null k", [](C& c) { c.k = nullptr; });
    paged("paged null tables", [](C& c) { c.tables = nullptr; });
    paged("paged odd k", [](C& c) { c.k = host + 1; });
    paged("paged bf16 over f16", [](C&) {}, PIMDL_BF16);
    paged("paged f16 over f32", [](C& c) { c.dtype = PIMDL_F32; }, PIMDL_F16);
    paged("paged cache dtype", [](C& c) { c.dtype = 9; });
    paged("paged page_tokens 8", [](C& c) { c.page_tokens = 8; });
    paged("paged page_tokens 24", [](C& c) { c.page_tokens = 24; });
    paged("paged page_tokens 2048", [](C& c) { c.page_tokens = 2048; });
    paged("paged no pages", [](C& c) { c.pages = 0; });
    paged("paged no seqs", [](C& c) { c.seqs = 0; });
    paged("paged no table", [](C& c) { c.table_width = 0; });
    paged("paged too long", [](C& c) { c.table_width = 1u << 27; });
    paged("paged heads", [](C&) {}, PIMDL_F32, 0);
    paged("paged batch", [](C&) {}, PIMDL_F32, 2, 3);
    paged("paged no tokens", [](C&) {}, PIMDL_F32, 2, 1, 0);
    paged("paged scale", [](C&) {}, PIMDL_F32, 2, 1, 1, -__builtin_inff());
    paged("paged stride", [](C&) {}, PIMDL_F32, 2, 1, 1, 1.0f, 127);
    append("append batch", [](C&) {}, PIMDL_F32, 64, 3);
    paged("paged head_dim", [](C& c) { c.head_dim = 300; });
    say("paged null", pimdl_attention_paged(ctx, nullptr, nullptr, ints, 1, 1, host, host, 2, 128, 128, 0, 0, 0, 1.0f));
    append("append host memory", [](C&) {});
    append("append stride", [](C&) {}, PIMDL_F32, 63);
    append("append bf16 to f16", [](C&) {}, PIMDL_BF16);

    typedef pimdl_page_book B;
    void* pools[2] = {host, host};
    const B b0 = {ints, ints, ints, ints, 2, 4, 4, 16, pools, 2, 1, 2048};
    auto book = [&](const char* name, std::function<void(B&)> f, int op = 1, uint32_t n = 1) {
        B b = b0; f(b); ctx->err.clear();
        say(name, op == 0 ? pimdl_pages_reserve(ctx, &b, ints, ints, n) : op == 1 ? pimdl_pages_fork(ctx, &b, ints, ints, n) : op == 2 ? pimdl_pages_free(ctx, &b, ints, n)
                  : op == 3 ? pimdl_pages_compact(ctx, &b) : pimdl_pages_copy(ctx, &b, ints, ints, n));
    };
    for (int op = 0; op < 5; ++op) book("book host memory", [](B&) {}, op);
    book("book no pages", [](B& b) { b.pages = 0; });
    book("book many pages", [](B& b) { b.pages = (1u << 24) + 1; }, 4);
    book("book no seqs", [](B& b) { b.seqs = 0; }, 0);
    book("book many seqs", [](B& b) { b.seqs = 16385; }, 2);
    book("book page_tokens", [](B& b) { b.page_tokens = 0; }, 3);
    book("book long rows", [](B& b) { b.table_width = 1u << 28; }, 0);
    book("book pools", [](B& b) { b.pools = nullptr; b.tables = nullptr; }, 4);
    book("book pool_count", [](B& b) { b.pool_count = 65; }, 4);
    book("book page_bytes", [](B& b) { b.page_bytes = 24; }, 4);
    book("book no page_bytes", [](B& b) { b.page_bytes = 0; }, 4);
    book("book copy nothing", [](B& b) { b.pool_count = 0; }, 4, 0);
    say("book null", pimdl_pages_free(ctx, nullptr, ints, 1));
    printf("sizes|%d|\n", (int)(sizeof(W) * 1000000 + sizeof(C) * 1000 + sizeof(B)));
    ctx->err.clear();
    printf("no context|%d|\n", pimdl_attention_window(nullptr, &w0));
    return 0;
}
"""

INVALID, UNSUPPORTED = -1, -2
WANT = {
    "window host memory": (INVALID, "starts must be a device pointer"), "window empty": (0, ""), "window no batch": (0, ""), "window null starts": (INVALID, "starts is null"),
    "window dtype": (INVALID, "dtype"), "window heads": (INVALID, "multiple of kv_heads"), "window no heads": (INVALID, "zero-sized"), "window no kv heads": (INVALID, "zero-sized"),
    "window head_dim 0": (INVALID, "zero-sized"), "window head_dim 257": (UNSUPPORTED, "head_dim=257"), "window q_stride": (INVALID, "q_stride"),
    "window out_stride": (INVALID, "out_stride"), "window kv_stride": (INVALID, "kv_stride"), "window scale inf": (INVALID, "scale"), "window scale nan": (INVALID, "scale"),
    "window tokens": (UNSUPPORTED, "tokens"), "window odd starts": (INVALID, "aligned"), "window null": (INVALID, "null"),
    "paged host memory": (INVALID, "cache k must be a device pointer"), "paged null k": (INVALID, "cache k is null"), "paged null tables": (INVALID, "device pointer"),
    "paged odd k": (INVALID, "aligned to 16"), "paged bf16 over f16": (UNSUPPORTED, "own type"), "paged f16 over f32": (UNSUPPORTED, "own type"),
    "paged cache dtype": (INVALID, "dtype"), "paged page_tokens 8": (UNSUPPORTED, "page_tokens=8"), "paged page_tokens 24": (UNSUPPORTED, "page_tokens=24"),
    "paged page_tokens 2048": (UNSUPPORTED, "page_tokens=2048"), "paged no pages": (INVALID, "zero-sized"), "paged no seqs": (INVALID, "zero-sized"),
    "paged no table": (INVALID, "zero-sized"), "paged too long": (UNSUPPORTED, "2^31"), "paged head_dim": (UNSUPPORTED, "head_dim"), "paged null": (INVALID, "cache is null"),
    "paged heads": (INVALID, "zero-sized"), "paged batch": (INVALID, "batch=3"), "paged no tokens": (0, ""), "paged scale": (INVALID, "scale"),
    "paged stride": (INVALID, "q_stride"), "append batch": (INVALID, "batch=3"),
    "append host memory": (INVALID, "device pointer"), "append stride": (INVALID, "kv_stride") , "append bf16 to f16": (UNSUPPORTED, "own type"),
    "book host memory": (INVALID, "device pointer"), "book no pages": (UNSUPPORTED, "pages=0"), "book many pages": (UNSUPPORTED, "pages="), "book no seqs": (UNSUPPORTED, "seqs=0"),
    "book many seqs": (UNSUPPORTED, "seqs=16385"), "book page_tokens": (INVALID, "page_tokens"), "book long rows": (UNSUPPORTED, "2^31"), "book pools": (INVALID, "pools is null"),
    "book pool_count": (UNSUPPORTED, "pool_count=65"), "book page_bytes": (INVALID, "page_bytes"), "book no page_bytes": (INVALID, "page_bytes"), "book copy nothing": (0, ""),
    "book null": (INVALID, "book is null"), "no context": (INVALID, ""),
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
            assert [int(code) // 10 ** 6, int(code) // 1000 % 1000, int(code) % 1000] == [ctypes.sizeof(t) for t in (pimdl.AttentionWindowDesc, pimdl.PagedCacheDesc, pimdl.PageBook)]
            continue
        want_code, want_text = WANT[name]
        assert int(code) == want_code and want_text in text, line
    assert set(got) - {"sizes"} == set(WANT)
