"""The draft-verification operators without a GPU: what they refuse, and the index arithmetic of
the paged cache (csrc/paged.cuh, compiled here by the host compiler).

Every call below is given a null context and must be refused for the argument under test before
the context is looked at; with good arguments it gets as far as the null context.
"""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

import k3cuda

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20   # a stand-in for a device address, 256-byte aligned; never followed


def cache(**kw):
    d = dict(latent=P, rope=P, page_table=P, n_pages=10, page_size=16, max_pages=4)
    d.update(kw)
    return k3cuda.PagedCache(**d)


def batch(**kw):
    d = dict(ctx_lens=P, cu_tokens=P, B=2, T=5)
    d.update(kw)
    return k3cuda.TokenBatch(**d)


def refused(fn, code, text):
    assert fn() == code
    msg = k3cuda.lib().k3cuda_last_error().decode()
    assert text in msg, msg


BAD_TABLES = [
    (dict(n_pages=0), {}, k3cuda.ERR_ARG, "n_pages=0"),
    (dict(max_pages=0), {}, k3cuda.ERR_ARG, "max_pages=0"),
    (dict(page_size=0), {}, k3cuda.ERR_ARG, "page_size=0"),
    (dict(page_size=-16), {}, k3cuda.ERR_ARG, "page_size=-16"),
    (dict(page_size=4), {}, k3cuda.ERR_UNSUPPORTED, "page_size=4"),
    (dict(page_size=48), {}, k3cuda.ERR_UNSUPPORTED, "page_size=48"),
    (dict(n_pages=1 << 27), {}, k3cuda.ERR_ARG, "32-bit"),
    (dict(max_pages=1 << 27), {}, k3cuda.ERR_ARG, "32-bit"),
    (dict(latent=None), {}, k3cuda.ERR_ARG, "null pointer"),
    (dict(page_table=None), {}, k3cuda.ERR_ARG, "null pointer"),
    (dict(rope=P + 8), {}, k3cuda.ERR_ARG, "16-byte"),
    (dict(page_table=P + 2), {}, k3cuda.ERR_ARG, "4-byte"),
    ({}, dict(B=-1), k3cuda.ERR_ARG, "B=-1"),
    ({}, dict(T=-1), k3cuda.ERR_ARG, "T=-1"),
    ({}, dict(ctx_lens=None), k3cuda.ERR_ARG, "null pointer"),
    ({}, dict(cu_tokens=P + 1), k3cuda.ERR_ARG, "4-byte"),
]


def append(c, b, **kw):
    a = dict(ct=P, ct_stride=576, q=P, q_stride=16 * 192, q_nope=P, q_rope=P, io=k3cuda.F32, H=16,
             w=P, eps=1e-6, inv=P, pos=P, style=k3cuda.ROPE_HALF, dn=128, dr=64, dl=512)
    a.update(kw)
    return lambda: k3cuda.lib().k3cuda_mla_paged_append(
        None, C.byref(c) if c else None, C.byref(b) if b else None, a["ct"], a["ct_stride"],
        a["q"], a["q_stride"], a["q_nope"], a["q_rope"], a["io"], a["H"], a["w"], a["eps"],
        a["inv"], a["pos"], a["style"], a["dn"], a["dr"], a["dl"])


def attend(c, b, **kw):
    a = dict(out=P, dt=k3cuda.BF16, qn=P, qr=P, mask=P, uk=P, uv=P, H=16, dn=128, dr=64, dl=512,
             dv=128, scale=0.1, ws=P, nws=1 << 40)
    a.update(kw)
    return lambda: k3cuda.lib().k3cuda_mla_tree_attend(
        None, a["out"], a["dt"], a["qn"], a["qr"], C.byref(c) if c else None,
        C.byref(b) if b else None, a["mask"], a["uk"], a["uv"], a["H"], a["dn"], a["dr"], a["dl"],
        a["dv"], a["scale"], a["ws"], a["nws"])


def logprobs(**kw):
    a = dict(x=P, dt=k3cuda.F32, stride=1000, T=3, V=1000, tok=P, G=2, lp=P, ent=P, K=4, ids=P,
             tlp=P, ws=P, nws=1 << 40)
    a.update(kw)
    return lambda: k3cuda.lib().k3cuda_token_logprobs(
        None, a["x"], a["dt"], a["stride"], a["T"], a["V"], a["tok"], a["G"], a["lp"], a["ent"],
        a["K"], a["ids"], a["tlp"], a["ws"], a["nws"])


@pytest.mark.parametrize("ckw,bkw,code,text", BAD_TABLES)
def test_cache_and_batch_refusals(ckw, bkw, code, text):
    refused(append(cache(**ckw), batch(**bkw)), code, text)
    refused(attend(cache(**ckw), batch(**bkw)), code, text)


def test_null_cache_or_batch():
    for call in (append, attend):
        refused(call(None, batch()), k3cuda.ERR_ARG, "null cache or batch")
        refused(call(cache(), None), k3cuda.ERR_ARG, "null cache or batch")


@pytest.mark.parametrize("kw,code,text", [
    (dict(io=7), k3cuda.ERR_ARG, "io_dtype"), (dict(style=2), k3cuda.ERR_ARG, "rope_style"),
    (dict(dl=256), k3cuda.ERR_UNSUPPORTED, "dl=256"), (dict(dr=32), k3cuda.ERR_UNSUPPORTED, "dr=32"),
    (dict(H=129), k3cuda.ERR_ARG, "H=129"), (dict(H=-1), k3cuda.ERR_ARG, "H=-1"),
    (dict(q=None), k3cuda.ERR_ARG, "H=16"), (dict(ct=None), k3cuda.ERR_ARG, "null pointer"),
    (dict(q_rope=None), k3cuda.ERR_ARG, "null pointer"),
    (dict(ct_stride=575), k3cuda.ERR_ARG, "strides"), (dict(ct_stride=578), k3cuda.ERR_ARG, "strides"),
    (dict(ct_stride=580, io=k3cuda.BF16), k3cuda.ERR_ARG, "strides"),
    (dict(q_stride=16 * 192 - 4), k3cuda.ERR_ARG, "strides"),
    (dict(ct=P + 4), k3cuda.ERR_ARG, "16-byte"), (dict(q_nope=P + 8), k3cuda.ERR_ARG, "16-byte"),
    (dict(pos=P + 2), k3cuda.ERR_ARG, "4-byte")])
def test_append_refusals(kw, code, text):
    refused(append(cache(), batch(), **kw), code, text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dt=5), k3cuda.ERR_ARG, "out_dtype"), (dict(H=0), k3cuda.ERR_ARG, "H=0"),
    (dict(H=129), k3cuda.ERR_ARG, "H=129"), (dict(dv=64), k3cuda.ERR_UNSUPPORTED, "dv=64"),
    (dict(dn=64), k3cuda.ERR_UNSUPPORTED, "dn=64"), (dict(qn=None), k3cuda.ERR_ARG, "null pointer"),
    (dict(uk=P + 2), k3cuda.ERR_ARG, "16-byte"), (dict(out=P + 4), k3cuda.ERR_ARG, "16-byte"),
    (dict(mask=P + 4), k3cuda.ERR_ARG, "8-byte")])
def test_attend_refusals(kw, code, text):
    refused(attend(cache(), batch(), **kw), code, text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(ws=None), k3cuda.ERR_WORKSPACE, "workspace"), (dict(nws=1000), k3cuda.ERR_WORKSPACE, "workspace"),
    (dict(ws=P + 64), k3cuda.ERR_ARG, "256-byte"), (dict(scale=float("nan")), k3cuda.ERR_ARG, "scale"),
    (dict(scale=float("-inf")), k3cuda.ERR_ARG, "scale"), (dict(scale=3e38), k3cuda.ERR_ARG, "scale")])
def test_attend_refuses_its_workspace_and_scale(kw, code, text):
    refused(attend(cache(), batch(), **kw), code, text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(T=-1), k3cuda.ERR_ARG, "T=-1"), (dict(V=0), k3cuda.ERR_ARG, "V=0"),
    (dict(V=(1 << 24) + 1, stride=1 << 25), k3cuda.ERR_UNSUPPORTED, "not built"),
    (dict(K=33), k3cuda.ERR_ARG, "K=33"), (dict(K=-1), k3cuda.ERR_ARG, "K=-1"),
    (dict(dt=9), k3cuda.ERR_ARG, "io_dtype"), (dict(G=-1), k3cuda.ERR_ARG, "G=-1"),
    (dict(tok=None), k3cuda.ERR_ARG, "null output"), (dict(ids=None), k3cuda.ERR_ARG, "null output"),
    (dict(stride=999), k3cuda.ERR_ARG, "row_stride=999"), (dict(x=P + 2), k3cuda.ERR_ARG, "aligned"),
    (dict(x=None), k3cuda.ERR_ARG, "null logits"),
    (dict(ws=P + 8, V=163840, stride=163840), k3cuda.ERR_ARG, "256-byte"),
    (dict(ws=None, V=163840, stride=163840), k3cuda.ERR_WORKSPACE, "workspace"),
    (dict(nws=8, V=163840, stride=163840), k3cuda.ERR_WORKSPACE, "workspace")])
def test_logprobs_refusals(kw, code, text):
    refused(logprobs(**kw), code, text)


def test_good_arguments_reach_the_context():
    for call in (append(cache(), batch()), append(cache(), batch(), H=0, q=None),
                 append(cache(), batch(), inv=None, pos=None), attend(cache(), batch()),
                 attend(cache(), batch(), mask=None), logprobs(), logprobs(K=0, G=0, ent=None),
                 append(cache(latent=None), batch(B=0)), attend(cache(), batch(T=0)),
                 logprobs(T=0)):
        refused(call, k3cuda.ERR_ARG, "null context")


def test_workspace_queries():
    n = C.c_size_t(7)
    L = k3cuda.lib()
    k3cuda.check(L.k3cuda_token_logprobs_workspace(0, 1000, 4, C.byref(n)))
    assert n.value == 0
    refused(lambda: L.k3cuda_token_logprobs_workspace(1, 1000, 4, None), k3cuda.ERR_ARG, "null")
    refused(lambda: L.k3cuda_token_logprobs_workspace(1, 0, 4, C.byref(n)), k3cuda.ERR_ARG, "V=0")
    refused(lambda: L.k3cuda_mla_tree_attend_workspace(1, 1, 16, 512, 128, None), k3cuda.ERR_ARG,
            "null")
    refused(lambda: L.k3cuda_mla_tree_attend_workspace(1, 1, 129, 512, 128, C.byref(n)),
            k3cuda.ERR_ARG, "H=129")
    refused(lambda: L.k3cuda_mla_tree_attend_workspace(1, 1, 16, 576, 128, C.byref(n)),
            k3cuda.ERR_UNSUPPORTED, "dl=576")
    # a workspace holds for every batch of at most these sizes
    last = 0
    for B, T in ((1, 1), (1, 64), (4, 64), (64, 64), (64, 1024), (64, 4096)):
        k3cuda.check(L.k3cuda_mla_tree_attend_workspace(B, T, 128, 512, 128, C.byref(n)))
        assert n.value >= last
        last = n.value


def test_logprobs_workspace_holds_for_smaller_calls():
    n = C.c_size_t()
    for V in (1, 777, 50257, 163841, 1 << 24):
        for T in (1, 2, 300, 591, 592, 700, 5000):
            k3cuda.check(k3cuda.lib().k3cuda_token_logprobs_workspace(T, V, 20, C.byref(n)))
            for T1 in {1, 2, 3, T // 7 + 1, T // 2 + 1, T}:
                for V1 in {1, V // 9 + 1, V // 2 + 1, V}:
                    for dt in (k3cuda.F32, k3cuda.BF16):
                        if T1 <= T:
                            refused(logprobs(T=T1, V=V1, stride=V1, K=19, dt=dt, nws=n.value),
                                    k3cuda.ERR_ARG, "null context")


SRC = r"""
#include <assert.h>
#include <stdio.h>
#include <random>
#include <vector>
#include "paged.cuh"
using namespace k3;
int main() {
    std::mt19937 g(1);
    auto rnd = [&](int lo, int hi) { return (int)(lo + (long long)(g() % (unsigned)((long long)hi - lo + 1))); };
    // tables that hold anything: no index ever leaves the arrays
    for (int it = 0; it < 20000; it++) {
        const int B = rnd(1, 6), mp = rnd(1, 5), sh = rnd(3, 7), ps = 1 << sh, np = rnd(1, 9), T = rnd(0, 40);
        const bool wild = it & 1;
        std::vector<int> table(B * mp), lens(B), cu(B + 1);
        for (int &x : table) x = wild && rnd(0, 3) == 0 ? (int)g() : rnd(0, np - 1);
        for (int &x : lens) x = wild && rnd(0, 3) == 0 ? (int)g() : rnd(0, mp * ps);
        for (int i = 0; i <= B; i++) cu[i] = wild && rnd(0, 3) == 0 ? (int)g() : (i ? cu[i - 1] : 0) + rnd(0, 9);
        const PagedView v{table.data(), np, ps, mp, lens.data(), cu.data(), B, T, sh};
        for (int b = 0; b < B; b++) {
            const PagedSeq s = paged_seq(v, b, 64);
            assert(s.n >= 0 && (s.n == 0 || (s.first >= 0 && s.first + s.n <= T && s.len >= 0)));
            assert(s.n <= 64 && (s.n == 0 || s.len + s.n <= mp * ps));
            assert(!s.code || s.n == 0);
            for (int p = 0; s.n && p < s.len + s.n; p++) {
                const long long row = paged_row(v, b, p);
                assert(row >= -1 && row < (long long)np * ps);
                const int page = table[b * mp + p / ps];
                assert(row == (page < 0 || page >= np ? -1 : (long long)page * ps + p % ps));
            }
        }
        for (int t = -2; t < 50; t++) {
            const int b = last_at_most(cu.data(), B, t);
            assert(b >= 0 && b < B);
        }
    }
    // offsets past 32 bits of elements
    { int table[1] = {(1 << 27) - 1}, len[1] = {5}, cu[2] = {0, 1};
      const PagedView v{table, 1 << 27, 8, 1, len, cu, 1, 1, 3};
      assert(paged_row(v, 0, 7) == (1ll << 30) - 1); }
    // the work line: every place lies in the cluster that line_cluster names
    for (int it = 0; it < 3000; it++) {
        const long long total = it < 1500 ? rnd(1, 500) : 1 + (long long)g() * 1000;
        const int G = (int)std::min<long long>(total, rnd(1, 148));
        assert(line_begin(total, G, 0) == 0 && line_begin(total, G, G) == total);
        for (int c = 0; c < G; c++) {
            const long long a = line_begin(total, G, c), e = line_begin(total, G, c + 1);
            assert(a < e && line_cluster(total, G, a) == c && line_cluster(total, G, e - 1) == c);
        }
    }
    // the bits of a tile against their definition
    for (int it = 0; it < 3000; it++) {
        const int n = rnd(0, 64), len = rnd(0, 300);
        const uint64_t mask = ((uint64_t)g() << 32) | g();
        for (int p0 = 0; p0 < 450; p0 += rnd(1, 64)) {
            const uint64_t w = tree_bits(mask, len, n, p0);
            for (int c = 0; c < 64; c++) {
                const int j = p0 + c - len;
                const bool see = j < 0 || (j < n && ((mask >> j) & 1));
                assert(((w >> c) & 1) == (see ? 1u : 0u));
            }
        }
    }
    puts("ok");
    return 0;
}
"""


@pytest.mark.skipif(not shutil.which("g++"), reason="no host C++ compiler")
def test_paged_index_arithmetic(tmp_path):
    src = tmp_path / "paged.cpp"
    src.write_text(SRC)
    exe = tmp_path / "paged"
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=address,undefined",
                        "-I" + os.path.join(ROOT, "kimi-k3-in-c_b200", "csrc"), str(src), "-o",
                        str(exe)], capture_output=True, text=True)
    if "asan" in r.stderr or "ubsan" in r.stderr:   # sanitizer libraries missing
        r = subprocess.run(["g++", "-std=c++17", "-O1", "-I" + os.path.join(
            ROOT, "kimi-k3-in-c_b200", "csrc"), str(src), "-o", str(exe)], capture_output=True,
            text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stderr


def test_struct_layout_matches_the_header(tmp_path):
    """PagedCache and TokenBatch against include/k3cuda.h, field by field."""
    if not shutil.which("gcc"):
        pytest.skip("no host C compiler")
    fields = {"k3cuda_paged_cache": k3cuda.PagedCache, "k3cuda_token_batch": k3cuda.TokenBatch}
    lines = ["#include <stddef.h>", '#include "k3cuda.h"']
    for name, cls in fields.items():
        lines.append(f'_Static_assert(sizeof({name}) == {C.sizeof(cls)}, "{name}");')
        for f, _ in cls._fields_:
            off = getattr(cls, f).offset
            lines.append(f'_Static_assert(offsetof({name}, {f}) == {off}, "{name}.{f}");')
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines) + "\n")
    r = subprocess.run(["gcc", "-std=gnu99", "-fsyntax-only", "-I" + os.path.join(ROOT, "include"),
                        str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert np.dtype(np.int32).itemsize == C.sizeof(C.c_int)


ORDER_SRC = r"""
#include <assert.h>
#include <stdio.h>
#include <random>
#include <vector>
#include "paged.cuh"
using namespace k3;
int main() {
    std::mt19937 g(2);
    auto rnd = [&](int lo, int hi) { return lo + (int)(g() % (unsigned)(hi - lo + 1)); };
    int none = 0, all = 0;
    for (int it = 0; it < 50000; it++) {
        const int B = rnd(1, 7), T = rnd(0, 30);
        std::vector<int> table(B, 0), lens(B, 0), cu(B + 1);
        for (int i = 0; i <= B; i++) {
            cu[i] = (i ? cu[i - 1] : rnd(0, 2)) + rnd(0, 6);
            if (it % 2 && rnd(0, 4) == 0) cu[i] = rnd(0, 1) ? (int)g() : rnd(-3, 35);
        }
        const PagedView v{table.data(), 1, 64, 1, lens.data(), cu.data(), B, T, 6};
        int n = 0;
        while (n < B && paged_in_order(v, n)) n++;
        // those that count: no code of the offsets, within the rows, each row in one at most
        std::vector<int> owner(T, -1);
        for (int b = 0; b < n; b++) {
            const PagedSeq s = paged_seq(v, b, 1 << 20);
            assert(s.code == PAGED_OK && s.n == cu[b + 1] - cu[b]);
            for (int i = 0; i < s.n; i++) {
                assert(owner.at(s.first + i) < 0);
                owner[s.first + i] = b;
            }
        }
        if (n < B) assert(paged_seq(v, n, 1 << 20).code == PAGED_OFFSETS);
        none += n == 0;
        all += n == B;
    }
    assert(none > 1000 && all > 1000);
    puts("ok");
    return 0;
}
"""


@pytest.mark.skipif(not shutil.which("g++"), reason="no host C++ compiler")
def test_sequences_in_order_share_no_row(tmp_path):
    src, exe = tmp_path / "order.cpp", tmp_path / "order"
    src.write_text(ORDER_SRC)
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-D_GLIBCXX_ASSERTIONS",
                        "-I" + os.path.join(ROOT, "kimi-k3-in-c_b200", "csrc"), str(src), "-o",
                        str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stderr


def test_attend_takes_no_more_tokens_than_its_grids():
    n = C.c_size_t()
    for T, ok in ((65535 * 128, True), (65535 * 128 + 1, False), (1 << 23, False)):
        q = lambda: k3cuda.lib().k3cuda_mla_tree_attend_workspace(  # noqa: E731
            1, T, 1, 512, 128, C.byref(n))
        if ok:
            k3cuda.check(q())
        else:
            refused(q, k3cuda.ERR_ARG, f"T={T}")
        refused(attend(cache(), batch(T=T), H=1), k3cuda.ERR_ARG,
                "null context" if ok else f"T={T}")
