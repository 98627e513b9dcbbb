"""Token tables: what is refused before any CUDA call, and that nothing falls back to the CPU."""
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch


def test_c_entry_points_refuse_before_any_cuda_call():
    # the last error belongs to a thread: a thread of its own leaves this one's as it was
    ThreadPoolExecutor(1).submit(_refusals).result()


def _refusals():
    from fbgemm_ascend_b200 import cabi
    lib = cabi.lib()
    FP32, INT8 = 0, 2
    one = 16      # an address that is never followed: every call below is refused first
    emb = lambda **k: lib.tbe_b200_token_embedding(one, k.get("wt", FP32), k.get("V", 4), k.get("D", 8), k.get("ws", 8), k.get("tok", one),
                                                   k.get("bits", 64), k.get("n", 2), 1.0, k.get("out", one), FP32, k.get("os", 8), None, None)
    assert emb(wt=INT8) == -2 and "element types" in cabi.last_error()
    assert emb(bits=16) == -1 and "token_bits" in cabi.last_error()
    assert emb(n=-1) == -1 and emb(ws=7) == -1 and emb(os=7) == -1
    assert emb(tok=None) == -1 and "NULL" in cabi.last_error()
    assert emb(out=None) == -1
    assert emb(n=0) == 0 and emb(D=0) == 0

    need = lib.tbe_b200_token_embedding_grad_scratch_bytes
    assert need(0, 4, 8) == 0 and need(100, 4, 8) == 0 and need(5000, 4, 8) > 0      # few tokens need none
    assert need(1 << 31, 4, 8) == -1 and need(4, 1 << 31, 8) == -1 and need(4, 0, 8) == -1 and need(4, 4, 0) == -1 and need(-1, 4, 8) == -1
    grad = lambda **k: lib.tbe_b200_token_embedding_grad(k.get("g", one), k.get("gt", FP32), k.get("gs", 8), one, k.get("bits", 64), k.get("n", 5000),
                                                         k.get("V", 4), k.get("D", 8), 1.0, k.get("pad", -1), 0, k.get("out", one), FP32,
                                                         k.get("os", 8), k.get("scratch", one), k.get("bytes", 1 << 30), None)
    assert grad(gt=INT8) == -2
    assert grad(bits=8) == -1 and grad(V=0) == -1 and grad(D=0) == -1 and grad(n=1 << 31) == -1
    assert grad(pad=4) == -1 and "padding_idx" in cabi.last_error()
    assert grad(pad=-2) == -1
    assert grad(os=7) == -1 and grad(gs=-1) == -1
    assert grad(g=None) == -1 and grad(out=None) == -1 and grad(scratch=None) == -1
    assert grad(bytes=need(5000, 4, 8) - 1) == -1 and "scratch" in cabi.last_error()
    assert grad(scratch=8) == -1

    q = lambda **k: lib.tbe_b200_quantize_to_group_rows(k.get("x", one), k.get("it", FP32), 8, k.get("E", 2), k.get("D", 8), k.get("g", 32),
                                                        k.get("rb", 16), k.get("rows", one), None)
    assert q(g=48) == -2 and "group_size" in cabi.last_error()
    assert q(it=INT8) == -2 and q(D=12) == -1 and "multiple of 8" in cabi.last_error()
    assert q(rb=24) == -1 and q(rb=0) == -1 and q(D=64, rb=16) == -1 and "row_bytes" in cabi.last_error()
    assert q(rows=8) == -1 and "aligned" in cabi.last_error()
    assert q(x=None) == -1 and q(E=-1) == -1 and q(E=0) == 0

    look = lambda **k: lib.tbe_b200_group_row_embedding(k.get("rows", one), k.get("V", 4), 16, 8, 32, k.get("tok", one), k.get("bits", 64),
                                                        k.get("n", 2), 1.0, k.get("out", one), k.get("ot", FP32), k.get("os", 8), None, None)
    assert look(ot=INT8) == -2 and look(bits=0) == -1 and look(os=7) == -1 and look(n=-1) == -1 and look(out=None) == -1
    assert look(tok=None, n=5) == -1 and "rows wanted" in cabi.last_error()
    assert look(n=0) == 0

    lin = lambda **k: lib.tbe_b200_group_row_linear(k.get("x", one), k.get("it", FP32), k.get("xs", 8), k.get("m", 1), k.get("rows", one), 4, 16,
                                                    k.get("D", 8), 32, k.get("bias"), k.get("bt", FP32), k.get("out", one), FP32, k.get("os", 4), None,
                                                    k.get("scratch", one), k.get("bytes", 1 << 30), None)
    assert lin(it=INT8) == -2 and lin(bias=one, bt=INT8) == -2 and lin(os=3) == -1 and lin(xs=4) == -1 and lin(D=0) == -1 and lin(m=-1) == -1
    assert lin(x=None) == -1 and lin(out=None) == -1
    assert lin(x=8) == -1 and "aligned" in cabi.last_error()
    assert lin(m=2, xs=9) == -1 and lin(m=0) == 0
    need = lib.tbe_b200_group_row_linear_scratch_bytes
    assert need(1, 8, 32, FP32) == 0 and need(17, 8, 32, FP32) > 0 and need(16, 8192, 32, FP32) > 0      # few vectors need none
    assert need(-1, 8, 32, FP32) == -1 and need(1, 0, 32, FP32) == -1 and need(1, 8, 48, FP32) == -1 and need(1, 8, 32, INT8) == -1
    assert lin(m=17, scratch=None) == -1 and lin(m=17, scratch=8) == -1 and lin(m=17, bytes=need(17, 8, 32, FP32) - 1) == -1 and "scratch" in cabi.last_error()


def test_c_entry_point_of_bounded_products_refuses():
    ThreadPoolExecutor(1).submit(_bounded_refusals).result()


def _bounded_refusals():
    from fbgemm_ascend_b200 import cabi
    lib = cabi.lib()
    call = lambda m, polls: lib.tbe_b200_group_row_linear_bounded(16, 0, 8, m, 16, 4, 16, 8, 32, None, 0, 16, 0, 4, None, 16, 1 << 30, polls, None)
    assert call(1, -1) == -1 and "max_polls" in cabi.last_error()
    assert call(0, 0) == 0 and call(0, 1 << 40) == 0


def test_no_cpu_path():
    import fbgemm_ascend_b200 as fa
    ops = torch.ops.tbe_b200
    w, t, r = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64), torch.zeros(4, 16, dtype=torch.uint8)
    for call in (lambda: ops.token_embedding(w, t), lambda: ops.token_embedding_grad(torch.zeros(3, 8), t, 4),
                 lambda: ops.token_embedding_grad_(w, torch.zeros(3, 8), t), lambda: ops.quantize_to_group_rows(w, 32),
                 lambda: ops.group_rows_to_float(r, 8, 32), lambda: ops.group_row_embedding(r, t, 8, 32), lambda: ops.group_row_linear(w, r, 32)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
    for make in (lambda: fa.TokenEmbedding(4, 8, device="cpu"), lambda: fa.GroupRowTable(4, 8, device="cpu")):
        with pytest.raises(RuntimeError):
            make()


def test_group_row_bytes():
    from fbgemm_ascend_b200.types import group_row_bytes
    assert [group_row_bytes(d, g) for d, g in ((8, 32), (32, 32), (64, 32), (4096, 128), (5000, 32), (1000, 256))] == [16, 32, 48, 2176, 3136, 528]


_PLAN = """
#include "tbe_token_plan.h"
#include <stdio.h>
int main() {
    long long n, bytes; int fits, sms, cluster;
    while (scanf("%lld %d %lld %d %d", &n, &fits, &bytes, &sms, &cluster) == 5)
        printf("%d %lld\\n", static_cast<int>(tbe::sort_form(n, fits)), static_cast<long long>(tbe::clearing_blocks(bytes, sms, cluster)));
}
"""


def test_plan_of_a_gradient_on_few_multiprocessors(tmp_path):
    """Blocks that clear beside a sort come in whole clusters and never crowd one out; where none has room, the count says so."""
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fbgemm_ascend_b200", "csrc")
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(_PLAN)
    subprocess.run(["g++", "-std=c++17", "-I" + csrc, str(src), "-o", str(exe)], check=True)

    def ask(rows):
        r = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, q)) for q in rows), capture_output=True, text=True, check=True)
        return [tuple(map(int, line.split())) for line in r.stdout.splitlines()]

    BLOCK, CLUSTER, TILES = 0, 1, 2
    forms = [(1, 1, BLOCK), (2048, 0, BLOCK), (2049, 1, CLUSTER), (2049, 0, TILES), (262_144, 1, CLUSTER), (262_144, 0, TILES), (262_145, 1, TILES)]
    assert [f for f, _ in ask([(n, fits, 0, 148, 16) for n, fits, _ in forms])] == [f for _, _, f in forms]
    asked = [(5000, 1, b, sms, c) for b in (0, 1, 65_536, 65_537, 10 << 20, 1 << 40) for sms in (1, 2, 15, 16, 17, 31, 32, 33, 47, 64, 132, 147, 148, 160) for c in (1, 16)]
    for (_, _, b, sms, c), (_, got) in zip(asked, ask(asked)):
        assert got % c == 0 and got >= 0 and (got == 0 or got + c <= sms), (b, sms, c, got)
        assert (got > 0) == (b > 0 and sms >= 2 * c), (b, sms, c, got)
        assert got * 65_536 < b + c * 65_536, (b, sms, c, got)
    assert [g for _, g in ask([(5000, 1, 1 << 30, sms, 16) for sms in (16, 17, 31, 32, 148)])] == [0, 0, 0, 16, 128]
