"""A split contraction's sums cross CTAs: every wait and arrival that orders them must be at
cluster scope (a barrier completed by another CTA and waited on at the default CTA scope
does not order that CTA's writes). No run can show a scope to be missing; the source does."""
from __future__ import annotations

import os
import re

import numpy as np
import pytest

import grouped_check as gc
from conftest import ROOT

CSRC = os.path.join(ROOT, "wgblas_b200", "csrc")


def source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def test_parts_are_joined_at_cluster_scope():
    text = source("grouped_common.cuh")
    body = text[text.index("bool join_parts("):]
    body = body[:body.index("\n}\n")]
    waits = re.findall(r"(mbar_wait\w*)\(x\.(full|empty)", body)
    assert sorted(b for _, b in waits) == ["empty", "full"]
    assert all(w == "mbar_wait_bounded_cluster" for w, _ in waits), waits
    arrivals = re.findall(r"mbarrier\.arrive[.\w:]*|mbar_arrive_cluster", body)
    assert arrivals == ["mbar_arrive_cluster"], arrivals


def test_a_pairs_accumulators_change_hands_at_cluster_scope():
    """TMEM reads are done when tcgen05.wait::ld returns and are ordered by the tcgen05 fences: the
    arrival releases no memory, but it and the wait must reach the other CTA."""
    text = source("grouped_common.cuh")
    arrive = text[text.index("void leader_arrive("):]
    assert "mbarrier.arrive.relaxed.cluster.shared::cluster.b64" in arrive[:arrive.index("\n}\n")]
    wait = text[text.index("bool leader_wait("):]
    assert "if constexpr (CG == 2) return wgtc::mbar_wait_bounded_cluster(" in wait[:wait.index("\n}\n")]
    for name in ("grouped.cu", "mx.cu"):
        waits = re.findall(r"(\w+(?:<CG>)?)\(&acc_empty\[b\], ", source(name))
        assert [w for w in waits if w != "mbar_init"] == ["leader_wait<CG>"], (name, waits)
        assert source(name).count("leader_arrive<CG>(&acc_empty[b])") == 1


def test_the_helpers_name_the_scope():
    text = source("tcgen05.cuh")
    assert "mbarrier.arrive.release.cluster.shared::cluster.b64" in text
    assert "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64" in text


@pytest.mark.gpu
@pytest.mark.parametrize("groups", [40, 160, 400], ids=lambda g: f"{g}groups")
@pytest.mark.parametrize("form", ["rows", "inner"])
def test_many_joins_in_a_row(wg, groups, form):
    """Split contractions of more tiles than there are clusters: a CTA's place for the others' sums is
    written again and again. Repeats give the same bits (parts are added in their order)."""
    torch = pytest.importorskip("torch")
    dev = wg.init()
    dev.set_stream(0)
    try:
        g = torch.Generator(device="cuda").manual_seed(groups)
        ends = torch.arange(groups + 1, dtype=torch.int32, device="cuda")
        if form == "rows":
            m, n, k = groups, 130, 2048
            a, w = (torch.randn(s, generator=g, device="cuda").bfloat16() for s in ((m, k), (groups, n, k)))
            c = torch.empty((m, n), device="cuda")

            def call():
                wg.gemmGrouped(dev, "transpose", groups, m, n, k, 1.0, a, k, w, k, n * k, ends, 0.0, c, n)

            want, mag = (torch.einsum("rk,rnk->rn", f(a.double()), f(w.double())) for f in (lambda x: x, torch.abs))
        else:
            m, n, k = 33, 130, 1000 * groups
            ends *= 1000
            a, w = (torch.randn((k, s), generator=g, device="cuda").bfloat16() for s in (m, n))
            c = torch.empty((groups, m, n), device="cuda")

            def call():
                wg.gemmGroupedInner(dev, groups, m, n, k, 1.0, a, m, w, n, ends, 0.0, c, n, m * n)

            a3, w3 = a.view(groups, 1000, m).double(), w.view(groups, 1000, n).double()
            want, mag = (f(a3).transpose(1, 2) @ f(w3) for f in (lambda x: x, torch.abs))
        call()
        dev.check()
        first = c.clone()
        gc.assert_close(first.double().cpu().numpy(), want.cpu().numpy(), mag.cpu().numpy(), 2048, 0.0, np.zeros(1),
                        "float32", form)
        for _ in range(50):
            c.fill_(float("nan"))
            call()
            assert torch.equal(c, first)
        dev.check()
    finally:
        dev.set_stream(None)
