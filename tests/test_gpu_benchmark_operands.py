"""The benchmark command multiplies noise with scales of its own, not constants."""
import pytest

from ccglib_b200 import benchmark, capi

pytestmark = pytest.mark.gpu


def test_scaled_gemm_operands(monkeypatch, capsys):
    import torch

    seen = []

    class Plan(capi.ScaledGemmPlan):
        def run(self, d_a, d_a_scale, d_b, d_b_scale, d_c, stream=0):
            super().run(d_a, d_a_scale, d_b, d_b_scale, d_c, stream)
            seen.append((self.desc, d_a, d_a_scale, d_c))

    created = []
    empty = torch.empty

    def remember(*args, **kw):
        created.append(empty(*args, **kw))
        return created[-1]

    monkeypatch.setattr(capi, "ScaledGemmPlan", Plan)
    monkeypatch.setattr(torch, "empty", remember)
    assert benchmark.main(["scaled_gemm", "--m", "200", "--n", "130", "--k", "500", "--csv",
                           "--benchmark_duration", "0.005"]) == 0
    capsys.readouterr()
    by_address = {t.data_ptr(): t for t in created}
    _, d_a, d_a_scale, d_c = seen[-1]
    assert len(torch.unique(by_address[d_a])) > 100
    assert len(torch.unique(by_address[d_a_scale])) > 100
    c = by_address[d_c].view(torch.float32)
    assert torch.isfinite(c).all() and len(torch.unique(c)) > 1000
