"""The benchmark command runs the quantiser, the scaled GEMM and the orthogonalisation and reports a time
and a rate for every size given."""
import pytest

from ccglib_b200 import benchmark

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("argv, columns", [
    (["quantize", "--b", "2", "--m", "200,300", "--k", "256,130", "--block_rows", "128",
      "--mem_order", "col", "--precision_out", "float8e5m2"], 4),
    (["scaled_gemm", "--m", "7,256", "--n", "300,256", "--k", "200,512", "--precision_out",
      "bfloat16"], 5),
    (["orthogonalize", "--b", "3", "--m", "20,200", "--n", "50,136", "--precision_in", "bfloat16"],
     4),
])
def test_reports_time_and_rate(argv, columns, capsys):
    assert benchmark.main(argv + ["--csv", "--benchmark_duration", "0.01"]) == 0
    lines = [x for x in capsys.readouterr().out.splitlines() if x and not x.startswith("#")]
    assert len(lines) == 2
    for line in lines:
        values = [float(v) for v in line.split(",")]
        assert len(values) == columns and values[-2] > 0 and values[-1] > 0
