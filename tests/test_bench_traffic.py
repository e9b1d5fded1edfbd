"""The committed counter summary that bench.py reports its traffic from was taken of the decode kernels as they stand."""

from test_bench_contract import _bench


def test_the_summary_is_of_these_sources():
    bench = _bench()
    traffic, source = bench.pmc_traffic("paged_decode_bf16_qwen3_0.6b_b64", bench.DECODE_SOURCES)
    assert traffic is not None, source
    assert 545366876 <= traffic < 1.05 * 545366876  # the algorithmic bytes of the workload
