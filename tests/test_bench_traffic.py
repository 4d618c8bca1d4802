"""bench.py reports measured HBM traffic only for kernels whose sources are those that the counters were read for."""
import bench


def test_the_measured_traffic_is_of_these_sources():
    assert bench.source_fingerprints() == bench.TRAFFIC_FAMILY_FINGERPRINT
