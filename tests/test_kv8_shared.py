"""What a cache says of pages in common: refusals that need no GPU."""
import q4hip


def test_no_cache():
    assert q4hip.lib().q4hip_kv8_shared(None, None, None, None) == q4hip.EINVAL
