"""A wait inside group norm that runs out is reported, whichever thread gave up, and the context stays usable."""
import pytest

pytestmark = pytest.mark.gpu


def test_a_wait_of_another_thread_than_the_first_is_reported(dev):
    from vtl_b200 import capi
    assert dev.check_status() == 0
    dev.wait_probe(2_000_000, arrive=2)  # one thread waits two milliseconds for nothing; the first one does not wait at all
    with pytest.raises(capi.VtlbError, match="group norm") as e:
        dev.check_status()
    assert e.value.code == capi.ETIMEOUT
    assert dev.check_status() == 0
    dev.wait_probe(2_000_000, arrive=True)
    assert dev.check_status() == 0
