"""Sizes that group norm does not count are refused before anything is launched."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("C", [2**31 - 1, 2**31 - 1023])
def test_more_channels_than_are_counted(dev, C):
    from vtl_b200.capi import EINVAL, VtlbError
    d, o = dev.to_device(np.ones(256, np.float32)), dev.zeros(256)
    launches = dev.launch_count()
    with pytest.raises(VtlbError, match="channels go to 2147482624") as e:
        dev.groupnorm_fwd_f32(d, 1, 1, C, 1, None, None, 1e-5, 0, o, o, o)
    assert e.value.code == EINVAL
    with pytest.raises(VtlbError, match="channels go to 2147482624"):
        dev.groupnorm_bwd_f32(d, d, 1, 2, C, 1, None, None, d, d, 0, o)
    assert dev.launch_count() == launches and (o.numpy() == 0).all()
    d.free(); o.free()
