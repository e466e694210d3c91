"""The residual norm's tensor types, without a GPU: one that is not served is refused by the
library, by its argument's name."""
import pytest
import torch

import busfill as bf
from test_layer_ops_abi import FAKE

OTHER = [torch.bfloat16, torch.float64, torch.int32]


@pytest.mark.parametrize("dtype", OTHER)
@pytest.mark.parametrize("name,needle", [("X", "xtype"), ("delta", "dtype"), ("weight", "wtype")])
def test_other_types_are_refused(dtype, name, needle):
    t = dict(X=torch.zeros(1, 64), delta=torch.zeros(1, 64), weight=torch.zeros(64))
    t[name] = t[name].to(dtype)
    x = t.pop("X")
    with pytest.raises(bf.BusfillInvalid, match=f"unknown {needle} -1"):
        bf.rms_norm(x, 1, 64, H=FAKE, stream=0, **t)


def test_an_address_needs_its_type():
    with pytest.raises(bf.BusfillInvalid, match="unknown xtype -1"):
        bf.rms_norm(FAKE, 1, 64, H=FAKE, stream=0)
    with pytest.raises(bf.BusfillInvalid, match="unknown dtype -1"):
        bf.rms_norm(FAKE, 1, 64, H=FAKE, delta=FAKE, xtype=bf.F32, stream=0)
