"""Expert modules without a device."""
from disagmoe_amd.models import experts


def test_names():
    from disagmoe_amd import models
    assert {"MoEExperts", "MoEExpertsSerial", "MoEExpertsFP8", "MoEExpertsW4"} <= set(models.__all__)
    assert models.MoEExpertsW4 is experts.MoEExpertsW4

