"""D's choice of norm, on the CPU."""


def test_a_discriminator_without_the_choice_is_the_reference_network():
    """A module pickled whole before D took `norm` has no such attribute: it has BatchNorms, and is planned with them."""
    import models.dehaze1113 as net
    old = net.D(9, 36)
    del old.__dict__["norm"]
    assert old.norm == "batch"
    assert net.D(9, 36, norm="layer").norm == "layer" and net.D(9, 36).norm == "batch"
