"""More calls that the row operators refuse on the host, before anything touches a device (the addresses here are never
dereferenced), and what they no longer refuse."""
from test_row_operators_args import B_, C_, D, E, F, adamw, probs, probs_back, refused


def test_log_probs_refuse_inputs_off_their_elements():
    refused(probs(target=B_ + 2), "target is not aligned")
    refused(probs(target=B_ + 4, target_is_int64=1), "target is not aligned")
    for name in ("target", "stats", "dlogp"):
        refused(probs_back(**{name: {"target": B_, "stats": C_, "dlogp": D}[name] + 2}), "an input is not aligned")
    refused(probs_back(dentropy=F + 1), "an input is not aligned")
    refused(probs_back(target=B_ + 4, target_is_int64=1), "an input is not aligned")


def test_adamw_refuses_device_scalars_off_their_elements():
    for name, off in (("rate_device", 2), ("grad_scale_device", 1), ("skip_device", 2), ("t_device", 4)):
        refused(adamw([{}], **{name: E + off}), "not aligned")
