"""More calls that the row operators refuse on the host, before anything touches a device (the addresses here are never
dereferenced), and what they no longer refuse."""
from pixienn_b200 import capi

from test_row_operators_args import A, B_, C_, D, E, F, adamw, probs, probs_back, refused


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


def test_adamw_refuses_device_scalars_inside_what_it_writes():
    """A block would read the scalar while another writes it."""
    for name in ("rate_device", "grad_scale_device", "skip_device", "t_device"):
        for inside in (A, A + 3992, C_ + 8, D + 3992):
            refused(adamw([{}], **{name: inside}), "device scalar")
    refused(adamw([{}, {"param": E, "grad": B_ + 8000, "m": C_ + 8000, "v": F}], t_device=F + 3992), "device scalar")
    refused(adamw([{"m_scale": E, "v_scale": F}], state_bits=8, rate_device=F + 12), "device scalar")
    refused(adamw([{"master": E}], param_type=capi.BF16, grad_type=capi.BF16, skip_device=E), "device scalar")


def test_adamw_seed_comes_with_8_bit_state():
    refused(adamw([{}], seed=1), "seed")
    refused(adamw([{"m_scale": E, "v_scale": F, "m": C_ + 2, "grad": A}], state_bits=8, seed=1), "overlap")        # (past the seed's check)
