"""Every operator that the dispatcher knows in this package's namespaces has a case in the files that run
torch.library.opcheck. (An attribute of torch.ops that was never looked up is not in its dir(), so
what is registered is asked of the dispatcher.)"""

import pytest
import torch

from tests import test_gpu_contract, test_gpu_int8_layers, test_gpu_narrow_layers


def _registered(ns: str) -> set[str]:
    import torchtitan_amd  # noqa: F401

    return {n.split("::")[1].split(".")[0] for n in torch._C._dispatch_get_all_op_names() if n.startswith(ns + "::")}


def _checked(names: list[str]) -> set[str]:
    return {n.replace("_no_shared", "").replace("_dw_only", "") for n in names}


@pytest.mark.parametrize("ns,names", [
    ("moe_mi355x", test_gpu_contract.OPCHECK_NAMES), ("moe_mi355x_mx", test_gpu_narrow_layers.OP_NAMES),
    ("moe_mi355x_int8", test_gpu_int8_layers.OP_NAMES)])
def test_every_operator_has_a_case(ns, names):
    assert _registered(ns) == _checked(names)


def test_every_kernel_is_behind_an_operator():
    """The bare kernels are those behind the operators that refuse derivatives."""
    for ns in ("moe_mi355x_mx", "moe_mi355x_int8"):
        bare = _registered(ns + "_bare")
        assert bare and bare <= _registered(ns)


def test_one_without_a_case_is_seen():
    lib = torch.library.Library("moe_mi355x_int8", "FRAGMENT")
    try:
        lib.define("without_a_case(Tensor x) -> Tensor")
        assert _registered("moe_mi355x_int8") - _checked(test_gpu_int8_layers.OP_NAMES) == {"without_a_case"}
    finally:
        lib._destroy()
