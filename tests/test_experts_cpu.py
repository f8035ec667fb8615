"""Host-side behaviour of the layer norm's and the expert routing's entry points: refusals, sizes,
construction (no GPU work: pointers are never dereferenced)."""
import copy
import ctypes
import pickle
from types import SimpleNamespace

import pytest
import torch

import flash_eq as fe
from flash_eq import _native as N

FAKE = ctypes.c_void_p(256)


def refused(rc, text):
    assert rc != 0 and text in N.load_library().feq_last_error().decode(), N.load_library().feq_last_error()


def test_cpu_tensors_are_refused():
    x, ids = torch.randn(4, 8), torch.zeros(4, 1, dtype=torch.int64)
    for call in (lambda: fe.expert_topk(x, 2), lambda: fe.ExpertPlan(ids, 2),
                 lambda: fe.EquivariantExpertMLP(fe.Repr([0, 1], 4), 2)(torch.randn(3, 4, 4))):
        with pytest.raises(fe.CUDANotAvailableError):
            call()


def test_invariant_norm_on_the_cpu_is_pytorchs():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 5, 8, generator=g, dtype=torch.float64)
    norm = fe.InvariantLayerNorm(8, epsilon=1e-3).double()
    with torch.no_grad():
        norm.weight.copy_(torch.randn(8, generator=g))
        norm.bias.copy_(torch.randn(8, generator=g))
    ref = torch.nn.functional.layer_norm(x, (8,), norm.weight, norm.bias, 1e-3)
    assert torch.equal(norm(x), ref)
    assert fe.InvariantLayerNorm(8, affine=False).weight is None
    with pytest.raises(ValueError, match=r"features must be \(..., 8\)"):
        norm(torch.randn(3, 7, dtype=torch.float64))
    with pytest.raises(ValueError, match="width must be positive"):
        fe.InvariantLayerNorm(0)


def test_layernorm_abi_refusals():
    lib = N.load_library()
    fwd = lambda rows=4, width=8, ldx=8, dt=0, mean=None, rstd=None: lib.feq_layernorm_fwd(
        FAKE, rows, width, ldx, dt, None, None, 0, 1e-5, FAKE, mean, rstd, None)
    refused(fwd(rows=-1), "layer norm of -1 rows")
    refused(fwd(width=0), "width 0")
    refused(fwd(ldx=7), "row stride 7 is smaller")
    refused(fwd(dt=3), "unknown element type 3")
    refused(fwd(mean=FAKE), "together")
    assert fwd(rows=0) == 0
    need = lib.feq_layernorm_bwd_workspace(1000, 192, 0)
    assert 0 < need <= 1000 * 2 * 192 * 4
    refused(lib.feq_layernorm_bwd(FAKE, 192, FAKE, 1000, 192, 192, 0, None, 0, FAKE, FAKE, None, FAKE, None, FAKE,
                                  need - 1, None), "workspace")


def test_topk_abi_refusals():
    lib = N.load_library()
    fwd = lambda rows=4, x=8, k=2, dt=0, mean=None, ws=0: lib.feq_expert_topk_fwd(
        FAKE, rows, x, dt, k, 1, FAKE, FAKE, mean, None, ws, None)
    refused(fwd(k=9), "9 of 8 experts")
    refused(fwd(k=0), "0 of 8 experts")
    refused(fwd(x=1025), "more than 1024 experts")
    refused(fwd(x=100, k=65), "more than 64 choices")
    refused(fwd(dt=7), "unknown element type")
    refused(fwd(rows=1000, mean=FAKE), "workspace")
    assert fwd(rows=0) == 0


def test_plan_and_row_abi_refusals():
    lib = N.load_library()
    refused(lib.feq_expert_plan(FAKE, 4, 0, FAKE, FAKE, FAKE, None, 0, None), "over 0 experts")
    refused(lib.feq_expert_plan(FAKE, 4, 1025, FAKE, FAKE, FAKE, None, 0, None), "more than 1024")
    refused(lib.feq_expert_plan(FAKE, 2 ** 31, 4, FAKE, FAKE, FAKE, None, 0, None), "2^31 - 1 slots")
    refused(lib.feq_expert_plan(FAKE, 10 ** 6, 4, FAKE, FAKE, FAKE, None, 0, None), "workspace")
    assert lib.feq_expert_plan_workspace(8192, 8) == 0 < lib.feq_expert_plan_workspace(8193, 8)
    refused(lib.feq_expert_dispatch(FAKE, 1, 4, 0, 8, 0, FAKE, FAKE, FAKE, None), "0 slots a row")
    refused(lib.feq_expert_dispatch(FAKE, 1, 4, 65, 8, 0, FAKE, FAKE, FAKE, None), "more than 64 slots")
    refused(lib.feq_expert_dispatch(FAKE, 70000, 4, 1, 8, 0, FAKE, FAKE, FAKE, None), "65535 planes")
    refused(lib.feq_expert_combine(FAKE, 1, 2 ** 30, 4, 8, 0, FAKE, FAKE, None, 0, FAKE, None), "2^31 - 1 slots")
    refused(lib.feq_expert_combine_bwd(FAKE, None, 1, 4, 1, 8, 0, FAKE, FAKE, FAKE, 0, None, FAKE, None), "NULL")


def test_linear_abi_refusals():
    lib = N.load_library()
    i32 = lambda *v: (ctypes.c_int32 * len(v))(*v)

    def fwd(lv=(0, 1), x=4, s=10, ci=8, co=8, dt=0, nb=1, cols=(0, -1)):
        return lib.feq_expert_linear_fwd(i32(*lv), len(lv), x, s, ci, co, dt, FAKE, FAKE, FAKE, FAKE, nb, i32(*cols), FAKE,
                                         None)
    refused(fwd(x=0), "of 0 experts")
    refused(fwd(x=1025), "more than 1024 experts")
    refused(fwd(s=2 ** 30 + 1), "more than 2^30 rows")
    refused(fwd(lv=(0, -1)), "negative degree")
    refused(fwd(lv=tuple([0] * 33), cols=tuple([-1] * 33)), "more than 32 irreps")
    refused(fwd(lv=(0, 64), cols=(0, -1)), "dimension exceeds 128")
    refused(fwd(cols=(-1, 0)), "bias column 0 of irrep 1")           # a vector irrep
    refused(fwd(cols=(1, -1)), "bias column 1 of irrep 0")           # no such column
    refused(fwd(lv=(0, 0), nb=2, cols=(0, 0)), "bias column 0 of irrep 1")
    refused(fwd(lv=(0, 0), nb=2, cols=(0, -1)), "not each of them")
    refused(fwd(dt=5), "unknown element type")
    lib_ws = lib.feq_expert_linear_bwd_workspace(i32(0, 1), 2, 4, 10000, 64, 64, 1)
    assert lib_ws > 0
    refused(lib.feq_expert_linear_bwd_w(i32(0, 1), 2, 4, 10000, 64, 64, 0, FAKE, FAKE, FAKE, 1, i32(0, -1), FAKE, FAKE, FAKE,
                                        lib_ws - 1, None), "workspace")


def test_construction():
    with pytest.raises(ValueError, match="top_k must be 1 to num_experts"):
        fe.ExpertRouter(fe.Repr([0, 1], 4), 2, top_k=3)
    with pytest.raises(ValueError, match="cannot modify the degrees"):
        fe.EquivariantExpertLinear(fe.Repr([0, 1], 4), fe.Repr([0], 4), 2)
    lin = fe.EquivariantExpertLinear(fe.Repr([0, 1, 0], 4), fe.Repr([0, 1, 0], 6), 5)
    assert lin.weight.shape == (5, 3, 6, 4) and lin.bias.shape == (5, 6, 2)
    assert fe.EquivariantExpertLinear(fe.Repr([1], 4), fe.Repr([1], 4), 2).bias is None


def test_blocks_without_experts_are_unchanged():
    """The option adds nothing to the default block: names, order and values of its seeded parameters."""
    rp = fe.Repr([0, 1], 8)
    torch.manual_seed(3)
    plain = fe.EquivariantTransformerBlock(rp, rp)
    assert plain.experts is None and "mlp_up.weight" in plain.state_dict()
    torch.manual_seed(3)
    mixed = fe.EquivariantTransformerBlock(rp, rp, num_experts=4, experts_per_node=2)
    keys = set(mixed.state_dict())
    assert {"experts.router.linear.weight", "experts.up.weight", "experts.down.bias"} <= keys
    assert not any(k.startswith("mlp_up") for k in keys)
    shared = [k for k in plain.state_dict() if k.startswith(("norm1", "attn"))]
    assert shared and all(torch.equal(plain.state_dict()[k], mixed.state_dict()[k]) for k in shared)
    model = fe.EquivariantTransformer(rp, rp, rp, num_layers=2, num_experts=3, experts_per_node=1)
    assert all(layer.experts.router.top_k == 1 for layer in model.layers)


def test_numbers_of_experts():
    rp = fe.Repr([0, 1], 8)
    for n, k in ((0, 1), (1025, 2)):
        with pytest.raises(ValueError, match="num_experts must be 1 to 1024"):
            fe.ExpertRouter(rp, n, k)
    with pytest.raises(ValueError, match="at most 64"):
        fe.ExpertRouter(rp, 100, 65)
    with pytest.raises(ValueError, match="must not be negative"):
        fe.EquivariantTransformerBlock(rp, rp, num_experts=-1)


def test_linear_abi_refuses_a_bias_without_columns():
    lib = N.load_library()
    one = (ctypes.c_int32 * 1)(0)
    for cols, n in ((None, 1), (one, 0)):
        assert lib.feq_expert_linear_fwd(one, 1, 2, 10, 4, 4, 0, FAKE, FAKE, FAKE, FAKE, n, cols, FAKE, None) != 0
        assert "bias" in lib.feq_last_error().decode()


@pytest.fixture
def host_plan(monkeypatch):
    """A function that makes plans of host tensors: one row for each of two experts, as the kernels would return it."""
    real = N.nodes()

    def expert_plan(ids, num_experts):
        n = ids.shape[0]
        place = torch.arange(n, dtype=torch.int32)
        return place, place[:, None].clone(), torch.arange(num_experts + 1, dtype=torch.int32)
    monkeypatch.setattr(N, "nodes", lambda: SimpleNamespace(expert_plan=expert_plan, plan_copy=real.plan_copy,
                                                            expert_linear=lambda *a: a))
    return lambda: fe.ExpertPlan(torch.tensor([0, 1]), 2)


def test_a_changed_plan_is_not_copied(host_plan):
    """A copy's tensors count their changes anew, so the plan's have to be looked at before."""
    for copied in (copy.copy, copy.deepcopy, lambda p: pickle.loads(pickle.dumps(p))):
        plan = host_plan()
        other = copied(copied(plan))
        assert other.positions.tolist() == plan.positions.tolist() and other.positions._version == 0
        assert other.positions.data_ptr() != plan.positions.data_ptr()
        for name in ("order", "positions", "offsets"):
            for plan in (host_plan(), other, copied(host_plan())):
                getattr(plan, name).add_(2 ** 30)
                with pytest.raises(RuntimeError, match="of an ExpertPlan have been modified"):
                    copied(plan)


def test_a_plans_sizes_are_those_of_its_tensors(host_plan):
    """The kernels' bounds come from them: none can be set, and no other object stands for a plan."""
    plan = host_plan()
    assert (plan.num_experts, plan.num_rows, plan.top_k, plan.num_slots) == (2, 2, 1, 2)
    for name in ("num_experts", "num_rows", "top_k", "num_slots", "order", "positions", "offsets"):
        with pytest.raises(AttributeError):
            setattr(plan, name, 1)
    assert repr(plan) == "ExpertPlan(rows=2, top_k=1, num_experts=2)"
    x, w = torch.randn(1, 8), torch.randn(2, 1, 4, 8)
    assert fe.expert_linear(x, w, plan)[4] == 2
    with pytest.raises(TypeError, match="plan must be an ExpertPlan, got SimpleNamespace"):
        fe.expert_linear(x, w, SimpleNamespace(offsets=plan.offsets, num_slots=1))


def test_blocks_pickled_before_the_experts_option():
    rp = fe.Repr([0, 1], 8)
    block = fe.EquivariantTransformerBlock(rp, rp)
    del block.experts
    assert pickle.loads(pickle.dumps(block)).experts is None
    mixed = pickle.loads(pickle.dumps(fe.EquivariantTransformerBlock(rp, rp, num_experts=2)))
    assert isinstance(mixed.experts, fe.EquivariantExpertMLP)


def test_linear_takes_all_the_slots_of_a_plan():
    """2^30 rows pass the check of sizes (and meet the next one, of the type)."""
    lib = N.load_library()
    one = (ctypes.c_int32 * 1)(0)
    for slots, text in ((2 ** 30, "unknown element type"), (2 ** 30 + 1, "more than 2^30 rows")):
        refused(lib.feq_expert_linear_fwd(one, 1, 2, slots, 1, 1, 9, FAKE, FAKE, FAKE, None, 0, None, FAKE, None), text)
        refused(lib.feq_expert_linear_bwd_w(one, 1, 2, slots, 1, 1, 9, FAKE, FAKE, FAKE, 0, None, FAKE, None, FAKE, 0, None),
                text)


def test_linear_abi_refuses_columns_that_there_are_not():
    """Numbers that would wrap around in the kernels' tables: below -1, and of 32 and more."""
    lib = N.load_library()
    i32 = lambda *v: (ctypes.c_int32 * len(v))(*v)

    def calls(lv, nb, cols):
        common = (i32(*lv), len(lv), 2, 10, 8, 8, 0)
        yield lib.feq_expert_linear_fwd(*common, FAKE, FAKE, FAKE, FAKE, nb, i32(*cols), FAKE, None)
        yield lib.feq_expert_linear_bwd_w(*common, FAKE, FAKE, FAKE, nb, i32(*cols), FAKE, FAKE, None, 0, None)
    for lv, nb, cols, text in (((0,), 1, (-200,), "bias column -200 of irrep 0"), ((0, 0), 1, (0, -2), "bias column -2 of irrep 1"),
                               ((0, 0), 34, (33, 1), "34 bias columns"), ((0,), 300, (256,), "300 bias columns"),
                               ((0, 0), 33, (32, 0), "33 bias columns")):
        for rc in calls(lv, nb, cols):
            refused(rc, text)
