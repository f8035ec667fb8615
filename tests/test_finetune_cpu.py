"""Host-side behaviour of the fine-tuning operators and layers: refusals, sizes, construction, pickles (no GPU work:
pointers are never dereferenced)."""
import copy
import ctypes
import pickle

import pytest
import torch

import flash_eq as fe
from flash_eq import _native as N

FAKE = 256


def refused(rc, text):
    assert rc != 0 and text in N.load_library().feq_last_error().decode(), N.load_library().feq_last_error()


def test_cpu_tensors_are_refused():
    g = fe.Graph(torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int64), 2)
    seed, linear = torch.zeros(1, dtype=torch.int64), fe.EquivariantLinear(fe.Repr([0, 1], 4), fe.Repr([0, 1], 4))
    for call in (lambda: fe.feature_dropout(torch.randn(4), 0.5, seed), lambda: fe.distance_buckets(torch.rand(3), torch.rand(2)),
                 lambda: fe.edge_attention_weights(torch.randn(2, 4, 4), g, 1, torch.zeros(())),
                 lambda: fe.edge_attention_weights_qk(torch.randn(3, 1, 4), torch.randn(3, 1, 4), g, torch.zeros(())),
                 lambda: fe.EquivariantDropout(fe.Repr([0, 1], 4), 0.5)(torch.randn(3, 4, 4)),
                 lambda: fe.DistanceBuckets(4)(torch.rand(3))):
        with pytest.raises(fe.CUDANotAvailableError):
            call()
    with pytest.raises(ValueError, match="has none"):
        linear(torch.randn(3, 4, 4), object())
    with pytest.raises(ValueError, match="has none"):
        fe.EquivariantTransformerBlock(fe.Repr([0, 1], 4), fe.Repr([0, 1], 4))(None, None, torch.randn(3, 4, 4), None, g,
                                                                              adapters=torch.zeros(3, dtype=torch.int64))


def test_dropout_abi_refusals():
    lib = N.load_library()

    def drop(lv=(0, 1), n=None, channels=8, dt=0, p=0.5, x=FAKE, seed=FAKE):
        a = (ctypes.c_int32 * max(len(lv), 1))(*lv)
        return lib.feq_dropout(a, len(lv) if n is None else n, channels, 0, dt, x, p, seed, FAKE, None)
    refused(drop(channels=-1), "-1 channels")
    refused(drop(dt=3), "unknown element type 3")
    for p in (-0.1, 1.0001, float("nan")):
        refused(drop(p=p), "not in [0, 1]")
    refused(drop(lv=()), "non-empty")
    refused(drop(lv=(0,) * 33), "more than 32 irreps")
    refused(drop(lv=(-1,)), "negative degree")
    refused(drop(lv=(64,)), "dimension exceeds 128")
    refused(drop(lv=(2 ** 31 - 1,)), "dimension exceeds 128")
    refused(drop(x=None), "NULL")
    refused(drop(seed=None), "NULL")
    refused(drop(channels=2 ** 62), "channels of 4 components")
    assert drop(channels=0) == 0
    refused(lib.feq_distance_buckets(FAKE, -1, FAKE, 2, FAKE, None), "negative sizes")
    refused(lib.feq_distance_buckets(FAKE, 4, None, 2, FAKE, None), "NULL")
    assert lib.feq_distance_buckets(None, 0, None, 0, None, None) == 0


def attention(**kw):
    a = N.FeqEdgeAttn(num_edges=10, num_nodes=4, num_k=4, heads=2, head_len=8, head_runs=1, dtype=0, ldq=32, ldk=32, head_stride=8,
                      q=FAKE, k=FAKE, q_idx=FAKE, k_idx=FAKE, perm=FAKE, offsets=FAKE, log_scale=FAKE)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_attention_abi_refusals():
    lib = N.load_library()
    fwd = lambda w=FAKE, out=None, **kw: lib.feq_edge_attn_fwd(ctypes.byref(attention(**kw)), w, out, None)
    refused(lib.feq_edge_attn_fwd(None, FAKE, None, None), "NULL")
    refused(fwd(num_edges=-1), "invalid graph sizes")
    refused(fwd(num_nodes=0), "invalid graph sizes")
    refused(fwd(num_edges=2 ** 31), "2^31 - 1 edges")
    refused(fwd(num_nodes=2 ** 25 + 1), "2^25 nodes")
    refused(fwd(num_k=2 ** 25 + 1), "2^25 nodes")
    refused(fwd(heads=0), "num_heads must be 1 to 1024")
    refused(fwd(heads=1025), "num_heads must be 1 to 1024")
    refused(fwd(head_len=0), "runs of 0 elements")
    refused(fwd(head_runs=129), "129 runs")
    refused(fwd(dtype=3), "unknown element type")
    refused(fwd(bias=FAKE, num_buckets=0, buckets=FAKE), "0 buckets")
    refused(fwd(bias=FAKE, num_buckets=4097, buckets=FAKE), "4097 buckets")
    refused(fwd(bias=FAKE, num_buckets=4), "buckets")
    refused(fwd(bias=FAKE, num_buckets=4, buckets=FAKE, bias_dtype=9), "unknown element type 9")
    refused(fwd(dropout=1.5, seed=FAKE, out=FAKE), "not in [0, 1]")
    refused(fwd(dropout=0.5, out=FAKE), "needs a seed")
    refused(fwd(dropout=0.5, seed=FAKE), "are the result")
    refused(fwd(dtype=1), "are the result")
    refused(fwd(decay=-1.0), "negative distance decay")
    refused(fwd(decay=1.0), "needs distances")
    refused(fwd(q_idx=None), "both be given")
    refused(fwd(log_scale=None), "NULL")
    refused(fwd(q=None), "NULL")
    refused(fwd(w=None), "NULL")
    assert fwd(num_edges=0) == 0
    a = attention(bias=FAKE, num_buckets=4, buckets=FAKE)
    need = lib.feq_edge_attn_bwd_workspace(ctypes.byref(a), 1, 1)
    assert need > 0 == lib.feq_edge_attn_bwd_workspace(ctypes.byref(a), 0, 0)

    def bwd(a=a, w=FAKE, gq=FAKE, gk=FAKE, gb=FAKE, gls=FAKE, gd=None, ws=FAKE, size=need, perm=FAKE):
        return lib.feq_edge_attn_bwd(ctypes.byref(a), perm, FAKE, w, FAKE, FAKE, gq, 32, gk, 32, gb, gls, gd, ws, size, None)
    refused(bwd(size=need - 1), "workspace")
    refused(bwd(ws=None), "NULL")
    refused(bwd(w=None), "NULL")
    refused(bwd(gk=None), "both be given")
    refused(bwd(gq=None, gk=None), "comes with those of q and k")
    refused(bwd(perm=None), "CSR of the edges by k_idx")
    refused(bwd(gd=FAKE), "no distance decay")
    refused(bwd(a=attention()), "no bias")
    refused(bwd(a=attention(num_edges=0)), "no edges")


def test_adapter_abi_refusals():
    lib = N.load_library()
    lv = (ctypes.c_int32 * 2)(0, 1)
    cols = (ctypes.c_int32 * 2)(0, -1)

    def fwd(n=2, x=3, rows=7, ci=8, co=9, r=4, dt=0, down=FAKE, scale=1.0, bias=None, nbias=1, low=None):
        return lib.feq_adapter_linear_fwd(lv, n, x, rows, ci, co, r, dt, FAKE, FAKE, down, FAKE, scale, FAKE, FAKE, bias, nbias, cols, FAKE, low,
                                          None)
    refused(fwd(n=0), "non-empty")
    refused(fwd(x=0), "0 experts")
    refused(fwd(x=1025), "more than 1024")
    refused(fwd(rows=-1), "-1 rows")
    refused(fwd(rows=2 ** 30 + 1), "2^30 rows")
    refused(fwd(ci=0), "0 to 9 channels")
    refused(fwd(co=65537), "65536 channels")
    refused(fwd(r=0), "rank 0")
    refused(fwd(r=65), "rank above 64")
    refused(fwd(dt=5), "unknown element type 5")
    refused(fwd(scale=float("inf")), "not finite")
    refused(fwd(down=None), "NULL")
    refused(fwd(bias=FAKE, nbias=2), "bias columns")
    refused(fwd(ci=129), "no room")
    assert fwd(rows=0) == 0
    low = lambda ci, co, r, train: lib.feq_adapter_linear_low_floats(lv, 2, 7, ci, co, r, train)
    assert low(64, 64, 16, 1) == low(128, 300, 64, 0) == 0
    assert low(129, 8, 1, 0) == 4 * 7 * 16 and low(64, 129, 17, 1) == low(64, 64, 17, 1) == 4 * 7 * 32
    need = lib.feq_adapter_linear_bwd_workspace(lv, 2, 3, 7, 8, 200, 4, 0, 1, 1)
    assert need > 0

    def bwd(co=200, gx=FAKE, gd=FAKE, gu=FAKE, gw=FAKE, gb=FAKE, low=FAKE, ws=FAKE, size=need, rows=7):
        return lib.feq_adapter_linear_bwd(lv, 2, 3, rows, 8, co, 4, 0, FAKE, FAKE, FAKE, FAKE, FAKE, 1.0, FAKE, FAKE, low, 1, cols, gx, gd, gu,
                                          gw, gb, ws, size, None)
    refused(bwd(size=need - 1), "workspace")
    refused(bwd(low=None), "reduced rows")
    refused(bwd(gx=None), "come with that of x")
    refused(bwd(gw=None), "comes with the weight's")
    refused(bwd(rows=0), "no rows")
    refused(bwd(ws=None), "NULL")


def test_layers_refuse_and_describe():
    r = fe.Repr([0, 1], 4)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="between 0 and 1"):
            fe.EquivariantDropout(r, p)
        with pytest.raises(ValueError, match="between 0 and 1"):
            fe.EquivariantEdgeAttention(2, 4, dropout=p if p == p else 2.0, counter_dropout=True)
    for n in (-1, 4097):
        with pytest.raises(ValueError, match="bias_buckets must be"):
            fe.EquivariantEdgeAttention(2, 4, bias_buckets=n)
    for n in (0, 4097):
        with pytest.raises(ValueError, match="num_buckets must be"):
            fe.DistanceBuckets(n)
    with pytest.raises(ValueError, match="buckets from"):
        fe.DistanceBuckets(4, 3.0, 3.0)
    with pytest.raises(ValueError, match="buckets from"):
        fe.DistanceBuckets(4, 0.0, 3.0, log_bins=True)
    for n, rank in ((0, 4), (1025, 4)):
        with pytest.raises(ValueError, match="num_adapters must be"):
            fe.LinearAdapters(r, r, n, rank)
    for rank in (0, 65):
        with pytest.raises(ValueError, match="rank must be"):
            fe.LinearAdapters(r, r, 2, rank)
    with pytest.raises(ValueError, match="alpha must be finite"):
        fe.LinearAdapters(r, r, 2, 4, float("inf"))
    with pytest.raises(ValueError, match="no EquivariantLinear"):
        fe.add_adapters(torch.nn.Linear(3, 3), 2)
    with pytest.raises(TypeError, match="must be an ExpertPlan"):
        fe.adapter_linear(torch.zeros(1), torch.zeros(1), torch.zeros(1), torch.zeros(1), None)
    for m in (fe.EquivariantDropout(r, 0.25), fe.DistanceBuckets(7), fe.LinearAdapters(r, r, 2, 4)):
        assert type(m).__name__ in repr(m)


def test_bucket_boundaries():
    b = fe.DistanceBuckets(5, 1.0, 9.0)
    assert b.boundaries.tolist() == [3.0, 5.0, 7.0, 9.0]
    assert fe.DistanceBuckets(1).boundaries.numel() == 0
    assert fe.DistanceBuckets(4, 1.0, 8.0, log_bins=True).boundaries.tolist() == pytest.approx([2.0, 4.0, 8.0], rel=1e-6)
    b = fe.DistanceBuckets(7, 0.0, 1.0)
    exact = b.boundaries.clone()
    for change in (lambda: b.bfloat16(), lambda: b.half(), lambda: b.double(), lambda: b.float()):
        change()
        assert b.boundaries.dtype == torch.float32 and torch.equal(b.boundaries, exact)
    assert not b.state_dict()


def test_adapters_start_as_nothing_and_follow_their_map():
    linear = fe.EquivariantLinear(fe.Repr([0, 1, 1], 4), fe.Repr([0, 1, 1], 6)).bfloat16()
    before = set(linear.state_dict())
    params = linear.add_adapters(3, 2, alpha=8)
    assert linear.adapters.scale == 4.0 and all(p.dtype == torch.bfloat16 and p.requires_grad for p in params)
    assert linear.adapters.down.shape == (3, 3, 2, 4) and linear.adapters.up.shape == (3, 3, 6, 2)
    assert (linear.adapters.up == 0).all() and (linear.adapters.down != 0).any()
    assert set(linear.state_dict()) - before == {"adapters.down", "adapters.up"}
    linear.add_adapters(2, 1)
    assert linear.adapters.down.shape[0] == 2
    twin = copy.deepcopy(linear)
    twin.load_state_dict(linear.state_dict())
    assert torch.equal(pickle.loads(pickle.dumps(twin)).adapters.down, linear.adapters.down)
    model = fe.EquivariantTransformer(fe.Repr([0, 1], 4), fe.Repr([0, 1], 4), fe.Repr([0], 4), num_layers=2, num_heads=2)
    assert len(fe.add_adapters(model, 2, 3)) == 2 * 3 * 2


def test_options_change_nothing_where_they_are_off():
    """Same parameters from the same seed, same state names, and pickles of modules made before the options."""
    def build(**kw):
        torch.manual_seed(3)
        return fe.EquivariantTransformer(fe.Repr([0, 1], 4), fe.Repr([0, 1], 4), fe.Repr([0], 4), num_layers=2, num_heads=2, dropout=0.1, **kw)
    plain, tuned = build(), build(bias_buckets=5, counter_dropout=True, feature_dropout=0.2)
    state = tuned.state_dict()
    extra = set(state) - set(plain.state_dict())
    assert extra == {f"layers.{i}.attn.attention.bias" for i in range(2)}
    for k, v in plain.state_dict().items():
        assert torch.equal(v, state[k])
    assert isinstance(plain.layers[0].attn.attention.dropout, torch.nn.Dropout)
    old = pickle.loads(pickle.dumps(plain))
    for m in old.modules():                              # as unpickled from before there were these attributes
        state = {k: v for k, v in m.__dict__.items() if k not in ("counter_dropout", "adapters", "feature_dropout", "buckets")}
        if isinstance(m, fe.EquivariantEdgeAttention):
            state["_parameters"] = {k: v for k, v in state["_parameters"].items() if k != "bias"}
        m.__dict__.clear()
        m.__setstate__(state)
    attention = old.layers[0].attn.attention
    assert attention.bias is None and attention.counter_dropout == 0.0 and old.buckets is None
    assert old.layers[0].feature_dropout is None and old.layers[0].mlp_up.adapters is None
    assert fe.EquivariantDropout(fe.Repr([0], 4), 0.5).eval()(torch.ones(2, 4, 1)).eq(1).all()


def test_bucket_boundaries_of_a_model_built_without_memory():
    want = fe.DistanceBuckets(9, 0.5, 8.0, True).boundaries
    with torch.device("meta"):
        b = fe.DistanceBuckets(9, 0.5, 8.0, True)
    assert b.boundaries.is_meta
    assert torch.equal(b.to_empty(device="cpu").boundaries, want)
