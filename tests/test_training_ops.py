"""The training operators -- edge attention, the norms around a block, channel dropout -- against 64-bit restatements (oracle/training_oracle.py), and what
they refuse.  Tolerances count roundings: u = 2^-24 is a float32 operation's, half a step of the type an output's own; each test says how many."""
import copy
import ctypes as C
import math
import os
import socket

import pytest
import torch

from diffusion_edf_amd import _lib
from diffusion_edf_amd.drop import EquivariantDropout, dropout_rng, equivariant_dropout, row_shape
from diffusion_edf_amd.edge_attention import EdgeAttention, EdgeSegments, edge_attention
from diffusion_edf_amd.layer_norm import EquivariantLayerNormV2, NormGateResidual, equivariant_layer_norm, norm_gate_residual
from diffusion_edf_amd.so3 import parse_irreps
from oracle import training_oracle as O

U = 2.0 ** -24
INF = float("inf")
FMAX = torch.finfo(torch.float32).max
TYPES = [torch.float32, torch.float16, torch.bfloat16]
LMAX2 = "64x0e+32x1e+16x2e"


def half_step(t):
    return torch.finfo(t).eps / 2


def close(got, want, tol, what):
    """|got - want| <= tol + half a step of got's type of |want| (+ the smallest float16 steps), NaN and infinities in the same places"""
    got, want = got.detach().cpu(), want.detach()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    err = (got.double() - want.double()).abs()
    bound = tol + half_step(got.dtype) * want.abs() + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / torch.as_tensor(bound).clamp(min=1e-300)).nan_to_num(INF).max()):.3g} times the bound"


# ---- on the CPU: the oracle itself, and refusals ----------------------------------------------------------------------------------------------

def test_oracle_philox_known_answers():
    """the published test vectors of Philox4x32-10 (Random123 kat_vectors): zero counter and key, all ones, digits of pi"""
    assert O.philox((0,) * 4, (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert O.philox((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert O.philox((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def test_oracle_attention_is_the_inference_oracles():
    """against the softmax of oracle/restatement.py's block: scatter over destinations, empty segments zero"""
    g = torch.Generator().manual_seed(0)
    dst = torch.tensor([0, 0, 0, 2, 2, 4])
    a, v, w = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((6, 4, 16), (6, 4, 60), (4, 16)))
    l = torch.randn(6, generator=g, dtype=torch.float64)
    t = torch.einsum("ehk,hk->eh", O.act(a), w) + l[:, None]
    z = torch.zeros(5, 4, dtype=torch.float64).index_add_(0, dst, t.exp())
    want = torch.zeros(5, 4, 60, dtype=torch.float64).index_add_(0, dst, (t.exp() / z[dst])[..., None] * v)
    assert (O.attention(a, v, w, dst, 5, l) - want).abs().max() < 1e-14


def _segments_without_gpu(n_edges, n_dst):
    s = object.__new__(EdgeSegments)
    s.n_dst, s.n_edges, s.device, s.dst, s.rowptr = n_dst, n_edges, torch.device("cpu"), torch.zeros(n_edges, dtype=torch.int32), torch.zeros(n_dst + 1, dtype=torch.int32)
    return s


def test_edge_attention_refusals():
    E, H, K, D = 6, 4, 16, 60
    a, v, w, seg = torch.randn(E, H, K), torch.randn(E, H, D), torch.randn(H, K), _segments_without_gpu(E, 3)
    table, bounds, length = torch.zeros(5, H), torch.linspace(0, 1, 4), torch.rand(E)
    rng = dropout_rng(1, device="cpu")
    bad = [
        (ValueError, (a[0], v, w, seg), {}), (ValueError, (a, v[:5], w, seg), {}), (ValueError, (a[:5], v[:5], w, seg), {}),
        (TypeError, (a.half(), v, w, seg), {}), (TypeError, (a.double(), v.double(), w, seg), {}),
        (ValueError, (a, v, w[:3], seg), {}), (ValueError, (a, v, w.half(), seg), {}), (ValueError, (a, v[:, :, :0], w, seg), {}),
        (ValueError, (a, v, w, seg), {"edge_logits": torch.zeros(E, H)}), (ValueError, (a, v, w, seg), {"edge_logits": torch.zeros(E).half()}),
        (ValueError, (a, v, w, seg), {"edge_length": length}), (ValueError, (a, v, w, seg), {"bias_table": table}),
        (ValueError, (a, v, w, seg), {"bias_table": table, "edge_length": length, "bias_boundaries": bounds[:3]}),
        (ValueError, (a, v, w, seg), {"bias_table": table[:, :3], "edge_length": length, "bias_boundaries": bounds}),
        (ValueError, (a, v, w, seg), {"bias_table": table, "edge_length": length[:5], "bias_boundaries": bounds}),
        (ValueError, (a, v, w, seg), {"dropout": 1.0, "rng": rng}), (ValueError, (a, v, w, seg), {"dropout": -0.1, "rng": rng}),
        (ValueError, (a, v, w, seg), {"dropout": float("nan"), "rng": rng}), (ValueError, (a, v, w, seg), {"dropout": 0.1}),
        (ValueError, (a, v, w, seg), {"dropout": 0.1, "rng": rng[:1]}), (ValueError, (a, v, w, seg), {"dropout": 0.1, "rng": rng.int()}),
        (NotImplementedError, (torch.zeros(E, 17, 1), torch.zeros(E, 17, 1), torch.zeros(17, 1), seg), {}),
        (NotImplementedError, (torch.zeros(E, 4, 65), v, torch.zeros(4, 65), seg), {}), (NotImplementedError, (a, torch.zeros(E, 4, 257), w, seg), {}),
        (NotImplementedError, (a, v, w, seg), {"bias_table": torch.zeros(600, 4), "edge_length": length, "bias_boundaries": torch.zeros(599)}),
        (RuntimeError, (a, v, w, seg), {}),          # nothing is wrong but the device: there is no CPU path
    ]
    for err, args, kw in bad:
        with pytest.raises(err):
            edge_attention(*args, **kw)
    for err, args in ((ValueError, (torch.zeros(3), 3)), (ValueError, (torch.zeros(3, 1, dtype=torch.int64), 3)), (ValueError, (torch.zeros(3, dtype=torch.int64), 0)),
                      (ValueError, (torch.zeros(0, dtype=torch.int64), -1)), (RuntimeError, (torch.zeros(3, dtype=torch.int64), 3))):
        with pytest.raises(err):
            EdgeSegments(*args)


def test_edge_attention_counts_value_channels_in_whole_quads(built_lib):
    """3 heads of 341 are 258 quads, of 340 255"""
    import ctypes as C
    seg, lib = _segments_without_gpu(6, 3), built_lib
    for D, fits in ((340, True), (341, False)):
        with pytest.raises(RuntimeError if fits else NotImplementedError) as e:          # (that fits: only the device is wrong)
            edge_attention(torch.zeros(6, 3, 8), torch.zeros(6, 3, D), torch.zeros(3, 8), seg)
        assert fits == (not isinstance(e.value, NotImplementedError))
        a = _lib.DedfEdgeAttn(type=0, n_edges=6, n_dst=3, heads=3, k=8, d=D, alpha=16, value=16, alpha_dot=16, dst=16, rowptr=16, alpha_stride=24, value_stride=3 * D)
        assert (lib.dedf_edge_attention_scratch_bytes(C.byref(a), 0) > 0) == fits


def test_row_operators_refusals():
    x, y = torch.randn(6, 240), torch.randn(6, 240)
    w, b = torch.ones(112), torch.zeros(64)
    rng = dropout_rng(1, device="cpu")
    bad = [
        (ValueError, (x[:, :239], y, LMAX2), {}), (ValueError, (x, y[:5], LMAX2), {}), (ValueError, (x, y.half(), LMAX2), {}), (TypeError, (x.double(), y.double(), LMAX2), {}),
        (ValueError, (x, y, LMAX2), {"gate": torch.ones(4, 112)}), (ValueError, (x, y, LMAX2), {"gate": torch.ones(6, 111)}), (ValueError, (x, y, LMAX2), {"gate": torch.ones(0, 112)}),
        (TypeError, (x, y, LMAX2), {"gate": torch.ones(6, 112).half()}), (ValueError, (x, y, LMAX2), {"post_weight": w}), (ValueError, (x, y, LMAX2), {"post_bias": b}),
        (ValueError, (x, y, LMAX2), {"post_weight": w[:64], "post_bias": b}), (ValueError, (x, y, LMAX2), {"next_weight": w, "next_bias": b[:63]}),
        (ValueError, (x, y, LMAX2), {"next_weight": w.half(), "next_bias": b}), (ValueError, (x, y, LMAX2), {"dropout": 1.5, "rng": rng}), (ValueError, (x, y, LMAX2), {"dropout": 0.5}),
        (ValueError, (x, y, LMAX2), {"eps": 0.0}), (ValueError, (x, y, "32x1e+64x0e"), {}), (NotImplementedError, (x, y, "240x0o"), {}),
        (NotImplementedError, (torch.zeros(2, 2049), torch.zeros(2, 2049), "2049x0e"), {}), (RuntimeError, (x, y, LMAX2), {"next_weight": w, "next_bias": b}),
    ]
    for err, args, kw in bad:
        with pytest.raises(err):
            norm_gate_residual(*args, **kw)
    for err, args in ((ValueError, (x[:, :9], LMAX2, w, b)), (ValueError, (x, LMAX2, None, None)), (ValueError, (x, LMAX2, w, None)), (RuntimeError, (x, LMAX2, w, b))):
        with pytest.raises(err):
            equivariant_layer_norm(*args)
    for err, args in ((ValueError, (x[:, :9], LMAX2, 0.1, rng)), (ValueError, (x, LMAX2, 1.0, rng)), (ValueError, (x, LMAX2, 0.1, None)), (RuntimeError, (x, LMAX2, 0.1, rng))):
        with pytest.raises(err):
            equivariant_dropout(*args)


def test_c_entries_refuse_before_any_launch(built_lib):
    lib = built_lib

    def attn(**kw):
        base = dict(n_edges=6, n_dst=3, heads=4, k=16, d=60, type=0, n_buckets=0, alpha=16, alpha_stride=64, value=16, value_stride=240, alpha_dot=16, dst=16, rowptr=16)
        a = _lib.DedfEdgeAttn()
        for k, v in {**base, **kw}.items():
            setattr(a, k, v)
        return a

    assert lib.dedf_edge_attention_scratch_bytes(C.byref(attn()), 0) > 0
    V = C.c_void_p
    for rc, kw in ((_lib.ERR_INVALID, dict(n_edges=-1)), (_lib.ERR_INVALID, dict(heads=0)), (_lib.ERR_INVALID, dict(alpha=None)), (_lib.ERR_INVALID, dict(rowptr=None)),
                   (_lib.ERR_INVALID, dict(dropout=1.0, rng=16)), (_lib.ERR_INVALID, dict(dropout=0.5)), (_lib.ERR_INVALID, dict(n_buckets=4)), (_lib.ERR_INVALID, dict(n_dst=0)),
                   (_lib.ERR_INVALID, dict(dropout=float("nan"), rng=16)), (_lib.ERR_INVALID, dict(value_stride=-1)),
                   (_lib.ERR_UNSUPPORTED, dict(type=3)), (_lib.ERR_UNSUPPORTED, dict(heads=17)), (_lib.ERR_UNSUPPORTED, dict(k=65)), (_lib.ERR_UNSUPPORTED, dict(d=257)),
                   (_lib.ERR_UNSUPPORTED, dict(n_edges=1 << 31)), (_lib.ERR_UNSUPPORTED, dict(n_buckets=513, bias_table=16, edge_length=16, bias_boundaries=16))):
        a = attn(**kw)
        assert lib.dedf_edge_attention(C.byref(a), V(16), None, None, None, V(16), 1 << 40, None) == rc, kw
        assert lib.dedf_edge_attention_backward(C.byref(a), V(16), V(16), V(16), None, None, None, None, None, V(16), 1 << 40, None) == rc, kw
        assert lib.dedf_edge_attention_scratch_bytes(C.byref(a), 1) == 0
    a = attn()
    assert lib.dedf_edge_attention(C.byref(a), None, None, None, None, V(16), 1 << 40, None) == _lib.ERR_INVALID
    assert lib.dedf_edge_attention(C.byref(a), V(16), None, None, None, V(16), 8, None) == _lib.ERR_INVALID
    assert lib.dedf_edge_attention(C.byref(a), V(16), None, None, None, V(24), 1 << 40, None) == _lib.ERR_INVALID
    assert lib.dedf_edge_attention(None, V(16), None, None, None, V(16), 1 << 40, None) == _lib.ERR_INVALID
    assert lib.dedf_edge_segments(None, 3, 2, V(16), V(16), V(16), None) == _lib.ERR_INVALID

    def norm(**kw):
        base = dict(type=0, n_rows=6, n_blocks=3, groups=1, mul=(C.c_int * 4)(64, 32, 16, 0), degree=(C.c_int * 4)(0, 1, 2, 0), x=16, y=16, scale=1.0, eps=1e-5)
        a = _lib.DedfNorm()
        for k, v in {**base, **kw}.items():
            setattr(a, k, v)
        return a

    three = lambda *v: (C.c_int * 4)(*v)          # noqa: E731
    for rc, kw in ((_lib.ERR_INVALID, dict(n_rows=-1)), (_lib.ERR_INVALID, dict(x=None)), (_lib.ERR_INVALID, dict(gate=16, groups=4)), (_lib.ERR_INVALID, dict(gate=16, groups=0)),
                   (_lib.ERR_INVALID, dict(eps=0.0)), (_lib.ERR_INVALID, dict(dropout=0.5)), (_lib.ERR_INVALID, dict(post_weight=16)), (_lib.ERR_INVALID, dict(degree=three(1, 1, 2, 0))),
                   (_lib.ERR_INVALID, dict(mul=three(64, 0, 16, 0))), (_lib.ERR_UNSUPPORTED, dict(n_blocks=5)), (_lib.ERR_UNSUPPORTED, dict(type=7)),
                   (_lib.ERR_UNSUPPORTED, dict(mul=three(2048, 1, 1, 0)))):
        a = norm(**kw)
        assert lib.dedf_norm_gate_residual(C.byref(a), V(16), None, None, None) == rc, kw
        assert lib.dedf_norm_gate_residual_backward(C.byref(a), V(16), None, V(16), None, None, None, None, None, None, V(16), 1 << 40, None) == rc, kw
    a = norm()
    assert lib.dedf_norm_gate_residual(C.byref(a), None, None, None, None) == _lib.ERR_INVALID
    assert lib.dedf_norm_gate_residual(C.byref(a), V(16), V(16), None, None) == _lib.ERR_INVALID          # z without next_weight
    assert lib.dedf_norm_gate_residual_backward(C.byref(a), None, None, V(16), None, None, None, None, None, None, V(16), 1 << 40, None) == _lib.ERR_INVALID
    assert lib.dedf_norm_gate_residual_backward(C.byref(a), V(16), None, V(16), None, None, None, None, None, None, V(16), 8, None) == _lib.ERR_INVALID
    mul, degree = three(64, 32, 16, 0), three(0, 1, 2, 0)
    assert lib.dedf_channel_dropout(0, 6, 3, mul, degree, V(16), 1.0, V(16), V(16), None, None) == _lib.ERR_INVALID
    assert lib.dedf_channel_dropout(0, 6, 3, mul, degree, V(16), 0.5, None, V(16), None, None) == _lib.ERR_INVALID
    assert lib.dedf_channel_dropout(9, 6, 3, mul, degree, V(16), 0.5, V(16), V(16), None, None) == _lib.ERR_UNSUPPORTED


def _calls_without_gpu():
    """each operator on its differentiable arguments, with what it takes beside them"""
    seg, rng = _segments_without_gpu(6, 3), dropout_rng(1, device="cpu")
    length, bounds = torch.rand(6), torch.linspace(0, 1, 4)
    attention = lambda a, v, w, l, t: edge_attention(a, v, w, seg, l, length, bounds, t)          # noqa: E731
    norm = lambda x, y, g, w, b, w2, b2: norm_gate_residual(x, y, LMAX2, gate=g, post_weight=w, post_bias=b, next_weight=w2, next_bias=b2)          # noqa: E731
    w, b = torch.ones(112), torch.zeros(64)
    yield attention, (torch.randn(6, 4, 16), torch.randn(6, 4, 60), torch.randn(4, 16), torch.zeros(6), torch.zeros(5, 4))
    yield norm, (torch.randn(6, 240), torch.randn(6, 240), torch.ones(1, 112), w, b, w.clone(), b.clone())
    yield lambda x: equivariant_dropout(x, LMAX2, 0.5, rng), (torch.randn(6, 240),)


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(grad):
    """a dual tensor in any place, with and without gradients wanted: a refusal, not an output without its tangent"""
    for call, args in _calls_without_gpu():
        for i in range(len(args)):
            with torch.autograd.forward_ad.dual_level():
                with_dual = [torch.autograd.forward_ad.make_dual(t.clone(), torch.ones_like(t)) if i == k else t.clone().requires_grad_(grad) for k, t in enumerate(args)]
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*with_dual)
        with pytest.raises(RuntimeError, match="needs GPU tensors"):          # nothing is wrong but the device
            call(*args)


def test_tracing_is_refused():
    for call, args in _calls_without_gpu():
        with pytest.raises(NotImplementedError, match="traced"):
            torch.jit.trace(lambda *a: call(*a), args)


def test_scratch_of_the_norms_at_the_largest_row_count(built_lib):
    """what a workgroup leaves does not depend on the number of rows once there are enough of them, up to 2^31 - 1"""
    def need(n, gates=0):
        a = _lib.DedfNorm(type=1, n_rows=n, n_blocks=1, groups=gates or 1, mul=(C.c_int * 4)(1, 0, 0, 0), degree=(C.c_int * 4)(0, 0, 0, 0), x=16, y=16, gate=16 if gates else None, scale=1.0, eps=1e-5)
        return built_lib.dedf_norm_scratch_bytes(C.byref(a))
    some = need(2 ** 30)
    assert 0 < some < 1 << 20
    assert [need(2 ** 31 - k) for k in (1, 2, 4_095, 4_096, 8_193, 2 ** 20)] == [some] * 6 and need(2 ** 31 - 1, 2 ** 31 - 1) == some


def test_modules_are_the_identity_in_eval_and_carry_the_reference_names():
    m = EquivariantDropout(LMAX2, 0.3).eval()
    x = torch.randn(3, 240)
    assert m(x) is x and not m.state_dict()
    assert set(EdgeAttention(4, 16, 0.1).state_dict()) == {"alpha_dot"} and EdgeAttention(4, 16).alpha_dot.shape == (1, 4, 16)
    assert EdgeAttention(4, 16, bias_boundaries=[1.0, 2.0]).bias_table.shape == (3, 4)
    assert {k: v.shape for k, v in EquivariantLayerNormV2(LMAX2).state_dict().items()} == {"affine_weight": (112,), "affine_bias": (64,)}
    assert set(NormGateResidual(LMAX2, post_norm=False).state_dict()) == {"next_norm.affine_weight", "next_norm.affine_bias"}


MASKED = [lambda **kw: EquivariantDropout(LMAX2, 0.3, **kw), lambda **kw: EdgeAttention(4, 16, 0.1, **kw), lambda **kw: NormGateResidual(LMAX2, drop_prob=0.1, **kw)]


@pytest.mark.parametrize("make", MASKED)
def test_modules_have_masks_of_their_own(make):
    """no seed: one drawn from torch's generator for every instance and every deepcopy; a given one: that, in copies too; casts and moves leave it"""
    torch.manual_seed(3)
    a, b = make(), make()
    torch.manual_seed(3)
    assert make().rng.tolist() == a.rng.tolist() and make().rng.tolist() == b.rng.tolist()
    a.rng[1] = 7
    c, d = copy.deepcopy(a), copy.deepcopy(torch.nn.Sequential(a, b))
    assert len({int(m.rng[0]) for m in (a, b, c, d[0], d[1])}) == 5 and d[0].rng[1] == 7 and type(c) is type(a) and c.training
    assert [(k, v.tolist()) for k, v in c.state_dict().items()] == [(k, v.tolist()) for k, v in a.state_dict().items()]
    assert all(p.data_ptr() != q.data_ptr() for p, q in zip(a.parameters(), c.parameters()))
    for seed in (0, -5, 2 ** 63 - 1):
        e = make(seed=seed)
        e.rng[1] = 4
        assert copy.deepcopy(e).half().double().to_empty(device="cpu").rng.tolist() == [seed, 4]
    with torch.device("meta"):
        f = make(seed=9)
    assert f.to_empty(device="cpu").rng.tolist() == [9, 0] and "rng" not in f.state_dict()


@pytest.mark.parametrize("cast", ["half", "bfloat16", "double", "float"])
def test_bucket_boundaries_survive_casts(cast):
    """boundaries that no 16-bit type holds, two of which lie closer than its steps: the same float32 values after a cast, a move with one, a cast back, and in the
    state dict"""
    bounds = [0.1, 2.1, 19.99, 19.9901]
    m = EdgeAttention(4, 16, bias_boundaries=bounds)
    want = torch.tensor(bounds)
    getattr(m, cast)()
    assert m.alpha_dot.dtype == m.bias_table.dtype == getattr(torch, {"half": "float16", "double": "float64", "float": "float32"}.get(cast, cast))
    assert m.bias_boundaries.dtype == torch.float32 and torch.equal(m.bias_boundaries, want) and torch.equal(m.state_dict()["bias_boundaries"], want)
    net = torch.nn.Sequential(m).to("cpu", torch.float16).float()
    assert torch.equal(net[0].bias_boundaries, want)
    other = EdgeAttention(4, 16, bias_boundaries=[1.0, 2.0, 3.0, 4.0]).half()
    other.load_state_dict(m.state_dict())
    assert torch.equal(other.bias_boundaries, want) and other.bias_boundaries.dtype == torch.float32
    assert EdgeAttention(4, 16).half().bias_boundaries is None


def _ddp_worker(rank, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.distributed.init_process_group("gloo", rank=rank, world_size=2)
    drop = EquivariantDropout(LMAX2, 0.3, seed=11 + rank)
    net = torch.nn.parallel.DistributedDataParallel(torch.nn.Sequential(torch.nn.Linear(240, 240), torch.nn.BatchNorm1d(240), drop).eval())
    for _ in range(2):
        net(torch.ones(3, 240)).sum().backward()
    q.put((rank, drop.rng.tolist()))
    torch.distributed.barrier()
    torch.distributed.destroy_process_group()


def test_data_parallel_ranks_keep_their_seeds():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = torch.multiprocessing.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_ddp_worker, args=(r, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    assert got == {0: [11, 0], 1: [12, 0]}


# ---- edge attention on the GPU ------------------------------------------------------------------------------------------------------------------

def _case(dtype, N, E, H=4, K=16, D=60, buckets=0, logits=True, drop=0.0, seed=0, dst=None):
    g = torch.Generator().manual_seed(seed)
    c = {"N": N, "drop": drop, "rng": (seed + 2 ** 40 + 5, 2 ** 33 + seed)}
    c["dst"] = torch.randint(0, max(N, 1), (E,), generator=g).sort().values if dst is None else dst
    c["alpha"], c["value"] = torch.randn(E, H, K, generator=g).to(dtype), torch.randn(E, H, D, generator=g).to(dtype)
    c["dot"] = torch.randn(H, K, generator=g) * 0.3
    c["logits"] = torch.randn(E, generator=g) * 2 if logits else None
    c["length"] = torch.rand(E, generator=g) * 10 if buckets else None
    c["bounds"] = (torch.linspace(0, 10, buckets + 1)[1:-1].contiguous() if buckets > 1 else None)
    if buckets > 1 and E:
        c["length"][: min(E, buckets - 1)] = c["bounds"][: min(E, buckets - 1)]          # lengths on the borders themselves
    c["table"] = torch.randn(buckets, H, generator=g) if buckets else None
    c["grad"] = torch.randn(N, H, D, generator=g).to(dtype)
    return c


LEAVES = ("alpha", "value", "dot", "logits", "table")


def _gpu(c, train=True):
    """-> out and gradients of the package's operator"""
    d = {k: (None if c[k] is None else c[k].cuda().requires_grad_(train)) for k in LEAVES}
    seg = EdgeSegments(c["dst"].cuda(), c["N"])
    rng = dropout_rng(*c["rng"])
    cu = lambda t: None if t is None else t.cuda()          # noqa: E731
    out = edge_attention(d["alpha"], d["value"], d["dot"], seg, edge_logits=d["logits"], edge_length=cu(c["length"]), bias_boundaries=cu(c["bounds"]), bias_table=d["table"],
                         dropout=c["drop"], rng=rng)
    if not train:
        return out, {}
    leaves = {k: t for k, t in d.items() if t is not None}
    return out, dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), c["grad"].cuda(), allow_unused=True)))


def _reference(c):
    """64-bit out, gradients, and the scale of each gradient's terms (the sums of their absolute values)"""
    E, H, _ = c["alpha"].shape
    d = {k: (None if c[k] is None else c[k].double().requires_grad_(True)) for k in LEAVES}
    mask = O.keep(E, H, 0, c["drop"], *c["rng"]) if c["drop"] else None
    out = O.attention(d["alpha"], d["value"], d["dot"], c["dst"], c["N"], d["logits"], c["length"], c["bounds"], d["table"], mask)
    leaves = {k: t for k, t in d.items() if t is not None}
    up = c["grad"].double()
    if not out.requires_grad:          # no rows or no edges: nothing depends on the inputs
        return out, {k: torch.zeros_like(t) for k, t in leaves.items()}
    grads = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), up, allow_unused=True)))
    return out.detach(), {k: torch.zeros_like(leaves[k]) if g is None else g for k, g in grads.items()}


def _check(c, dtype=None):
    """Roundings of a logit: K terms of act (about 8 operations) and their sum, relative to S = max sum |act w|: ds = (K + 8) u S, which moves a probability
    by 2 ds relative.  A row of n edges is summed with at most n + 8 roundings of its terms, so out is off by (2 ds + (n + 8) u) max|v| m, m the dropout
    factor.  dP and delta are sums of D products: dt is off by p (2 ds + (2 D + n + 16) u) G with G = 2 max sum_c |dout v| m; the leaves' gradients
    are dt times w act' (at most 2.4 |w|), 1, or act, summed over the edges (p sums to one in a row: N rows give at most N terms of scale G)."""
    out, grads = _gpu(c)
    want, ref = _reference(c)
    E, H, K = c["alpha"].shape
    D, N = c["value"].shape[2], c["N"]
    if E == 0 or N == 0:
        close(out, want, 0.0, "out")
        for k, g in grads.items():
            close(g, ref[k], 0.0, k)
        return out, grads
    fin = lambda t: t.double().abs().nan_to_num(0.0, 0.0, 0.0)          # noqa: E731
    S = float((fin(O.act(c["alpha"].double())) * c["dot"].double().abs()).sum(-1).max())
    ds = (K + 8) * U * S
    n = int(torch.bincount(c["dst"], minlength=1).max())
    m = 1.0 / (1.0 - c["drop"])
    vmax, wmax, amax = float(fin(c["value"]).max()), float(c["dot"].abs().max()), float(fin(O.act(c["alpha"].double())).max())
    G = 2 * m * float((fin(c["grad"])[c["dst"]] * fin(c["value"])).sum(-1).max())
    close(out, want, (2 * ds + (n + 8) * U) * vmax * m, "out")
    dt = (2 * ds + (2 * D + n + 16) * U) * G
    tol = {"value": (2 * ds + 16 * U) * m * float(fin(c["grad"]).max()), "alpha": dt * 2.4 * wmax, "logits": H * dt, "dot": N * dt * amax, "table": N * dt}
    for k, g in grads.items():
        close(g, ref[k], tol[k], "d_" + k)
    return out, grads


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,E,kw", [
    (1, 1, {}), (3, 2, {}), (40, 333, dict(buckets=8)), (7, 500, dict(drop=0.3, buckets=3)), (200, 201, dict(logits=False)), (1, 700, dict(drop=0.1)),
    (50, 400, dict(D=40)), (50, 400, dict(D=74, drop=0.2)), (9, 130, dict(H=1, K=1, D=1)), (9, 130, dict(H=3, K=5, D=7, buckets=2)), (9, 130, dict(H=2, K=3, D=6)),
    (9, 130, dict(H=8, K=31, D=51, drop=0.35)), (5, 90, dict(H=16, K=16, D=64, drop=0.5, buckets=1)), (5, 90, dict(H=4, K=64, D=256, buckets=16)), (4, 60, dict(H=1, K=2, D=1023)),
    (4, 60, dict(H=3, K=21, D=85)), (4, 60, dict(H=1, K=256, D=2)), (6, 300, dict(buckets=512)), (6, 300, dict(H=16, K=16, D=64, buckets=128)), (70, 1_000, dict(D=20, K=5)),
])
def test_edge_attention(dtype, N, E, kw):
    _check(_case(dtype, N, E, **kw))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,K,D", [
    (8, 16, 30), (8, 17, 31), (8, 9, 65), (8, 16, 64), (16, 13, 13), (16, 4, 5), (16, 9, 64), (2, 128, 6), (1, 129, 130), (1, 61, 62), (1, 255, 1021), (3, 23, 340), (2, 7, 509),
    (5, 51, 9), (13, 17, 4), (4, 4, 4), (5, 5, 5), (7, 6, 6), (1, 4, 7), (6, 3, 9), (6, 9, 3), (16, 2, 64), (15, 17, 65), (15, 17, 3), (9, 12, 1), (16, 16, 2), (8, 1, 20), (7, 3, 10), (2, 2, 12), (5, 1, 60), (16, 3, 4),
])
def test_edge_attention_heads_of_any_width(dtype, H, K, D):
    """head widths that are no multiples of 4 (each remainder, in features and values), widths below 4, feature rows of up to 16, 32 and 75 quads, value rows of
    up to 64, 128 and 256"""
    _check(_case(dtype, 11, 150, H=H, K=K, D=D, buckets=3, drop=0.15, seed=H * K))


@pytest.mark.gpu
@pytest.mark.parametrize("H,K,D", [(3, 5, 7), (8, 17, 31), (3, 23, 337), (6, 3, 9), (5, 3, 2), (1, 7, 13)])
def test_edge_attention_heads_of_any_width_across_ranges(H, K, D):
    g = torch.Generator().manual_seed(D)
    _check(_case(torch.float32, 3, 9_001, H=H, K=K, D=D, buckets=5, drop=0.0, dst=torch.randint(0, 3, (9_001,), generator=g).sort().values))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [60, 74, 256])
@pytest.mark.parametrize("shift", [0, 1, 17, 63])
def test_edge_attention_rows_at_the_borders_of_ranges(D, shift):
    """ranges are 16 edges here and a workgroup's 64: rows that begin and end at such borders, one before and one behind them, inside one workgroup's edges and over
    several of them, of 9 records and more"""
    n = torch.tensor([shift + 1, 64, 64, 128, 1, 63, 65, 127, 129, 192, 16, 48, 256, 15, 17, 32, 320, 128, 700, 0, 64, 1, 2_000, 63, 1, 130, 62, 16])
    dst = torch.repeat_interleave(torch.arange(len(n)), n)
    _check(_case(torch.float32, len(n), len(dst), D=D, drop=0.1, dst=dst, seed=shift))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,N,E", [(torch.float32, 2_500, 50_003), (torch.float32, 900, 98_304), (torch.float16, 3_000, 65_537), (torch.bfloat16, 40, 70_001)])
def test_edge_attention_ranges_of_several_batches(dtype, N, E):
    """more batches of 16 edges than waves, the last range short"""
    _check(_case(dtype, N, E, H=2, K=4, D=8, drop=0.1, seed=E))


@pytest.mark.gpu
@pytest.mark.parametrize("K", [6, 7, 8])
def test_edge_attention_a_weight_of_minus_infinity(K):
    """positive features and one weight of -inf, also where two quads hold it: logits of -inf, so that head takes no part anywhere and the other is as without it"""
    c = _case(torch.float32, 5, 70, H=2, K=K, D=12, seed=K)
    c["alpha"] = c["alpha"].abs() + 0.1
    want, _ = _gpu(c, train=False)
    for k in range(K):
        dot = c["dot"].clone()
        dot[0, k] = -float("inf")
        out, _ = _gpu(dict(c, dot=dot), train=False)
        assert not out[:, 0].any() and torch.equal(out[:, 1], want[:, 1])


@pytest.mark.gpu
@pytest.mark.parametrize("H,K,D", [(1, 16, 20), (2, 3, 2), (3, 5, 7), (8, 16, 30), (8, 20, 9), (16, 9, 8), (15, 17, 3), (16, 2, 64)])
def test_edge_attention_masks_and_far_logits_with_any_heads(H, K, D):
    """heads that see one and two edges a lane and more: masked edges of NaN and infinities, a bucket that is out for one head alone, logits that lie far apart side
    by side, a NaN that reaches its own row and head only"""
    c = _case(torch.float32, 6, 200, H=H, K=K, D=D, buckets=4, seed=H, drop=0.2)
    dead = (torch.rand(200, generator=torch.Generator().manual_seed(1)) < 0.3) | (c["dst"] == 2) | (c["dst"] == 5)
    c["logits"][dead] = -INF
    clean_out, clean = _check(c)
    c["alpha"][dead], c["value"][dead] = float("nan"), INF
    out, grads = _gpu(c)
    assert torch.equal(out, clean_out) and not out[2].any() and all(torch.equal(grads[k], clean[k]) for k in grads)
    c = _case(torch.float32, 6, 200, H=H, K=K, D=D, buckets=4, seed=4)
    c["table"][1, H - 1] = -INF
    _check(c)
    for gap in (20.0, 30.0, 1e4):
        c = _case(torch.float32, 40, 400, H=H, K=K, D=D, seed=int(gap))
        c["logits"] = c["logits"] - gap * (c["dst"] % 3).float()
        _check(c)
    c = _case(torch.float32, 8, 300, H=H, K=K, D=D, seed=9)
    c["alpha"][int((c["dst"] == 4).nonzero()[3]), H // 2, K - 1] = float("nan")
    bad = _gpu(c)[0].isnan()
    assert bad[4, H // 2].all() and int(bad.sum()) == D


def _masked_rows_beside_far_ones(c, gap, seed):
    """every second row's logits `gap` below its neighbours', runs of up to 20 edges at -inf at most rows' ends, so that a group of edges holds nothing of a row
    but masked edges, beside a row that lies far from it"""
    g = torch.Generator().manual_seed(seed)
    E, dst = len(c["dst"]), c["dst"]
    c["logits"] = c["logits"] - gap * (dst % 2).float()
    first = torch.searchsorted(dst, torch.arange(c["N"] + 1))
    for n in range(c["N"]):
        a, b = int(first[n]), int(first[n + 1])
        for front in (True, False):
            run = min(int(torch.randint(0, 21, (1,), generator=g)), max(b - a - 1, 0))
            if front:
                c["logits"][a:a + run] = -INF
            else:
                c["logits"][max(b - run, a):b] = -INF
        if n % 7 == 3:
            c["logits"][a:b] = -INF
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [60.0, 95.0, 120.0, 1e4])
@pytest.mark.parametrize("H,K,D", [(1, 16, 20), (4, 16, 60), (3, 5, 7), (8, 16, 30), (16, 16, 8), (16, 9, 8), (15, 17, 3)])
def test_edge_attention_masked_edges_beside_far_rows(H, K, D, gap):
    """a row keeps its weight and gradients where its only edges in a group of 16, 8 or 4 are masked ones, in all heads or in one, next to a row whose logits lie
    far above or below"""
    g = torch.Generator().manual_seed(int(gap) + H)
    n = torch.randint(3, 60, (24,), generator=g)
    n[5] = 0
    c = _case(torch.float32, 24, int(n.sum()), H=H, K=K, D=D, buckets=4, dst=torch.repeat_interleave(torch.arange(24), n), drop=0.1, seed=int(gap))
    _check(_masked_rows_beside_far_ones(c, gap, H))
    c = _case(torch.float32, 24, int(n.sum()), H=H, K=K, D=D, buckets=4, dst=c["dst"], seed=int(gap) + 1)
    c["table"][1, H // 2] = -INF          # out for one head
    c["length"] = torch.where(_masked_rows_beside_far_ones(dict(c, logits=torch.zeros(len(c["dst"]))), 0.0, H)["logits"] == -INF, torch.full_like(c["length"], 3.0), c["length"])
    c["logits"] = c["logits"] - gap * (c["dst"] % 2).float()
    _check(c)


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [95.0, 1e4])
def test_edge_attention_masked_edges_beside_far_rows_across_ranges(gap):
    """the same with several batches a wave, and with records of rows that cross ranges"""
    g = torch.Generator().manual_seed(int(gap))
    for N, E in ((40, 9_001), (900, 70_003)):
        c = _case(torch.float32, N, E, H=2, K=4, D=8, buckets=3, dst=torch.randint(0, N, (E,), generator=g).sort().values, seed=N)
        _check(_masked_rows_beside_far_ones(c, gap, N))


@pytest.mark.gpu
@pytest.mark.parametrize("H,K,D", [(8, 17, 31), (3, 5, 7), (6, 3, 9)])
def test_edge_attention_columns_at_an_odd_element(H, K, D):
    """value as columns of a wider tensor with NaN around them, at an odd element: the same bits, and a gradient of those columns alone"""
    c = _case(torch.float32, 5, 70, H=H, K=K, D=D, seed=2, drop=0.0)
    want, ref = _gpu(c)
    a, v, seg = c["alpha"].cuda(), c["value"].cuda(), EdgeSegments(c["dst"].cuda(), 5)
    wide = torch.full((70, 3 + H * D + 2), float("nan"), device="cuda")
    wide[:, 3:3 + H * D] = v.reshape(70, H * D)
    wide.requires_grad_(True)
    out = edge_attention(a, wide[:, 3:3 + H * D].view(70, H, D), c["dot"].cuda(), seg, edge_logits=c["logits"].cuda())
    assert torch.equal(out, want)
    g, = torch.autograd.grad(out, wide, c["grad"].cuda())
    assert torch.equal(g[:, 3:3 + H * D].reshape(70, H, D), ref["value"]) and not g[:, :3].any() and not g[:, 3 + H * D:].any()


@pytest.mark.gpu
def test_edge_attention_without_edges_or_rows():
    for N, E in ((0, 0), (5, 0)):
        out, grads = _check(_case(torch.float32, N, E, buckets=4, drop=0.1))
        assert out.shape == (N, 4, 60) and all(float(g.abs().sum()) == 0.0 for g in grads.values())


@pytest.mark.gpu
@pytest.mark.parametrize("N,E", [(1, 5_000), (3, 60_001), (2_000, 2_500)])
def test_edge_attention_rows_across_ranges(N, E):
    """rows far longer than a wave's range of edges, and far more rows than edges (most of them empty), the first and the last row empty among them"""
    g = torch.Generator().manual_seed(E)
    dst = (torch.randint(0, N, (E,), generator=g) if N < 100 else 1 + torch.randint(0, N // 3, (E,), generator=g)).sort().values
    _check(_case(torch.float32, N, E, H=2, K=4, D=8, buckets=5, dst=dst, drop=0.0))


@pytest.mark.gpu
def test_edge_attention_masked_edges_take_no_part():
    """an edge logit or a bucket's bias of -inf: neither probabilities nor NaN or infinities in alpha and value of such an edge reach anything; a row of masked
    edges only is zero, and so are its gradients"""
    for dtype in TYPES:
        c = _case(dtype, 6, 200, buckets=4, seed=3, drop=0.2)
        dead = torch.rand(200, generator=torch.Generator().manual_seed(1)) < 0.3
        dead |= (c["dst"] == 2) | (c["dst"] == 5)
        c["logits"][dead] = -INF
        clean_out, clean = _gpu(c)
        _check(c)
        c["alpha"][dead], c["value"][dead] = float("nan"), INF
        out, grads = _gpu(c)
        assert torch.equal(out, clean_out) and not out[2].any() and not out[5].any()
        for k in grads:
            assert torch.equal(grads[k], clean[k]), k
        assert not grads["alpha"][dead.cuda()].any() and not grads["value"][dead.cuda()].any() and not grads["logits"][dead.cuda()].any()
    c = _case(torch.float32, 6, 200, buckets=4, seed=4)
    c["table"][1] = -INF          # a whole bucket out
    c["table"][2, 3] = -INF       # a bucket out for one head
    _check(c)


@pytest.mark.gpu
@pytest.mark.parametrize("lowest", [-65504.0, -1e4, torch.finfo(torch.bfloat16).min, torch.finfo(torch.float32).min])
def test_edge_attention_lowest_finite_masks(lowest):
    """masks of a type's lowest value: in a mixed row such edges get nothing; in a row of them alone the 64-bit formula decides (float32's lowest swallows the
    scores: equal shares; float16's does not)"""
    c = _case(torch.float32, 5, 150, seed=7)
    c["logits"][:] = 0.0
    c["logits"][torch.rand(150, generator=torch.Generator().manual_seed(2)) < 0.4] = lowest
    c["logits"][c["dst"] == 3] = lowest
    _check(c)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,K,D", [(1, 16, 20), (4, 16, 60), (3, 5, 7), (8, 16, 30), (16, 16, 8), (16, 9, 8), (15, 17, 3)])
def test_edge_attention_lowest_masks_in_logits_and_bias(dtype, H, K, D):
    """edge logits and a bucket's bias at float32's lowest value at once: their sum is finite in 64 bits alone.  Such edges get nothing beside others and equal shares
    among themselves: one group of 16 edges inside a row, a row that is masked as a whole, single edges, the last batch, one head alone.  The largest values in
    both places: such edges share their row alone"""
    n = torch.tensor([48, 37, 3, 20, 16, 29])          # 153 edges: a last batch of 9
    dst = torch.repeat_interleave(torch.arange(6), n)
    for low, heads in ((-FMAX, slice(None)), (-FMAX, slice(H - 1, H)), (FMAX, slice(None)), (FMAX, slice(0, 1))):
        c = _case(dtype, 6, len(dst), H=H, K=K, D=D, buckets=4, dst=dst, seed=H + K)
        dead = torch.zeros(len(dst), dtype=torch.bool)
        dead[16:32] = dead[48:85] = dead[90:92] = dead[144:] = True
        c["length"] = torch.where(dead, torch.full_like(c["length"], 3.0), torch.where(c["length"] < 5, c["length"] / 2.5, c["length"]))          # (bucket 1: 2.5 to 5)
        c["table"][1, heads] = low
        c["logits"][dead] = low
        _check(c)


@pytest.mark.gpu
def test_edge_attention_lowest_masks_in_logits_and_bias_across_ranges():
    """the same where a wave walks several groups, rows cross ranges, and workgroups leave one record"""
    low, E = -FMAX, 70_003
    g = torch.Generator().manual_seed(5)
    for N in (3, 900):
        c = _case(torch.float32, N, E, H=2, K=4, D=8, buckets=4, dst=torch.randint(0, N, (E,), generator=g).sort().values, seed=N)
        dead = (torch.arange(E) // 32 % 3 == 1) | (c["dst"] == 1)
        dead[-7:] = True
        c["length"] = torch.where(dead, torch.full_like(c["length"], 3.0), torch.where(c["length"] < 5, c["length"] / 2.5, c["length"]))
        c["table"][1] = low
        c["logits"][dead] = low
        _check(c)


@pytest.mark.gpu
def test_edge_attention_nan_reaches_its_own_rows_only():
    c = _case(torch.float32, 8, 300, seed=9)
    e = int((c["dst"] == 4).nonzero()[3])
    c["alpha"][e, 1, 2] = float("nan")
    out, _ = _gpu(c)
    bad = out.isnan()
    assert bad[4, 1].all() and int(bad.sum()) == 60
    c = _case(torch.float32, 8, 300, seed=9)
    c["logits"][e] = INF
    out, _ = _gpu(c)
    assert out[4].isnan().all() and not out[[0, 1, 2, 3, 5, 6, 7]].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_edge_attention_views(dtype):
    """alpha and value as columns of one wide tensor, at an odd offset, of every second edge, broadcast over the edges, heads transposed; gradients of a
    shared value"""
    c = _case(dtype, 11, 150, D=20, seed=5, drop=0.1)
    want, ref = _gpu(c)
    seg, rng = EdgeSegments(c["dst"].cuda(), 11), dropout_rng(*c["rng"])
    call = lambda a, v: edge_attention(a, v, c["dot"].cuda(), seg, edge_logits=c["logits"].cuda(), dropout=0.1, rng=rng)          # noqa: E731
    a, v = c["alpha"].cuda(), c["value"].cuda()
    for offset in (0, 1, 4):
        wide = torch.full((150, offset + 64 + 80 + 3), float("nan"), dtype=dtype, device="cuda")
        wide[:, offset:offset + 64], wide[:, offset + 64:offset + 144] = a.reshape(150, 64), v.reshape(150, 80)
        assert torch.equal(call(wide[:, offset:offset + 64].view(150, 4, 16), wide[:, offset + 64:offset + 144].view(150, 4, 20)), want)
    double = torch.stack([v, v.flip(0)], 1).reshape(300, 4, 20)
    assert torch.equal(call(a, double[::2]), want)
    assert torch.equal(call(a.transpose(1, 2).contiguous().transpose(1, 2), v.transpose(0, 1).contiguous().transpose(0, 1)), want)
    one = v[:1].clone().requires_grad_(True)
    out = call(a, one.expand(150, 4, 20))
    c2 = dict(c, value=c["value"][:1].expand(150, 4, 20).contiguous())
    w2, r2 = _gpu(c2)
    assert torch.equal(out, w2)
    g, = torch.autograd.grad(out, one, c["grad"].cuda())
    total = r2["value"].double().sum(0, keepdim=True).cpu()
    # (150 rounded terms are summed in `dtype` by autograd's own expand: half a step of the running sum each)
    close(g, total, 150 * half_step(dtype) * float(r2["value"].double().abs().sum(0).max()), "d_one")


@pytest.mark.gpu
def test_edge_attention_offsets_past_32_bits():
    """more than 2^31 value elements: the last edges' rows lie behind what 32-bit element offsets reach"""
    E, D = 2_200_000, 1024
    value = torch.zeros(E, 1, D, dtype=torch.float16, device="cuda")
    assert E * D > 2 ** 31
    dst = torch.zeros(E, dtype=torch.int64, device="cuda")
    dst[-5:] = torch.tensor([1, 1, 2, 2, 2], device="cuda")
    value[-5:] = torch.arange(1, 6, device="cuda", dtype=torch.float16)[:, None, None]
    value.requires_grad_(True)
    alpha = torch.zeros(E, 1, 1, dtype=torch.float16, device="cuda")
    out = edge_attention(alpha, value, torch.ones(1, 1, device="cuda"), EdgeSegments(dst, 3))
    assert torch.equal(out[:, 0, 0].cpu(), torch.tensor([0.0, 1.5, 4.0], dtype=torch.float16)) and bool((out == out[:, :, :1]).all())
    g, = torch.autograd.grad(out, value, torch.ones_like(out))
    assert torch.equal(g[-5:, 0, 7].cpu(), torch.tensor([0.5, 0.5, 1 / 3, 1 / 3, 1 / 3]).half())


@pytest.mark.gpu
def test_edge_attention_edges_up_to_the_limit():
    """2^31 - 1 edges, nearly all of them of one row: every one has its equal share, and the last ones, a row of their own, theirs"""
    E = 2 ** 31 - 1
    dst = torch.zeros(E, dtype=torch.int64, device="cuda")
    dst[-5:] = 1
    seg = EdgeSegments(dst, 2)
    del dst
    value = torch.ones(E, 1, 1, dtype=torch.bfloat16, device="cuda")
    value[-5:, 0, 0] = torch.arange(1, 6, device="cuda").bfloat16()
    value.requires_grad_(True)
    alpha = torch.zeros(1, 1, 1, dtype=torch.bfloat16, device="cuda").expand(E, 1, 1)
    out = edge_attention(alpha, value, torch.ones(1, 1, device="cuda"), seg)
    # the sums of 2^31 ones: a range's 2^19 or so are whole numbers in float32, some thousand records are joined with one rounding each
    close(out[:, 0, 0], torch.tensor([1.0, 3.0], dtype=torch.float64), 4_100 * U, "out")
    g, = torch.autograd.grad(out, value, torch.ones_like(out))
    close(g[-5:, 0, 0], torch.full((5,), 0.2, dtype=torch.float64), 8 * U, "d_value")
    share = g[:-5, 0, 0]
    assert bool((share == share[0]).all())
    close(share[:1] * 2.0 ** 31, torch.full((1,), 2.0 ** 31 / (E - 5), dtype=torch.float64), 4_100 * U, "share")


@pytest.mark.gpu
@pytest.mark.parametrize("N,H", [(67_200_000, 4), (2 ** 31 - 2, 1)])
def test_edge_attention_rows_up_to_the_limit(N, H):
    """more rows and heads than a launch has threads for at 16 each, and as many rows as there may be, nearly all of them empty"""
    dst = torch.tensor([0, 0, N // 2, N - 257, N - 1, N - 1, N - 1], device="cuda")
    value = torch.arange(1, 8, dtype=torch.float16, device="cuda")[:, None, None].expand(7, H, 1).contiguous().requires_grad_(True)
    logits = torch.zeros(7, device="cuda", requires_grad=True)
    out = edge_attention(torch.zeros(7, H, 1, dtype=torch.float16, device="cuda"), value, torch.ones(H, 1, device="cuda"), EdgeSegments(dst, N), edge_logits=logits)
    want = {0: 1.5, N // 2: 3.0, N - 257: 4.0, N - 1: 6.0}
    o = out.detach()
    assert {r: float(o[r, H - 1, 0]) for r in want} == want and int(o.count_nonzero()) == 4 * H and float(o.sum(dtype=torch.float64)) == 14.5 * H
    up = torch.ones_like(out)
    dv, dl = torch.autograd.grad(out, [value, logits], up)
    half = torch.tensor([0.5, 0.5, 1, 1, 1 / 3, 1 / 3, 1 / 3], dtype=torch.float64)
    close(dv[:, H - 1, 0], half, 4 * U, "d_value")
    # dt = p (v - out): 16 roundings of terms up to 7
    close(dl, H * half * (torch.arange(1.0, 8.0, dtype=torch.float64) - torch.tensor([1.5, 1.5, 3, 4, 6, 6, 6], dtype=torch.float64)), 16 * 7 * H * U, "d_logits")


@pytest.mark.gpu
def test_edge_attention_repeats_bit_for_bit_and_draws_by_the_offset():
    c = _case(torch.float32, 300, 5_000, buckets=8, drop=0.25, seed=1)
    out, grads = _gpu(c)
    for _ in range(3):
        o, g = _gpu(c)
        assert torch.equal(o, out) and all(torch.equal(g[k], grads[k]) for k in g)
    other, _ = _gpu(dict(c, rng=(c["rng"][0], c["rng"][1] + 1)))
    assert not torch.equal(other, out)


@pytest.mark.gpu
def test_edge_attention_gradients_against_differences():
    """central differences of the 64-bit forward pass along random directions: <gradient, direction> to 1e-4 of |gradient| |direction| / sqrt(n), the scale of
    such a product (the gradients are float32's, 1e-5 off at most; the differences' own error is h^2 = 1e-8)"""
    c = _case(torch.float32, 20, 300, buckets=6, drop=0.15, seed=21)
    _, grads = _gpu(c)
    mask = O.keep(300, 4, 0, c["drop"], *c["rng"])

    def loss(d):
        return float((O.attention(d["alpha"], d["value"], d["dot"], c["dst"], 20, d["logits"], c["length"], c["bounds"], d["table"], mask) * c["grad"].double()).sum())

    base = {k: c[k].double() for k in LEAVES}
    g = torch.Generator().manual_seed(0)
    for k in LEAVES:
        direction = torch.randn(base[k].shape, generator=g, dtype=torch.float64)
        h = 1e-4
        slope = (loss({**base, k: base[k] + h * direction}) - loss({**base, k: base[k] - h * direction})) / (2 * h)
        got = float((grads[k].double().cpu() * direction).sum())
        assert abs(got - slope) <= 1e-4 * float(grads[k].double().norm().cpu()), (k, got, slope)


@pytest.mark.gpu
def test_edge_segments_refuses_bad_lists():
    for bad in ([0, 2, 1], [0, 1, 3], [-1, 0, 1], [2, 1, 0]):
        with pytest.raises(ValueError):
            EdgeSegments(torch.tensor(bad, device="cuda"), 3)
    s = EdgeSegments(torch.tensor([1, 1, 4], device="cuda"), 6)
    assert s.rowptr.tolist() == [0, 0, 2, 2, 2, 3, 3] and s.dst.tolist() == [1, 1, 4] and len(s) == 3
    a = torch.zeros(3, 4, 16, device="cuda")
    with pytest.raises(ValueError):          # the rng is somewhere else
        edge_attention(a, torch.zeros(3, 4, 8, device="cuda"), torch.zeros(4, 16, device="cuda"), s, dropout=0.1, rng=dropout_rng(0, device="cpu"))
    with pytest.raises(ValueError):
        edge_attention(a, torch.zeros(3, 4, 8, device="cuda"), torch.zeros(4, 16), s)


@pytest.mark.gpu
def test_no_second_derivatives():
    c = _case(torch.float32, 3, 20)
    v = c["value"].cuda().requires_grad_(True)
    out = edge_attention(c["alpha"].cuda(), v, c["dot"].cuda().requires_grad_(True), EdgeSegments(c["dst"].cuda(), 3))
    g, = torch.autograd.grad(out.square().sum(), v, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ---- norms and dropout on the GPU -----------------------------------------------------------------------------------------------------------------

IRREPS = [LMAX2, "64x0e+32x1e+16x2e+8x3e", "64x0e+32x1e", "192x0e+96x1e+48x2e", "5x0e+3x1e+1x2e", "1x0e", "7x1e+2x3e", "513x0e", "500x0e+300x1e+128x2e", "4x0e+4x1e+4x2e+4x7e", "3x2e"]


def _norm_case(dtype, irreps, R, groups=0, post=True, nxt=True, drop=0.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    blocks = parse_irreps(irreps)
    sh = row_shape(irreps)
    c = {"irreps": irreps, "blocks": blocks, "drop": drop, "rng": (seed + 77, 3 + 2 ** 35), "scale": 0.7}
    c["x"], c["y"] = (torch.randn(R, sh.width, generator=g) + 0.3).to(dtype), (torch.randn(R, sh.width, generator=g) * 1.5 - 0.2).to(dtype)
    c["gate"] = (0.5 + 0.3 * torch.randn(groups, sh.channels, generator=g)).to(torch.float32 if groups == 1 else dtype) if groups else None
    for k, on in (("post", post), ("next", nxt)):
        c[k + "_weight"] = 1 + 0.2 * torch.randn(sh.channels, generator=g) if on else None
        c[k + "_bias"] = 0.2 * torch.randn(sh.scalars, generator=g) if on and sh.scalars else None
    c["dh"], c["dz"] = torch.randn(R, sh.width, generator=g).to(dtype), (torch.randn(R, sh.width, generator=g).to(dtype) if nxt else None)
    return c


NORM_LEAVES = ("x", "y", "gate", "post_weight", "post_bias", "next_weight", "next_bias")


def _norm_gpu(c, use=("h", "z")):
    d = {k: None if c[k] is None else c[k].cuda().requires_grad_(True) for k in NORM_LEAVES}
    rng = dropout_rng(*c["rng"])
    h, z = norm_gate_residual(d["x"], d["y"], c["irreps"], scale=c["scale"], gate=d["gate"], post_weight=d["post_weight"], post_bias=d["post_bias"], dropout=c["drop"], rng=rng,
                              next_weight=d["next_weight"], next_bias=d["next_bias"])
    outs = [(o, c[g].cuda()) for n, o, g in (("h", h, "dh"), ("z", z, "dz")) if o is not None and n in use]
    leaves = {k: t for k, t in d.items() if t is not None}
    return h, z, dict(zip(leaves, torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [g for _, g in outs], allow_unused=True)))


def _norm_reference(c, use=("h", "z")):
    d = {k: None if c[k] is None else c[k].double().requires_grad_(True) for k in NORM_LEAVES}
    mask = O.keep(len(c["x"]), row_shape(c["irreps"]).channels, 1 << 16, c["drop"], *c["rng"]) if c["drop"] else None
    pair = lambda k: None if d[k + "_weight"] is None else (d[k + "_weight"], d[k + "_bias"])          # noqa: E731
    h, z = O.norm_gate_residual(d["x"], d["y"], c["blocks"], c["scale"], d["gate"], pair("post"), mask, pair("next"))
    outs = [(o, c[g].double()) for n, o, g in (("h", h, "dh"), ("z", z, "dz")) if o is not None and n in use]
    leaves = {k: t for k, t in d.items() if t is not None}
    grads = dict(zip(leaves, torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [g for _, g in outs], allow_unused=True)))
    return h, z, grads


def _norm_check(c, use=("h", "z")):
    """A norm of W components: mean and mean square are sums of W terms, each value then has about W + 16 roundings of terms of its own scale (values of a
    few units times r); r is at most 1 / sqrt(smallest mean square + eps), which the cases keep at L.  So a value is off by (W + 16) u L M, M the largest value.
    Both norms and their backward passes follow each other: 4 times that through each, and the gate, weights (at most 2) and scale between them.
    Parameter gradients sum R rows (and 2l+1 components)."""
    h, z, grads = _norm_gpu(c, use)
    wh, wz, ref = _norm_reference(c, use)
    W, R = c["x"].shape[1], len(c["x"])
    f32 = lambda t: None if t is None else t.detach().double()          # noqa: E731
    M = 1.0 + max(float(t.abs().max()) for t in map(f32, (c["x"], c["y"], wh, wz, c["dh"])) if t is not None)
    small = 1.0
    for t, on in ((c["y"], c["post_weight"] is not None), (f32(wh), c["next_weight"] is not None)):
        at = 0
        for m, l in c["blocks"] if on else ():
            b = t.double()[:, at:at + m * (2 * l + 1)]
            at += m * (2 * l + 1)
            b = b - b.mean(1, keepdim=True) if l == 0 else b
            small = min(small, float((b.square().mean(1) + 1e-5).min()))
    L = small ** -0.5
    one = (W + 16) * U * L * M * 2 / (1 - c["drop"])
    close(h, f32(wh), 2 * one, "h")
    if z is not None:
        close(z, f32(wz), 4 * one * L, "z")
    for k, g in grads.items():
        if ref[k] is None:
            assert g is None or not g.any(), k
            continue
        many = {"x": 1, "y": L, "gate": 7 * R / (1 if c["gate"] is None else len(c["gate"]))}.get(k, 15 * R)
        close(g, ref[k], 16 * one * L * M * many, "d_" + k)
    return h, z, grads


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("irreps", IRREPS)
def test_norm_gate_residual(dtype, irreps):
    _norm_check(_norm_case(dtype, irreps, 12, groups=3, drop=0.3, seed=len(irreps)))


@pytest.mark.gpu
@pytest.mark.parametrize("R,kw,use", [
    (1, dict(), ("h", "z")), (5, dict(groups=1), ("h", "z")), (5, dict(groups=5), ("h", "z")), (206, dict(groups=2, drop=0.1), ("h", "z")), (700, dict(groups=1, drop=0.1), ("h", "z")),
    (9, dict(post=False, groups=3), ("h", "z")), (9, dict(nxt=False, groups=9), ("h",)), (9, dict(post=False, nxt=False), ("h",)), (9, dict(), ("h",)), (9, dict(groups=1), ("z",)),
])
def test_norm_gate_residual_forms(R, kw, use):
    _norm_check(_norm_case(torch.float32, LMAX2, R, **kw), use)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,groups", [(30, 1), (30, 30), (30, 5), (9_000, 2), (9_000, 90)])
def test_norm_gate_types(dtype, R, groups):
    """a gate in the features' type and in float32, of one row, of groups cut into many and into few slices, one a node; small rows keep the oracle quick"""
    for gate_type in (dtype, torch.float32):
        c = _norm_case(dtype, "5x0e+3x1e+1x2e", R, groups=groups, drop=0.0, seed=groups)
        c["gate"] = c["gate"].to(gate_type)
        h, z, grads = _norm_gpu(c)
        _, _, ref = _norm_reference(c)
        assert grads["gate"].dtype == gate_type
        # a sum of n = 5 R / groups products of values of a few units: float32 chains of at most 64 terms, 64 bits after, as in the test of many rows below
        want = ref["gate"]
        close(grads["gate"], want, 64 * 16 * U * float(want.abs().max()), "d_gate")


@pytest.mark.gpu
def test_edge_attention_far_logits_side_by_side():
    """rows whose logits lie 100 and 10 000 apart next to each other, and float32 values of 1e-20: every row keeps its own precision"""
    for gap in (20.0, 30.0, 100.0, 1e4):
        c = _case(torch.float32, 40, 400, seed=int(gap))
        c["logits"] = c["logits"] - gap * (c["dst"] % 3).float()
        _check(c)
        c["value"] *= 1e-20
        c["grad"] *= 1e20
        _check(c)


@pytest.mark.gpu
def test_norm_backward_over_many_rows_against_the_formula():
    """more rows than waves: every wave sums several rows, slices of a pose's rows are joined; float32 parameters' gradients against 64 bits"""
    for groups in (0, 1, 50, 10_300):
        c = _norm_case(torch.float32, LMAX2, 10_300, groups=groups, drop=0.0, seed=groups)
        _, _, grads = _norm_gpu(c)
        _, _, ref = _norm_reference(c)
        for k, g in grads.items():
            # sums of n = 10 300 x 5 terms at most, float32 within a workgroup, 64 bits after: relative to the root sum of squares of random terms, n u would be
            # the worst order's bound; the longest float32 chain is (rows of a wave, at most 4) + 4 waves + 5 components
            scale = float(ref[k].abs().max())
            assert float((g.double().cpu() - ref[k]).abs().max()) <= 64 * 16 * U * scale, (groups, k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("irreps", [LMAX2, "5x0e+3x1e+1x2e", "192x0e+96x1e+48x2e"])
def test_equivariant_layer_norm(dtype, irreps):
    c = _norm_case(dtype, irreps, 11, seed=2)
    m = EquivariantLayerNormV2(irreps).cuda()
    with torch.no_grad():
        m.affine_weight.copy_(c["next_weight"])
        m.affine_bias.copy_(c["next_bias"])
    x = c["x"].cuda().requires_grad_(True)
    z = m(x)
    g = torch.autograd.grad(z, [x, m.affine_weight, m.affine_bias], c["dz"].cuda())
    xr, w, b = (t.double().requires_grad_(True) for t in (c["x"], c["next_weight"], c["next_bias"]))
    wz = O.layer_norm(xr, c["blocks"], w, b, 1e-5)
    ref = torch.autograd.grad(wz, [xr, w, b], c["dz"].double())
    W = x.shape[1]
    # 1x2e alone: a mean square over 5 values can be small, its root's inverse L is measured; else as in _norm_check
    L = 10.0
    close(z, wz, (W + 16) * U * L * 8, "z")
    for k, got, want, n in zip(("x", "weight", "bias"), g, ref, (L, 55, 11)):
        close(got, want, (W + 16) * U * L * 8 * 4 * n, "d_" + k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("irreps", IRREPS)
def test_equivariant_dropout(dtype, irreps):
    """kept values are x / (1 - p): one float32 product with a rounded factor (2 u) and the type's rounding; dropped ones are zero, NaN and infinities too"""
    sh, p, key = row_shape(irreps), 0.4, (2 ** 50 + 9, 2 ** 40 + 1)
    g = torch.Generator().manual_seed(8)
    x, up = torch.randn(13, sh.width, generator=g).to(dtype), torch.randn(13, sh.width, generator=g).to(dtype)
    mask = O.per_channel(O.keep(13, sh.channels, 1 << 16, p, *key), parse_irreps(irreps))
    leaf = x.cuda().requires_grad_(True)
    out = equivariant_dropout(leaf, irreps, p, dropout_rng(*key))
    close(out, x.double() * mask, 2 * U * float(x.double().abs().max()) * 2, "out")
    got, = torch.autograd.grad(out, leaf, up.cuda())
    close(got, up.double() * mask, 2 * U * float(up.double().abs().max()) * 2, "d_x")
    x[mask == 0] = float("nan")
    assert torch.equal(equivariant_dropout(x.cuda(), irreps, p, dropout_rng(*key)), out)
    same = x.cuda()
    assert equivariant_dropout(same, irreps, 0.0) is same


@pytest.mark.gpu
def test_dropout_inside_the_residual_is_the_dropout_beside_it():
    """dropout fused into norm_gate_residual draws what equivariant_dropout draws"""
    c = _norm_case(torch.float32, LMAX2, 40, post=False, nxt=False, drop=0.3)
    h, _, _ = _norm_gpu(c, ("h",))
    dropped = equivariant_dropout(c["y"].cuda(), LMAX2, 0.3, dropout_rng(*c["rng"]))
    close(h, (c["x"].double() + c["scale"] * dropped.double().cpu()), 4 * U * float(h.detach().abs().max()) + 4 * U * float(dropped.abs().max()), "h")


@pytest.mark.gpu
def test_dropout_rate_and_independence():
    """3 296 000 channels at p = 0.1: the share dropped within 6 standard deviations, 6 sqrt(p (1 - p) / n) = 1e-3; neighbouring offsets and rows agree as
    often as independent draws would"""
    x = torch.ones(103_000, 32, device="cuda")
    a = equivariant_dropout(x, "32x0e", 0.1, dropout_rng(7, 0)) == 0
    b = equivariant_dropout(x, "32x0e", 0.1, dropout_rng(7, 1)) == 0
    for share, want in ((a, 0.1), (b, 0.1), (a & b, 0.01), (a[1:] & a[:-1], 0.01), (a[:, 1:] & a[:, :-1], 0.01)):
        assert abs(float(share.double().mean()) - want) <= 6 * math.sqrt(want * (1 - want) / share.numel())


@pytest.mark.gpu
def test_stacked_modules_drop_different_places():
    """two layers of a network made with the defaults, and copies of one, drop independent channels and edges: both drop one of n places with probability p^2"""
    x, p = torch.ones(4_000, 240, device="cuda"), 0.5
    first = EquivariantDropout(LMAX2, p).cuda()
    layers = [first, EquivariantDropout(LMAX2, p).cuda(), copy.deepcopy(first)]
    dropped = [m(x)[:, :64] == 0 for m in layers]
    residual = [NormGateResidual(LMAX2, post_norm=False, next_norm=False, drop_prob=p).cuda() for _ in range(2)]
    dropped += [m(torch.zeros_like(x), x)[0][:, :64] == 0 for m in residual]
    seg, alpha, value = EdgeSegments(torch.arange(64_000, device="cuda"), 64_000), torch.zeros(64_000, 4, 16, device="cuda"), torch.ones(64_000, 4, 4, device="cuda")
    edges = [EdgeAttention(4, 16, p).cuda()(alpha, value, seg)[:, :, 0].reshape(4_000, 64) == 0 for _ in range(2)]
    n = 4_000 * 64
    for group in (dropped, edges):
        for i, a in enumerate(group):
            for b in group[:i]:
                assert abs(float((a & b).sum()) / n - 0.25) < 6 * (0.25 * 0.75 / n) ** 0.5


@pytest.mark.gpu
def test_row_operators_at_the_largest_row_count():
    """2^31 - 1 rows of one channel: every row is written and read once, with a gate a row and with none; small whole numbers, so nothing rounds"""
    R = 2 ** 31 - 1
    rows = lambda n: torch.arange(n, dtype=torch.float16, device="cuda").repeat(R // n + 1)[:R, None]          # noqa: E731
    x, y, up = rows(11), rows(7), rows(3)
    gate = 1 + rows(5)
    leaves = [t.requires_grad_(True) for t in (x, y, gate)]
    h, _ = norm_gate_residual(x, y, "1x0e", scale=0.5, gate=gate)
    dx, dy, dg = torch.autograd.grad(h, leaves, up)
    with torch.no_grad():
        assert torch.equal(h, x + 0.5 * gate * y)
        del h
        assert torch.equal(dx, up) and torch.equal(dy, 0.5 * gate * up) and torch.equal(dg, 0.5 * y * up)
        del dx, dy, dg, gate, leaves
    h, _ = norm_gate_residual(x, y, "1x0e", scale=0.5)
    dx, dy = torch.autograd.grad(h, [x, y], up)
    with torch.no_grad():
        assert torch.equal(h, x + 0.5 * y) and torch.equal(dx, up) and torch.equal(dy, 0.5 * up)
        del h, dx, dy
        one = torch.ones(R, 1, dtype=torch.float16, device="cuda")
        out = equivariant_dropout(one, "1x0e", 0.5, dropout_rng(5, 9))
        assert bool(((out == 0) | (out == 2)).all()) and abs(float(out.sum(dtype=torch.float64)) / R - 1.0) < 6 * R ** -0.5          # (variance 1 a row)
        for r in [*range(40), *range(R - 40, R)]:
            assert float(out[r, 0]) == (2.0 if O.philox((r, 65536, 9, 0), (5, 0))[0] >= 2 ** 31 else 0.0), r


@pytest.mark.gpu
def test_row_operators_without_rows():
    x = torch.zeros(0, 240, device="cuda", requires_grad=True)
    w, b = torch.ones(112, device="cuda", requires_grad=True), torch.zeros(64, device="cuda", requires_grad=True)
    h, z = norm_gate_residual(x, torch.zeros_like(x), LMAX2, next_weight=w, next_bias=b)
    assert h.shape == z.shape == (0, 240)
    gw, gb = torch.autograd.grad(z.sum() + h.sum(), [w, b])
    assert not gw.any() and not gb.any()
    assert equivariant_dropout(x, LMAX2, 0.5, dropout_rng(0)).shape == (0, 240)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("groups", [0, 1, 3, 5_000])
def test_a_gate_on_no_rows(dtype, groups):
    """an empty batch goes through with any gate, as it does without one; the gate's gradient is zero, in its own type"""
    for gate_type in {dtype, torch.float32}:
        c = {k: torch.zeros(0, 240, dtype=dtype, device="cuda", requires_grad=True) for k in "xy"}
        gate = torch.ones(groups, 112, dtype=gate_type, device="cuda", requires_grad=True)
        w, b = torch.ones(112, device="cuda", requires_grad=True), torch.zeros(64, device="cuda", requires_grad=True)
        for _ in range(2):
            junk = torch.full((groups * 112 + 1,), float("nan"), dtype=gate_type, device="cuda")          # (what the gradient's memory may hold before)
            del junk
            h, z = norm_gate_residual(c["x"], c["y"], LMAX2, gate=gate, post_weight=w, post_bias=b, next_weight=w, next_bias=b, dropout=0.3, rng=dropout_rng(1))
            assert h.shape == z.shape == (0, 240) and h.dtype == dtype
            grads = torch.autograd.grad(h.sum() + z.sum(), [c["x"], c["y"], gate, w, b])
            assert [g.shape for g in grads] == [(0, 240), (0, 240), (groups, 112), (112,), (64,)] and grads[2].dtype == gate_type and not any(bool(g.any()) for g in grads)
    block = NormGateResidual(LMAX2).cuda()
    h, z = block(torch.zeros(0, 240, device="cuda"), torch.zeros(0, 240, device="cuda"), torch.nn.Parameter(torch.ones(1, 112, device="cuda")))
    assert h.shape == z.shape == (0, 240)


@pytest.mark.gpu
def test_row_operators_views():
    """features as columns of a wider tensor, at an odd offset: read through a copy; misaligned contiguous storage: read in place"""
    c = _norm_case(torch.float16, LMAX2, 9, seed=6)
    want = _norm_gpu(c)
    flat = torch.empty(9 * 240 + 1, dtype=torch.float16, device="cuda")
    off = flat[1:].view(9, 240).copy_(c["x"])
    wide = torch.empty(9, 250, dtype=torch.float16, device="cuda")
    wide[:, 3:243] = c["y"].cuda()
    h, z = norm_gate_residual(off, wide[:, 3:243], LMAX2, scale=c["scale"], post_weight=c["post_weight"].cuda(), post_bias=c["post_bias"].cuda(),
                              next_weight=c["next_weight"].cuda(), next_bias=c["next_bias"].cuda())
    assert torch.equal(h, want[0]) and torch.equal(z, want[1])


# ---- together, as a training step uses them ---------------------------------------------------------------------------------------------------------

class _Block(torch.nn.Module):
    """norm -> messages along the edges -> attention -> dropout -> gated residual and the next norm: the training form of a graph attention block with
    plain linear layers in the place of the tensor products"""

    def __init__(self):
        super().__init__()
        self.norm = EquivariantLayerNormV2(LMAX2)
        self.to_alpha, self.to_value, self.proj = torch.nn.Linear(240, 64), torch.nn.Linear(240, 240), torch.nn.Linear(240, 240)
        self.attention = EdgeAttention(4, 16, alpha_drop=0.1, bias_boundaries=[2.0, 4.0, 6.0], seed=1)
        self.drop = EquivariantDropout(LMAX2, 0.1, seed=2)
        self.residual = NormGateResidual(LMAX2, scale=0.5, drop_prob=0.1, seed=3)
        self.gate = torch.nn.Parameter(torch.full((1, 112), 0.8))

    def forward(self, x, src, segments, logits, length):
        m = self.norm(x)[src]
        out = self.attention(self.to_alpha(m).view(-1, 4, 16), self.to_value(m).view(-1, 4, 60), segments, logits, length)
        return self.residual(x, self.drop(self.proj(out.flatten(1))), self.gate)


def _block_reference(block, x, src, dst, logits, length, calls):
    """the same in 64 bits on the CPU: -> (h, z) and a dict of its 64-bit parameters"""
    P = {k: v.detach().cpu().double().requires_grad_(True) for k, v in block.named_parameters()}
    blocks, E, N = parse_irreps(LMAX2), len(src), len(x)
    lin = lambda t, n: t @ P[n + ".weight"].T + P[n + ".bias"]          # noqa: E731
    m = O.layer_norm(x, blocks, P["norm.affine_weight"], P["norm.affine_bias"], 1e-5)[src]
    keep = lambda rows, cols, first, seed: O.keep(rows, cols, first, 0.1, seed, calls)          # noqa: E731
    out = O.attention(lin(m, "to_alpha").view(E, 4, 16), lin(m, "to_value").view(E, 4, 60), P["attention.alpha_dot"][0], dst, N, logits, length,
                      torch.tensor([2.0, 4.0, 6.0]), P["attention.bias_table"], keep(E, 4, 0, 1))
    y = lin(out.flatten(1), "proj") * O.per_channel(keep(N, 112, 1 << 16, 2), blocks)
    h, z = O.norm_gate_residual(x, y, blocks, 0.5, P["gate"], (P["residual.post_norm.affine_weight"], P["residual.post_norm.affine_bias"]), keep(N, 112, 1 << 16, 3),
                                (P["residual.next_norm.affine_weight"], P["residual.next_norm.affine_bias"]))
    return h, z, P


def _block_inputs():
    from diffusion_edf_amd.connectivity import radius_graph
    g = torch.Generator().manual_seed(4)
    xyz = torch.rand(150, 3, generator=g) * 12
    dst, src = radius_graph(xyz.cuda(), 4.0, max_num_neighbors=1000)
    length = (xyz.cuda()[src] - xyz.cuda()[dst]).norm(dim=1)
    logits = (1 - length / 4.0).clamp(min=1e-12).log()
    return torch.randn(150, 240, generator=g), src, dst, logits, length


@pytest.mark.gpu
def test_a_block_in_training_against_64_bits():
    """Two steps of the block on a radius graph, masks counted on.  Linear layers in between add sums of 240 products: every value passes about 4 norms, 3
    products of 240 terms and an attention of up to 60 edges, (4 x 256 + 3 x 240 + 60 x 2) roundings of values of their own scale at most: 2e3 u = 1.2e-4 of
    an output's scale; gradients go through as many again, 2.4e-4 of a gradient's largest value."""
    torch.manual_seed(0)
    block = _Block().cuda()
    x, src, dst, logits, length = _block_inputs()
    seg = EdgeSegments(dst, 150)
    for step in range(2):
        leaf = x.cuda().requires_grad_(True)
        h, z = block(leaf, src, seg, logits, length)
        loss = (h * z.detach().tanh()).sum() + z.square().sum() * 0.1
        names = [n for n, _ in block.named_parameters()]
        grads = dict(zip(["x"] + names, torch.autograd.grad(loss, [leaf] + list(block.parameters()))))
        xr = x.double().requires_grad_(True)
        wh, wz, P = _block_reference(block, xr, src.cpu(), dst.cpu(), logits.cpu().double(), length.cpu(), step)
        wl = (wh * z.detach().tanh().cpu().double()).sum() + wz.square().sum() * 0.1
        want = dict(zip(["x"] + names, torch.autograd.grad(wl, [xr] + [P[n] for n in names])))
        for got, ref in ((h, wh), (z, wz)):
            assert float((got.detach().cpu().double() - ref.detach()).abs().max()) <= 1.2e-4 * float(ref.detach().abs().max()), step
        for n, g in grads.items():
            assert float((g.cpu().double() - want[n]).abs().max()) <= 2.4e-4 * float(want[n].abs().max()), (step, n)
    assert block.attention.rng.tolist() == [1, 2] and block.drop.rng.tolist() == [2, 2] and block.residual.rng.tolist() == [3, 2]


@pytest.mark.gpu
def test_a_captured_training_step_draws_anew_and_matches_the_eager_one():
    """forward and backward of the block in one graph; each replay counts the masks on and takes new inputs from its buffers; between replays the program's own
    eager work runs.  Every replay equals the eager step with the same counters, bit for bit."""
    torch.manual_seed(1)
    block = _Block().cuda()
    x, src, dst, logits, length = _block_inputs()
    seg = EdgeSegments(dst, 150)
    params = list(block.parameters())

    def step(leaf):
        h, z = block(leaf, src, seg, logits, length)
        loss = h.square().sum() + (h * z).sum()
        return [h.detach(), z.detach()] + list(torch.autograd.grad(loss, [leaf] + params))

    buffer = x.cuda().requires_grad_(True)
    rngs = [block.attention.rng, block.drop.rng, block.residual.rng]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(buffer)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for r in rngs:
        r[1] = 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(buffer)
    for i in range(4):
        with torch.no_grad():
            buffer.copy_(x.cuda() * (1 + 0.1 * i))
        before = [r.clone() for r in rngs]
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        after = [r.clone() for r in rngs]
        assert all(int(b[1]) + 1 == int(a[1]) for b, a in zip(before, after))
        for r, b in zip(rngs, before):
            r.copy_(b)
        want = step((x.cuda() * (1 + 0.1 * i)).requires_grad_(True))
        # (the index_add of m = norm(x)[src] in torch's own backward sums in no fixed order: what passes through it may differ in the last places)
        for k, (a, b) in enumerate(zip(got, want)):
            if k < 2:
                assert torch.equal(a, b), (i, k)
            else:
                assert float((a - b).abs().max()) <= 1e-4 * float(b.abs().max()), (i, k)


@pytest.mark.gpu
def test_a_captured_backward_accumulates_into_parameters():
    """loss.backward() inside a capture, as training loops capture a step: the parameters' gradients after each replay are the eager ones (same masks; torch's own
    index_add in between sums in no fixed order, as above)"""
    torch.manual_seed(2)
    block = _Block().cuda()
    x, src, dst, logits, length = _block_inputs()
    seg, x = EdgeSegments(dst, 150), x.cuda()
    rngs = [block.attention.rng, block.drop.rng, block.residual.rng]

    def step():
        for p in block.parameters():
            p.grad = None
        h, z = block(x, src, seg, logits, length)
        (h.square().sum() + (h * z).sum()).backward()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    static = [p.grad for p in block.parameters()]
    for i in range(3):
        for r in rngs:
            r[1] = 5 + i
        graph.replay()
        torch.cuda.synchronize()
        got = [g.clone() for g in static]
        eager = _Block().cuda()
        eager.load_state_dict(block.state_dict())
        for r in (eager.attention.rng, eager.drop.rng, eager.residual.rng):
            r[1] = 5 + i
        h, z = eager(x, src, seg, logits, length)
        (h.square().sum() + (h * z).sum()).backward()
        for a, p in zip(got, eager.parameters()):
            assert float((a - p.grad).abs().max()) <= 1e-4 * float(p.grad.abs().max()), i


@pytest.mark.gpu
def test_modules_in_half_precision():
    """half() casts the parameters; the operators use them in float32 and return gradients in their type"""
    block = _Block().cuda().half()
    x, src, dst, logits, length = _block_inputs()
    h, z = block(x.cuda().half(), src, EdgeSegments(dst, 150), logits, length)
    assert h.dtype == z.dtype == torch.float16
    (h.float().square().sum() + z.float().sum()).backward()
    assert all(p.grad is not None and p.grad.dtype == torch.float16 and bool(p.grad.isfinite().all()) for p in block.parameters())


@pytest.mark.gpu
@pytest.mark.parametrize("cast", ["half", "bfloat16"])
def test_edges_keep_their_buckets_in_half_precision(cast):
    """lengths next to boundaries that a 16-bit type rounds past them: a table of one bias a bucket, which the cast holds exactly, tells which was taken"""
    bounds = torch.tensor([0.1, 2.1, 19.99, 19.9901])
    length = torch.cat([bounds, torch.nextafter(bounds, torch.zeros(4)), torch.nextafter(bounds, torch.full((4,), 99.0))])
    m = EdgeAttention(1, 4, bias_boundaries=bounds)
    with torch.no_grad():
        m.bias_table.copy_(torch.arange(5.0)[:, None])
    m = getattr(m.cuda(), cast)()
    # one row of each edge beside one of the first bucket: its share is exp(bucket) / (exp(bucket) + 1)
    n = len(length)
    seg = EdgeSegments(torch.arange(n, device="cuda").repeat_interleave(2), n)
    both = torch.stack([length, torch.zeros(n)], 1).flatten().cuda()
    dtype = m.alpha_dot.dtype
    value = torch.tensor([1.0, 0.0], dtype=dtype, device="cuda").repeat(n)[:, None, None]
    share = m(torch.zeros(2 * n, 1, 4, dtype=dtype, device="cuda"), value, seg, edge_length=both)[:, 0, 0]
    bucket = (length[:, None] >= bounds[None, :]).sum(1).double()
    close(share, torch.sigmoid(bucket), 16 * U, "share")          # (neighbouring buckets' shares lie 0.029 or more apart)


@pytest.mark.gpu
def test_two_captured_graphs_share_nothing():
    """two graphs of the operators alone, replayed in turn and out of order, against their eager results bit for bit: no workspace between them"""
    cases = [_case(torch.float32, 60, 900, buckets=4, drop=0.2, seed=s) for s in (1, 2)]
    norms = [_norm_case(torch.float32, LMAX2, 60, groups=1, drop=0.2, seed=s) for s in (1, 2)]
    eager = [(_gpu(c, train=False)[0], _norm_gpu(n)[:2]) for c, n in zip(cases, norms)]
    graphs = []
    for c, n in zip(cases, norms):
        seg, rng, nrng = EdgeSegments(c["dst"].cuda(), c["N"]), dropout_rng(*c["rng"]), dropout_rng(*n["rng"])
        cu = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
        nu = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in n.items()}

        def call(cu=cu, nu=nu, seg=seg, rng=rng, nrng=nrng):
            o = edge_attention(cu["alpha"], cu["value"], cu["dot"], seg, edge_logits=cu["logits"], edge_length=cu["length"], bias_boundaries=cu["bounds"], bias_table=cu["table"],
                               dropout=cu["drop"], rng=rng)
            return o, norm_gate_residual(nu["x"], nu["y"], LMAX2, scale=nu["scale"], gate=nu["gate"], post_weight=nu["post_weight"], post_bias=nu["post_bias"], dropout=nu["drop"],
                                         rng=nrng, next_weight=nu["next_weight"], next_bias=nu["next_bias"])

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out, call))
    for turn in ((0, 1), (1, 0), (0, 0, 1), (1, 1, 0)):
        for i in turn:
            graphs[i][1][0].zero_()
            graphs[i][0].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            o, (h, z) = graphs[i][1]
            assert torch.equal(o, eager[i][0]) and torch.equal(h, eager[i][1][0]) and torch.equal(z, eager[i][1][1]), (turn, i)


@pytest.mark.gpu
def test_operators_on_a_stream_of_their_own():
    c, n = _case(torch.float32, 500, 9_000, buckets=4, drop=0.2, seed=11), _norm_case(torch.float32, LMAX2, 500, groups=5, drop=0.2)
    want, wg = _gpu(c)
    wh, wz, wn = _norm_gpu(n)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out, g = _gpu(c)
        h, z, gn = _norm_gpu(n)
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(h, wh) and torch.equal(z, wz)
    assert all(torch.equal(g[k], wg[k]) for k in g) and all(torch.equal(gn[k], wn[k]) for k in gn)
