"""Refusals and host-side rules of expert routing, 8-bit integer products and
draft verification.  CPU only: every call here is turned down before a launch,
or touches no device at all."""
import numpy as np
import pytest
import torch

from vibeblade_amd import _lib
from vibeblade_amd.group4 import GroupQTensor
from vibeblade_amd.int8 import K_MAX, Int8QTensor, int8_gemm, quantize_tokens
from vibeblade_amd.moe import ExpertRouter, MoEExpertSet
from vibeblade_amd.moe_profiler import HotColdMap
from vibeblade_amd.tensor import EXPERTS_MAX, QTensor, moe_grouped_ffn, route_experts, verify_draft

OK, INVAL, UNSUPPORTED = 0, -1, -2
PTR = 0x1000  # never dereferenced: the calls below are refused or empty


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def args_of(defaults, kw):
    assert set(kw) <= set(defaults)
    return list({**defaults, **kw}.values())


def route_args(**kw):
    return args_of(dict(logits=PTR, type=0, ld=64, n_tokens=2, n_exp=64, topk=4, scores=0, bias=None, groups=1, groups_kept=1,
                        group_score=0, renorm=1, scale=1.0, out_idx=PTR, out_w=PTR, stream=None), kw)


@pytest.mark.parametrize("bad", [dict(type=3), dict(type=-1), dict(n_tokens=-1), dict(n_tokens=1 << 31), dict(n_exp=0),
                                 dict(n_exp=513), dict(ld=-1), dict(topk=0), dict(topk=65), dict(n_exp=3), dict(groups=0),
                                 dict(groups=65, n_exp=130), dict(groups=5), dict(groups=8, groups_kept=0),
                                 dict(groups=8, groups_kept=9), dict(groups=32, groups_kept=1), dict(scores=2),
                                 dict(group_score=-1), dict(scale=float("inf")), dict(scale=float("nan")), dict(logits=None),
                                 dict(out_idx=None), dict(out_w=None)])
def test_route_experts_refuses(lib, bad):
    assert lib.vb_route_experts(*route_args(**bad)) == INVAL
    assert b"vb_route_experts" in lib.vb_last_error()


def test_route_experts_without_tokens_does_nothing(lib):
    assert lib.vb_route_experts(*route_args(n_tokens=0, logits=None, out_idx=None, out_w=None)) == OK


def test_int8_bytes(lib):
    # whole blocks of 16 rows x 64, then a scale per row of the last tile
    assert lib.vb_int8_bytes(16, 64) == 1024 + 64
    assert lib.vb_int8_bytes(1, 1) == 1024 + 64
    assert lib.vb_int8_bytes(17, 65) == 4 * 1024 + 128
    assert lib.vb_int8_bytes(128256, 16384) == 128256 * 16384 + 4 * 128256
    assert lib.vb_int8_bytes(16, K_MAX) == 2048 * 1024 + 64
    assert lib.vb_int8_bytes(1 << 26, 64) == (1 << 26) * 68
    for bad in ((0, 64), (16, 0), (-1, 64), (1 << 31, 64), ((1 << 26) + 1, 64), (16, K_MAX + 1)):
        assert lib.vb_int8_bytes(*bad) == -1


def gemm_args(**kw):
    return args_of(dict(w=PTR, rows=32, k=128, x=PTR, x_type=0, x_ld=128, m=4, bias=None, y=PTR, y_type=0, workspace=PTR,
                        workspace_bytes=1 << 40, stream=None), kw)


@pytest.mark.parametrize("bad", [dict(w=None), dict(x=None), dict(y=None), dict(w=PTR + 8), dict(x_type=3, x=PTR + 4),
                                 dict(x_type=4), dict(x_type=-1), dict(y_type=3), dict(x_ld=-1), dict(m=-1), dict(m=1 << 31), dict(m=1 << 26, rows=1 << 20, x_type=3),
                                 dict(rows=0), dict(k=0), dict(k=K_MAX + 1)])
def test_int8_gemm_refuses(lib, bad):
    assert lib.vb_int8_gemm(*gemm_args(**bad)) == INVAL
    assert b"vb_int8_gemm" in lib.vb_last_error()


def test_int8_gemm_without_tokens_does_nothing(lib):
    assert lib.vb_int8_gemm(*gemm_args(m=0, x=None, y=None, workspace=None, workspace_bytes=0)) == OK


def test_int8_workspace(lib):
    for bad in ((-1, 16, 64, 0), (1, 0, 64, 0), (1, 16, 0, 0), (1, 16, K_MAX + 1, 0), (1, 16, 64, 4), (1, 16, 64, -1)):
        assert lib.vb_int8_workspace(*bad) == -1
    for m, rows, k, kind in ((1, 1024, 4096, 0), (8, 4096, 14336, 1), (203, 5121, 4100, 0), (4096, 14336, 4096, 2),
                             (300, 1000, 100, 3), (0, 16, 64, 0)):
        need = lib.vb_int8_workspace(m, rows, k, kind)
        assert need >= 0
        if need:
            assert lib.vb_int8_gemm(*gemm_args(m=m, rows=rows, k=k, x_type=kind, x_ld=k, workspace_bytes=need - 1)) == INVAL
            assert lib.vb_int8_gemm(*gemm_args(m=m, rows=rows, k=k, x_type=kind, x_ld=k, workspace=PTR + 4,
                                               workspace_bytes=need)) == INVAL


@pytest.mark.parametrize("call", [
    lambda lib: lib.vb_int8_pack(None, 64, PTR, PTR, 16, 64, None),
    lambda lib: lib.vb_int8_pack(PTR, 64, None, PTR, 16, 64, None),
    lambda lib: lib.vb_int8_pack(PTR, 64, PTR, PTR + 8, 16, 64, None),
    lambda lib: lib.vb_int8_pack(PTR, -1, PTR, PTR, 16, 64, None),
    lambda lib: lib.vb_int8_pack(PTR, 64, PTR, PTR, 0, 64, None),
    lambda lib: lib.vb_int8_quantize(PTR, 3, 64, 16, 64, PTR, None),
    lambda lib: lib.vb_int8_quantize(PTR, 0, -64, 16, 64, PTR, None),
    lambda lib: lib.vb_int8_quantize(None, 0, 64, 16, 64, PTR, None),
    lambda lib: lib.vb_int8_quantize(PTR, 0, 64, 16, 64, PTR + 4, None),
    lambda lib: lib.vb_int8_quantize(PTR, 0, 64, 16, K_MAX + 1, PTR, None),
    lambda lib: lib.vb_int8_dequant_rows(PTR, None, 16, 64, None),
    lambda lib: lib.vb_int8_dequant_rows(PTR + 4, PTR, 16, 64, None),
])
def test_int8_layout_refuses(lib, call):
    assert call(lib) == INVAL


def verify_args(**kw):
    return args_of(dict(target=PTR, type=0, target_seq=500, target_row=100, draft=PTR, draft_seq=400, draft_row=100,
                        drafted=PTR, token_bytes=8, drafted_row=4, lengths=None, uniforms=PTR, uniforms_row=5, n_seqs=2,
                        n_drafts=4, vocab=100, temperature=1.0, draft_temperature=1.0, tokens=PTR, accepted=PTR, workspace=PTR,
                        workspace_bytes=1 << 40, stream=None), kw)


@pytest.mark.parametrize("bad", [dict(type=3), dict(n_seqs=-1), dict(n_drafts=-1), dict(n_drafts=64), dict(vocab=0),
                                 dict(vocab=(1 << 28) + 1), dict(target_seq=-1), dict(target_row=-1), dict(draft_seq=-1),
                                 dict(draft_row=-1), dict(drafted_row=-1), dict(uniforms_row=-1), dict(temperature=0.0),
                                 dict(temperature=float("nan")), dict(draft_temperature=float("inf")),
                                 dict(draft_temperature=-1.0), dict(target=None), dict(drafted=None), dict(uniforms=None),
                                 dict(tokens=None), dict(accepted=None), dict(token_bytes=2), dict(workspace=None),
                                 dict(workspace=PTR + 8), dict(workspace_bytes=16)])
def test_verify_draft_refuses(lib, bad):
    assert lib.vb_verify_draft(*verify_args(**bad)) == INVAL
    assert b"vb_verify_draft" in lib.vb_last_error()


def test_verify_draft_without_sequences_does_nothing(lib):
    assert lib.vb_verify_draft(*verify_args(n_seqs=0, target=None, drafted=None, uniforms=None, tokens=None, accepted=None,
                                            workspace=None, workspace_bytes=0)) == OK


def test_verify_draft_workspace(lib):
    for bad in ((-1, 4, 100, 1), (1, 64, 100, 1), (1, -1, 100, 1), (1, 4, 0, 1), (1, 4, (1 << 28) + 1, 0)):
        assert lib.vb_verify_draft_workspace(*bad) == -1
    assert lib.vb_verify_draft_workspace(0, 4, 100, 1) == 0
    for case in ((1, 4, 128256, 0), (64, 4, 128256, 1), (8, 5, 32003, 1), (1, 0, 1, 0), (1000, 63, 7, 1)):
        assert lib.vb_verify_draft_workspace(*case) > 0


def routed_args(**kw):
    return args_of(dict(wg=PTR, wu=PTR, wd=PTR, n_exp=4, x=PTR, n_tokens=2, idx=PTR, weights=PTR, routing_ld=2, first_expert=0,
                        topk=2, y=PTR, h=256, i=256, gate_up_type=12, down_type=12, workspace=PTR, workspace_bytes=0,
                        stream=None), kw)


@pytest.mark.parametrize("bad", [dict(idx=None), dict(weights=None), dict(routing_ld=1), dict(first_expert=-1), dict(n_exp=65),
                                 dict(topk=9, routing_ld=9), dict(n_tokens=513), dict(x=None), dict(y=None), dict(wg=None)])
def test_routed_experts_refuse(lib, bad):
    assert lib.vb_moe_grouped_ffn_routed(*routed_args(**bad)) == INVAL


def test_routed_experts_refuse_types_and_small_workspaces(lib):
    assert lib.vb_moe_grouped_ffn_routed(*routed_args(gate_up_type=1)) == UNSUPPORTED
    assert lib.vb_moe_grouped_ffn_routed(*routed_args()) == -4
    assert lib.vb_moe_grouped_ffn_routed(*routed_args(n_tokens=0, idx=None, weights=None, x=None, y=None)) == OK


def test_routed_experts_of_no_tokens_with_more_choices_than_experts(lib):
    """A call's experts may be fewer than a token's choices: so without tokens too."""
    assert lib.vb_moe_grouped_ffn_routed(*routed_args(n_exp=1, n_tokens=0, idx=None, weights=None, x=None, y=None)) == OK
    assert lib.vb_moe_grouped_ffn_routed(*routed_args(n_exp=1, n_tokens=0)) == OK
    assert lib.vb_moe_grouped_ffn_routed(*routed_args(n_exp=1)) == -4  # past the arguments' checks: no workspace


def test_host_tensors_are_refused():
    z = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="cuda"):
        route_experts(z, 2)
    with pytest.raises(ValueError, match="cuda"):
        quantize_tokens(z)
    with pytest.raises(ValueError, match="cuda"):
        Int8QTensor.from_int8(torch.zeros(2, 8, dtype=torch.int8), torch.ones(2))
    with pytest.raises(ValueError, match="cuda"):
        Int8QTensor(torch.zeros(1088, dtype=torch.uint8), 16, 64)
    with pytest.raises(ValueError, match="cuda"):
        verify_draft(torch.zeros(1, 2, 8), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 2))


@pytest.mark.parametrize("kind", [QTensor, GroupQTensor])
def test_int8_gemm_takes_its_own_weights_alone(kind):
    """Other weights have rows, k and a pointer too, to fewer bytes than the kernels read."""
    w = object.__new__(kind)
    w.data, w.rows, w.k, w.qtype = torch.zeros(32, 144, dtype=torch.uint8), 32, 256, 12
    with pytest.raises(ValueError, match="W must be an Int8QTensor"):
        int8_gemm(w, torch.zeros(1, 256))
    with pytest.raises(ValueError, match="W must be an Int8QTensor"):
        int8_gemm(torch.zeros(32, 256), torch.zeros(1, 256))


def test_router_options_are_named():
    w = torch.zeros(8, 4).numpy()
    with pytest.raises(TypeError, match="unknown"):
        ExpertRouter(w, 2, score="sigmoid")
    with pytest.raises(ValueError, match="bias"):
        ExpertRouter(w, 2, bias=[0.0] * 3)
    assert ExpertRouter(w, 2).options == {}
    assert EXPERTS_MAX == 512
    assert callable(moe_grouped_ffn) and callable(int8_gemm)


def test_hit_rate_passes_over_ids_of_no_expert():
    m = HotColdMap({0: [0, 1]}, {0: [2, 3]}, 1, 4)
    assert m.hit_rate(0, np.array([[0, -1], [2, -1], [1, 0]])) == 0.75  # as the executor counts the same routing
    assert m.hit_rate(0, np.array([[-1, -1]])) == 0.0
    assert m.hit_rate(0, np.array([0, 2])) == 0.5


def test_experts_batch_refuses_ids_of_no_expert():
    """-1 is no expert in a routing, not the last one."""
    rng = np.random.RandomState(0)
    gate, up, down = (rng.randn(4, *s).astype(np.float32) for s in ((6, 8), (6, 8), (8, 6)))
    experts = MoEExpertSet(gate, up, down)
    for bad in ([1, -1], np.array([[0, 3], [-1, 2]])):
        with pytest.raises(IndexError, match="no expert"):
            experts.get_experts_batch(bad)
    for ids in ([1, 3, 1], np.array([], dtype=np.int64)):
        for got, want in zip(experts.get_experts_batch(ids), (gate, up, down)):
            assert np.array_equal(got, np.transpose(want[np.asarray(ids)], (0, 2, 1)))
