"""Refusals and host-side rules of block_norm, token_logprobs and the 4-bit
group products.  CPU only: every call here is turned down before a launch, or
touches no device at all."""
import ctypes

import pytest
import torch

from vibeblade_amd import _lib
from vibeblade_amd.group4 import GroupQTensor, group_gemv
from vibeblade_amd.tensor import block_norm, token_logprobs

OK, INVAL = 0, -1
PTR = 0x1000  # never dereferenced: the calls below are refused or empty


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def norm_args(**kw):
    a = dict(branch=PTR, branch_type=0, branch_ld=8, post_w=PTR, gate=None, gate_type=0, gate_row=0, gate_col=0,
             scale=1.0, x=PTR, x_type=0, x_ld=8, y=PTR, y_ld=8, pre_w=PTR, n=PTR, n_type=0, n_ld=8, rows=2, dim=8,
             eps=1e-5, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("bad", [dict(branch_type=3), dict(x_type=-1), dict(n_type=7), dict(gate=PTR, gate_type=9),
                                 dict(rows=-1), dict(dim=0), dict(dim=1 << 31), dict(eps=-1.0), dict(eps=float("nan")),
                                 dict(branch=None), dict(x=None), dict(y=None), dict(n=None), dict(y_ld=7), dict(n_ld=7),
                                 dict(x_ld=-8), dict(branch_ld=-1), dict(gate=PTR, gate_col=2),
                                 dict(gate=PTR, gate_row=-1)])
def test_block_norm_refuses(lib, bad):
    assert lib.vb_block_norm(*norm_args(**bad)) == INVAL
    assert b"vb_block_norm" in lib.vb_last_error()


def test_block_norm_without_rows_does_nothing(lib):
    assert lib.vb_block_norm(*norm_args(rows=0, branch=None, x=None, y=None, n=None)) == OK


def lp_args(**kw):
    a = dict(logits=PTR, type=0, ld=100, rows=2, vocab=100, temperature=1.0, tokens=PTR, token_bytes=8, n_tokens=1,
             logprobs=PTR, entropy=PTR, top=3, top_ids=PTR, top_logprobs=PTR, workspace=PTR, workspace_bytes=1 << 30,
             stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("bad", [dict(type=3), dict(rows=-1), dict(vocab=0), dict(vocab=1 << 31), dict(ld=-1),
                                 dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")),
                                 dict(temperature=float("inf")), dict(temperature=1e-40), dict(n_tokens=-1),
                                 dict(token_bytes=2), dict(tokens=None), dict(logprobs=None), dict(top=-1), dict(top=65),
                                 dict(top_ids=None), dict(top_logprobs=None), dict(logits=None)])
def test_token_logprobs_refuses(lib, bad):
    assert lib.vb_token_logprobs(*lp_args(**bad)) == INVAL
    assert b"vb_token_logprobs" in lib.vb_last_error()


def test_token_logprobs_vocabulary_within_a_slice_offset(lib):
    assert lib.vb_token_logprobs_workspace(600, 1 << 28, 1) >= 0
    assert lib.vb_token_logprobs_workspace(600, (1 << 28) + 1, 1) == -1
    assert lib.vb_token_logprobs(*lp_args(vocab=(1 << 28) + 1, ld=0)) == INVAL


def test_token_logprobs_workspace(lib):
    for bad in ((-1, 10, 1), (1, 0, 1), (1, 1 << 31, 1), (1, 10, 65), (1, 10, -1)):
        assert lib.vb_token_logprobs_workspace(*bad) == -1
    for rows, vocab, top in ((0, 10, 0), (1, 1, 1), (1, 128256, 20), (1500, 151669, 0), (1 << 20, 200000, 64)):
        need = lib.vb_token_logprobs_workspace(rows, vocab, top)
        assert need >= 0
        if need:
            assert lib.vb_token_logprobs(*lp_args(rows=rows, vocab=vocab, ld=vocab, top=top,
                                                  workspace_bytes=need - 1)) == INVAL
            assert lib.vb_token_logprobs(*lp_args(rows=rows, vocab=vocab, ld=vocab, top=top, workspace=PTR + 8,
                                                  workspace_bytes=need)) == INVAL
    assert lib.vb_token_logprobs(*lp_args(rows=0, logits=None, tokens=None, logprobs=None)) == OK


@pytest.mark.parametrize("group", [0, -32, 16, 48, 96, 100, 192])
def test_group4_has_no_layout_for_other_groups(lib, group):
    assert lib.vb_group4_bytes(16, 256, group, 0) == -1
    assert lib.vb_group4_pack(PTR, PTR, None, PTR, 16, 256, group, None) == INVAL


def test_group4_bytes(lib):
    # whole blocks of 16 rows x 256: codes 2048, then per group of 16 rows 32 bytes of scales and 8 of zero points
    assert lib.vb_group4_bytes(16, 256, 128, 0) == 2048 + 2 * 32
    assert lib.vb_group4_bytes(16, 128, 32, 1) == 2048 + 8 * 40
    assert lib.vb_group4_bytes(17, 257, 64, 1) == 4 * (2048 + 4 * 40)
    assert lib.vb_group4_bytes(1, 1, 1024, 0) == 2048 + 2 * 32
    assert lib.vb_group4_bytes(128256, 16384, 128, 1) == 8016 * 64 * (2048 + 2 * 40)
    for bad in ((0, 128), (16, 0), (-1, 128), (1 << 31, 128), (16, 1 << 31)):
        assert lib.vb_group4_bytes(*bad, 128, 0) == -1


@pytest.mark.parametrize("call", [
    lambda lib: lib.vb_group4_pack(None, PTR, None, PTR, 16, 128, 128, None),
    lambda lib: lib.vb_group4_pack(PTR, None, None, PTR, 16, 128, 128, None),
    lambda lib: lib.vb_group4_pack(PTR, PTR, None, PTR + 8, 16, 128, 128, None),
    lambda lib: lib.vb_group4_quantize(PTR, 3, 128, 16, 128, 128, PTR, PTR, None, None),
    lambda lib: lib.vb_group4_quantize(PTR, 0, -1, 16, 128, 128, PTR, PTR, None, None),
    lambda lib: lib.vb_group4_quantize(None, 0, 128, 16, 128, 128, PTR, PTR, None, None),
    lambda lib: lib.vb_group4_dequant_rows(PTR, None, 16, 128, 128, 0, None),
    lambda lib: lib.vb_group4_dequant_rows(PTR + 4, PTR, 16, 128, 128, 0, None),
    lambda lib: lib.vb_group4_gemv(PTR, 16, 128, 128, 0, PTR, 3, 128, 1, PTR, PTR, 1 << 30, None),
    lambda lib: lib.vb_group4_gemv(PTR, 16, 128, 128, 0, PTR, 0, 128, -1, PTR, PTR, 1 << 30, None),
    lambda lib: lib.vb_group4_gemv(PTR, 16, 128, 128, 0, PTR, 0, -1, 2, PTR, PTR, 1 << 30, None),
    lambda lib: lib.vb_group4_gemv(PTR, 16, 0, 128, 0, PTR, 0, 128, 1, PTR, PTR, 1 << 30, None),
    lambda lib: lib.vb_group4_gemv(PTR, 16, 128, 48, 0, PTR, 0, 128, 1, PTR, PTR, 1 << 30, None),
    lambda lib: lib.vb_group4_gemv(None, 16, 128, 128, 0, PTR, 0, 128, 1, PTR, PTR, 1 << 30, None),
    lambda lib: lib.vb_group4_gemv(PTR + 8, 16, 128, 128, 0, PTR, 0, 128, 1, PTR, PTR, 1 << 30, None),
])
def test_group4_refuses(lib, call):
    assert call(lib) == INVAL


def test_group4_workspace(lib):
    for bad in ((-1, 16, 128, 128, 0, 0), (1, 0, 128, 128, 0, 0), (1, 16, 128, 48, 0, 0), (1, 16, 128, 128, 0, 3)):
        assert lib.vb_group4_workspace(*bad) == -1
    assert lib.vb_group4_workspace(0, 16, 128, 128, 0, 0) == 0
    for m, rows, k, group, zeros, kind in ((8, 4096, 14336, 64, 1, 1), (70, 100, 4096, 32, 1, 0), (1, 64, 1 << 20, 32, 1, 0)):
        need = lib.vb_group4_workspace(m, rows, k, group, zeros, kind)
        assert need > 0 and need % 16 == 0
        for ws, nbytes in ((PTR, need - 1), (None, need), (PTR + 8, need)):
            assert lib.vb_group4_gemv(PTR, rows, k, group, zeros, PTR, kind, k, m, PTR, ws, nbytes, None) == INVAL
            assert b"workspace" in lib.vb_last_error()


def test_group4_gemv_of_no_tokens_does_nothing(lib):
    assert lib.vb_group4_gemv(PTR, 16, 128, 128, 0, None, 0, 128, 0, None, None, 0, None) == OK


def test_python_calls_take_gpu_tensors_only():
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="cuda"):
        block_norm(x, x)
    with pytest.raises(ValueError, match="cuda"):
        token_logprobs(x, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="cuda"):
        GroupQTensor.from_packed(torch.zeros((2, 4), dtype=torch.uint8), torch.zeros((2, 1), dtype=torch.float16), k=8)
    with pytest.raises(ValueError, match="cuda"):
        GroupQTensor(torch.zeros(2112, dtype=torch.uint8), 16, 128, 128, False)
    with pytest.raises(ValueError, match="cuda"):
        group_gemv(None, x)


def test_ctypes_signatures_have_the_header_s_argument_count():
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "vbhip.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name in ("vb_block_norm", "vb_token_logprobs", "vb_token_logprobs_workspace", "vb_group4_bytes",
                 "vb_group4_pack", "vb_group4_quantize", "vb_group4_dequant_rows", "vb_group4_workspace", "vb_group4_gemv"):
        args = re.search(name + r"\(([^)]*)\)", text).group(1).split(",")
        sig = _lib.SIGNATURES[name][1]
        assert len(args) == len(sig), name
        for a, c in zip(args, sig):
            want = ctypes.c_void_p if "*" in a else ctypes.c_float if "float" in a else \
                ctypes.c_size_t if "size_t" in a else ctypes.c_int64 if "int64_t" in a else ctypes.c_int32
            assert c is want, (name, a)


@pytest.fixture
def launches(monkeypatch):
    """Calls on CPU tensors up to their launches, which are written down and not made."""
    from vibeblade_amd import group4, tensor
    made = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)  # a CPU device's index
    for module in (tensor, group4):
        monkeypatch.setattr(module, "_gpu_tensor", lambda t, what: t.device)
        monkeypatch.setattr(module, "_launch", lambda dev, fn, *args: made.append((fn, args)))
    return made


def test_block_norm_refuses_out_over_what_other_rows_read(launches):
    buf = torch.zeros(40, 64)
    x, b, w = torch.zeros(6, 64), torch.ones(6, 64), torch.ones(64)
    row = torch.zeros(6, 200)
    for x_, branch, kw in (
            (buf[:6], b, dict(out=buf[1:7])),                                # shifted by a row
            (buf[1:7], b, dict(out=buf[:6])),
            (buf.view(-1)[:384].view(6, 64), b, dict(out=buf.view(-1)[1:385].view(6, 64))),  # by a value
            (buf[:12:2], b, dict(out=buf[:6])),                              # another row stride
            (buf[:1].expand(6, 64), b, dict(out=buf[:6])),
            (x, buf[:6], dict(out=buf[5:11])),
            (x, buf[3].expand(6, 64), dict(out=buf[:6])),
            (x, buf[:6].view(torch.bfloat16)[:, 64:], dict(out=buf[:6])),    # half of each row, another type
            (x, b, dict(out=buf[:6], gate=buf[2])),
            (x, b, dict(out=buf[:6], gate=buf[:6, :1])),
            (x, b, dict(out=buf[:6], gate=buf[1:7])),
            (x, b, dict(out=buf[:6], post_w=buf[5])),
            (x, b, dict(out=buf[:6], pre_w=buf[0])),
            (x[:1], b[:1], dict(out=buf[:1], post_w=buf[0])),
            (x[:1], b[:1], dict(out=buf[:1], pre_w=buf[0])),                 # read once y is stored
            (row[:, :64], b, dict(out=row[:, 63:127])),
            (row.as_strided((5, 64), (200, 1), 140), b[:5], dict(out=row[:5, :64])),  # ends in the next row
            (buf[:2], b[:2], dict(out=buf.view(-1)[10:138].view(2, 64))),
            (buf[0], b[0], dict(out=buf.view(-1)[1:65]))):
        with pytest.raises(ValueError, match="overlaps"):
            block_norm(x_, branch, **kw)
    assert not launches


def test_block_norm_takes_out_beside_or_over_its_operands(launches):
    buf, wide = torch.zeros(40, 64), torch.zeros(6, 256)
    x, b, w = torch.zeros(6, 64), torch.ones(6, 64), torch.ones(64)
    for x_, branch, kw in (
            (x, b, dict(out=x)), (x, x, dict(out=x)), (x, b, dict(out=b)), (x, b, dict(out=x, gate=x)),
            (buf[:1], b[:1], dict(out=buf[1:2], gate=buf[1])),
            (buf[:6], buf[6:12], dict(out=buf[12:18], gate=buf[18], post_w=buf[19], pre_w=buf[20])),
            (wide[:, :64], wide[:, 64:128], dict(out=wide[:, 128:192], gate=wide[:, 192:])),  # columns of one buffer
            (wide[:, :64], wide[:, 64:128], dict(out=wide[:, :64], gate=wide[:, 192:193])),
            (buf[1:13:2], b, dict(out=buf[:12:2])),                            # every second row and the others
            (wide[1:2, :64], b[:1], dict(out=wide.view(-1)[256:320].view(1, 64))),  # one row, two strides
            (x[:0], x[:0], dict(out=x[:0])), (x.t()[:6, :6], b[:, :6], dict(out=x[:, :6]))):
        launches.clear()
        y, _ = block_norm(x_, branch, **kw)
        assert y is kw["out"] and [fn for fn, _ in launches] == ["vb_block_norm"]


def host_weights(rows, k, group=32, zeros=False):
    """A GroupQTensor's fields around bytes on the host (for calls that make no launch)."""
    w = object.__new__(GroupQTensor)
    w.data = torch.zeros(_lib.load().vb_group4_bytes(rows, k, group, int(zeros)) + 64, dtype=torch.uint8)
    w.rows, w.k, w.group, w.zeros = rows, k, group, zeros
    return w


def test_group_gemv_takes_out_between_the_rows_of_x(launches):
    w, buf = host_weights(16, 32), torch.zeros(3, 100)
    x = buf[:, :32]
    for out in (buf[0, 32:80], buf[1, 40:88], buf.view(-1)[252:300]):
        launches.clear()
        group_gemv(w, x, out=out)
        assert [fn for fn, _ in launches] == ["vb_group4_gemv"]
    launches.clear()
    for out in (buf[0, 31:79], buf.view(-1)[60:108], buf.view(-1)[180:228], buf.view(-1)[231:279]):
        with pytest.raises(ValueError, match="overlaps"):
            group_gemv(w, x, out=out)
    assert not launches


def test_group_gemv_refuses_out_over_the_weights(launches):
    w = host_weights(16, 32)
    used = _lib.load().vb_group4_bytes(16, 32, 32, 0)
    w.data, spare = w.data[:used], w.data.view(torch.float32)
    x = torch.zeros(32)
    for at in (0, 10, used // 4 - 1):
        with pytest.raises(ValueError, match="overlaps"):
            group_gemv(w, x, out=spare[at:at + 16])
    assert not launches
    group_gemv(w, x, out=spare[used // 4:used // 4 + 16])
    assert launches


def test_workspaces_are_sized_on_the_device_that_runs_the_call(monkeypatch):
    """The entry points size a workspace by the CUs of the current device: that of the tensors, for both calls."""
    from contextlib import contextmanager
    from types import SimpleNamespace
    from vibeblade_amd import group4, tensor
    current, seen = [0], []

    @contextmanager
    def device(index):
        was, current[0] = current[0], index
        yield
        current[0] = was

    def entry(name):
        return lambda *args: seen.append((name, current[0])) or (32 if name.endswith("workspace") else 0)

    fake = SimpleNamespace(**{name: entry(name) for name in ("vb_token_logprobs_workspace", "vb_token_logprobs",
                                                             "vb_group4_workspace", "vb_group4_gemv")})
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(_lib, "load", lambda: fake)
    monkeypatch.setattr(_lib, "init", lambda index: None)
    monkeypatch.setattr(tensor, "_raw_stream", lambda index: 0)
    for module in (tensor, group4):
        monkeypatch.setattr(module, "_gpu_tensor", lambda t, what: torch.device("cuda", 1))
    token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64))
    w = SimpleNamespace(device=torch.device("cuda", 1), data=torch.zeros(1, dtype=torch.uint8), rows=4, k=10, group=32,
                        zeros=False, ptr=lambda: 0)
    group_gemv(w, torch.zeros(10))
    assert seen == [(name, 1) for name in ("vb_token_logprobs_workspace", "vb_token_logprobs", "vb_group4_workspace",
                                           "vb_group4_gemv")]
    assert current == [0]


@pytest.mark.parametrize("group", [(1 << 32) + 128, (1 << 32) + 32, 1 << 32, 1 << 31, (1 << 40) + 256])
def test_group4_refuses_groups_past_32_bits(launches, group):
    """The entry points take 32 bits, of which ctypes would pass the low ones: another group, with more scales."""
    packed, scales = torch.zeros((2, 512), dtype=torch.uint8), torch.zeros((2, 1), dtype=torch.float16)
    with pytest.raises(ValueError, match="group"):
        GroupQTensor.from_packed(packed, scales, k=1024, group=group)
    with pytest.raises(ValueError, match="group"):
        GroupQTensor(packed, 2, 1024, group, False)
    assert not launches


def test_token_logprobs_refuses_more_tokens_than_32_bits_count(launches):
    for t in ((1 << 31), (1 << 32) + 1):
        with pytest.raises(ValueError, match="tokens"):
            token_logprobs(torch.zeros(1, 10), torch.zeros((1, 1), dtype=torch.int32).expand(1, t))
    assert not launches


@pytest.mark.parametrize("rows,dim", [(1, 1), (0, 64), (0, 1), (4, 1), (1, 64), (4, 64)])
def test_block_norm_hands_over_gates_of_any_stride(launches, rows, dim):
    """Columns apart, also where there are too few values for torch to call such a gate strided."""
    x = torch.zeros(rows, dim)
    for gate in (torch.zeros(rows, 5 * dim)[:, ::5], torch.zeros(5 * dim)[::5], torch.zeros(dim, rows).t(),
                 torch.zeros(rows, 1, 7)[:, :, 3], torch.zeros(3, rows, dim).permute(1, 2, 0)[:, :, 1]):
        launches.clear()
        block_norm(x, x.clone(), gate=gate)
        (_, args), = launches
        assert args[6] >= 0 and args[7] in (0, 1)  # gate_row, gate_col


def test_group4_refuses_zero_points_past_four_bits(launches):
    packed, scales = torch.zeros((3, 32), dtype=torch.uint8), torch.zeros((3, 2), dtype=torch.float16)
    for bad in (16, 255):
        zeros = torch.full((3, 2), 15, dtype=torch.uint8)
        zeros[2, 1] = bad
        with pytest.raises(ValueError, match="zero points"):
            GroupQTensor.from_packed(packed, scales, zeros, k=64, group=32)
    assert not launches


def test_rows_meet_as_their_bytes_do():
    import random
    from vibeblade_amd.tensor import _rows_meet
    rng = random.Random(0)
    seen = [0, 0]
    for _ in range(20000):
        width, q_width = rng.randint(1, 9), rng.randint(1, 9)
        rows, q_rows = rng.randint(0, 5), rng.randint(0, 5)
        p_ld, q_ld = width + rng.randint(0, 12), rng.randint(0, 20)
        p, q = rng.randint(100, 160), rng.randint(100, 160)
        ours = {p + i * p_ld + j for i in range(rows) for j in range(width)}
        theirs = {q + i * q_ld + j for i in range(q_rows) for j in range(q_width)}
        want = bool(ours & theirs)
        seen[want] += 1
        assert _rows_meet(p, p_ld, width, rows, q, q_ld, q_width, q_rows) == want
    assert min(seen) > 2000
