"""The serving operators on the CPU: what their entry points refuse, in Python and at the C ABI, before any CUDA call; the
declared symbols; and the oracles' own forms."""

import ctypes

import pytest
import torch

from ckb200 import _native, attention, build, rope, verify
from oracle import serving
from test_abi import declared


@pytest.fixture(scope="module", autouse=True)
def libs():
    build.build()


@pytest.mark.parametrize("op", build.SERVING_OPS)
def test_library_exports_every_declared_symbol(op):
    names = declared(op)
    lib = ctypes.CDLL(build.lib_path(op))
    assert names and all(hasattr(lib, n) for n in names)
    assert names == set(_native.SIGNATURES[op])


def _qk(**change):
    a = dict(q=torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16), k=torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16),
             position_ids=torch.zeros(2, 3, dtype=torch.int64), q_weight=torch.ones(64), k_weight=torch.ones(64),
             cos=torch.zeros(8, 64), sin=torch.zeros(8, 64))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 3, 4, 64)), dict(k=torch.zeros(2, 3, 2, 64, dtype=torch.float16)),
    dict(k=torch.zeros(2, 3, 2, 32, dtype=torch.bfloat16)), dict(q=torch.zeros(2, 3, 0, 64, dtype=torch.bfloat16)),
    dict(q_weight=torch.ones(32)), dict(k_weight=torch.ones(64, dtype=torch.bfloat16)), dict(q_weight=torch.ones(64).double()),
    dict(cos=None), dict(cos=None, sin=None), dict(theta=1e4), dict(cos=torch.zeros(8, 32), sin=torch.zeros(8, 32)),
    dict(cos=torch.zeros(0, 64), sin=torch.zeros(0, 64)), dict(position_ids=torch.zeros(2, 3, dtype=torch.int32)),
    dict(position_ids=torch.zeros(3, 2, dtype=torch.int64)), {}])
def test_qk_norm_rope_refusals(change):
    with pytest.raises(ValueError, match="CUDA" if not change else "^rope candidate"):
        rope.qk_norm_rope(**_qk(**change))


def _cached(**change):
    a = dict(_qk(), v=torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16), slot_mapping=torch.zeros(2, 3, dtype=torch.int64),
             key_cache=torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16), value_cache=torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    dict(v=torch.zeros(2, 3, 2, 64)), dict(v=torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)),
    dict(key_cache=torch.zeros(4, 16, 2, 64)), dict(value_cache=torch.zeros(4, 16, 4, 64, dtype=torch.bfloat16)),
    dict(value_cache=torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16)),
    dict(key_cache=torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16).transpose(1, 2)),
    dict(slot_mapping=torch.zeros(2, 3, dtype=torch.int32)), dict(slot_mapping=torch.zeros(6, dtype=torch.int64)), {}])
def test_qk_norm_rope_kv_cache_refusals(change):
    with pytest.raises(ValueError, match="CUDA" if not change else "^rope candidate"):
        rope.qk_norm_rope_kv_cache(**_cached(**change))


def test_in_place_refuses_what_cannot_be_written():
    with pytest.raises(ValueError, match="expanded"):
        rope._strided(torch.zeros(1, 1, 1, 64).expand(2, 3, 4, 64), "q")
    with pytest.raises(ValueError, match="contiguous last dim"):
        rope._strided(torch.zeros(2, 3, 64, 4).transpose(2, 3), "q")
    x = torch.zeros(2, 3, 8, 64)[:, :, 2:6]
    assert rope._strided(x) is x and rope._strided(x, "q") is x


def test_qk_norm_abi_refusals():
    fn = _native.load("rope").ckb_rope_qk_norm_launch
    p = 16  # a pointer that is only compared with null: every call below returns before a launch
    strides = (ctypes.c_longlong * 15)()
    good = [p, p, p, p, p, p, p, None, p, p, p, p, p, p, strides, 8, 64, 2, 3, 4, 2, 64, 1, 0, 0, 1e-6, None]

    def call(**at):
        a = list(good)
        for i, v in at.items():
            a[int(i[1:])] = v
        return fn(*a)

    assert call(_17=0) == 0 and call(_18=0) == 0  # no tokens
    for change in (dict(_0=None), dict(_1=None), dict(_2=None), dict(_3=None), dict(_4=None), dict(_6=None), dict(_8=None),
                   dict(_10=None), dict(_12=None), dict(_13=None), dict(_14=None), dict(_15=0), dict(_17=1 << 31),
                   dict(_17=1 << 20, _18=1 << 20), dict(_19=0), dict(_20=0), dict(_21=63), dict(_21=0), dict(_22=0),
                   dict(_22=3), dict(_23=3), dict(_24=-1), dict(_5=None), dict(_9=None, _11=None)):
        assert call(**change) == -1, change


def _attend(**change):
    a = dict(q=torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16), key_cache=torch.zeros(9, 16, 2, 64, dtype=torch.bfloat16),
             value_cache=torch.zeros(9, 16, 2, 64, dtype=torch.bfloat16), block_tables=torch.zeros(2, 4, dtype=torch.int64),
             seq_lens=torch.zeros(2, dtype=torch.int64))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 3, 4, 64)), dict(q=torch.zeros(2, 4, 64, dtype=torch.bfloat16)),
    dict(q=torch.zeros(2, 0, 4, 64, dtype=torch.bfloat16)), dict(q=torch.zeros(2, 3, 3, 64, dtype=torch.bfloat16)),
    dict(q=torch.zeros(2, 3, 4, 60, dtype=torch.bfloat16)), dict(q=torch.zeros(2, 3, 4, 264, dtype=torch.bfloat16)),
    dict(key_cache=torch.zeros(9, 16, 2, 64).half()), dict(value_cache=torch.zeros(9, 16, 2, 128, dtype=torch.bfloat16)),
    dict(value_cache=torch.zeros(8, 16, 2, 64, dtype=torch.bfloat16)),
    dict(key_cache=torch.zeros(9, 2, 16, 64, dtype=torch.bfloat16).transpose(1, 2)),
    dict(block_tables=torch.zeros(2, 4, dtype=torch.int32)), dict(block_tables=torch.zeros(3, 4, dtype=torch.int64)),
    dict(block_tables=torch.zeros(2, 0, dtype=torch.int64)), dict(seq_lens=torch.zeros(2, dtype=torch.int32)),
    dict(seq_lens=torch.zeros(2, 1, dtype=torch.int64)), dict(shared_prefix=8), dict(shared_prefix=-16),
    dict(shared_prefix=80), dict(shared_prefix=16.0), dict(scale=0.0), dict(scale=float("nan")), dict(scale=-1.0), {}])
def test_attention_refusals(change):
    with pytest.raises(ValueError, match="CUDA" if not change else "^attention: "):
        attention.paged_attention(**_attend(**change))
    with pytest.raises(ValueError):
        attention.run(_attend(**change))


def test_attention_abi_refusals():
    lib = _native.load("attention")
    strides = (ctypes.c_longlong * 3)(768, 256, 64)
    sizes = (2, 3, 4, 2, 64, 16, 4, 0)
    need = lib.ckb_attention_workspace(*sizes)
    assert need > 0
    for i, v in ((0, 0), (0, 4097), (1, 0), (2, 3), (2, 0), (3, 0), (4, 0), (4, 12), (4, 264), (5, 0), (6, 0), (6, 1 << 40),
                 (7, 8), (7, -16), (7, 80)):
        assert lib.ckb_attention_workspace(*sizes[:i], v, *sizes[i + 1:]) == -1, (i, v)
    assert lib.ckb_attention_workspace(1, 1, 32, 8, 128, 16, 8192, 0) < 64 << 20  # a long table costs nothing
    p = 16
    good = [p, p, p, p, p, p, p, need, strides, 2, 3, 4, 2, 64, 9, 16, 4, 0, 0.125, 1, None]
    fn = lib.ckb_attention_paged_launch
    assert fn(*good[:9], 0, *good[10:]) == 0
    odd = (ctypes.c_longlong * 3)(768, 256, 60)
    for i, v in ((0, None), (0, 8), (1, None), (1, 24), (2, 24), (3, None), (4, None), (5, None), (5, 8), (6, None), (6, 8),
                 (7, need - 1), (8, None), (8, odd), (9, 4097), (10, 0), (11, 3), (13, 60), (14, -1), (15, 0), (16, 0),
                 (17, 8), (18, 0.0), (18, -1.0), (18, float("nan")), (18, float("inf")), (19, 0), (19, 3)):
        assert fn(*good[:i], v, *good[i + 1:]) == -1, (i, v)


def test_attention_workspace_grows_with_the_batch_and_covers_the_prefix():
    lib = _native.load("attention")
    one = lib.ckb_attention_workspace(16, 1, 32, 8, 128, 16, 512, 0)
    assert lib.ckb_attention_workspace(64, 1, 32, 8, 128, 16, 512, 0) > one
    assert lib.ckb_attention_workspace(16, 1, 32, 8, 128, 16, 512, 4096) > one
    assert lib.ckb_attention_workspace(1, 1, 32, 8, 128, 16, 512, 4096) == lib.ckb_attention_workspace(1, 1, 32, 8, 128, 16, 512, 0)


def test_the_oracle_of_the_attention_is_torchs():
    g = torch.Generator().manual_seed(1)
    kc, vc = (torch.randn(6, 4, 2, 8, generator=g) for _ in range(2))
    tables = torch.tensor([[3, 1, 0], [3, 5, 2]])
    q = torch.randn(2, 2, 4, 8, generator=g)
    for prefix in (0, 4):
        got, _ = serving.attend(q, kc, vc, tables, torch.tensor([9, 6]), 0.3, prefix)
        for b, n in enumerate((9, 6)):
            k, v = (c[tables[b]].flatten(0, 1)[:n].repeat_interleave(2, 1).double() for c in (kc, vc))
            for t in range(2):
                m = n - 1 + t
                want = torch.nn.functional.scaled_dot_product_attention(
                    q[b, t][:, None].double(), k[:m].transpose(0, 1), v[:m].transpose(0, 1), scale=0.3)[:, 0]
                torch.testing.assert_close(got[b, t], want)


def _drafts(**change):
    a = dict(target_probs=torch.zeros(2, 4, 10), draft_tokens=torch.zeros(2, 3, dtype=torch.int64), uniforms=torch.zeros(2, 4),
             draft_probs=torch.zeros(2, 3, 10), num_drafts=torch.zeros(2, dtype=torch.int64))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    dict(target_probs=torch.zeros(2, 4, 10).half()), dict(target_probs=torch.zeros(2, 10)), dict(target_probs=torch.zeros(2, 4, 0)),
    dict(target_probs=torch.zeros(2, 0, 10)), dict(draft_tokens=torch.zeros(2, 4, dtype=torch.int64)),
    dict(draft_tokens=torch.zeros(2, 3, dtype=torch.int32)), dict(uniforms=torch.zeros(2, 3)), dict(uniforms=torch.zeros(2, 4).double()),
    dict(draft_probs=torch.zeros(2, 4, 10)), dict(draft_probs=torch.zeros(2, 3, 10).bfloat16()),
    dict(num_drafts=torch.zeros(3, dtype=torch.int64)), dict(num_drafts=torch.zeros(2, dtype=torch.int32)), {}])
def test_verify_refusals(change):
    with pytest.raises(ValueError, match="CUDA" if not change else "^verify: "):
        verify.verify_drafts(**_drafts(**change))
    with pytest.raises(ValueError):
        verify.run(_drafts(**change))


def test_verify_abi_refusals():
    fn = _native.load("verify").ckb_verify_launch
    p = 16
    good = [p, p, p, None, p, p, p, 40, 10, 30, 10, 2, 3, 10, 0, None]
    assert fn(*good[:11], 0, *good[12:]) == 0
    for i, v in ((0, None), (2, None), (4, None), (5, None), (6, None), (11, 1 << 31), (12, -1), (12, 1 << 20), (13, 0),
                 (13, (1 << 30) + 1), (14, 2), (14, -1)):
        assert fn(*good[:i], v, *good[i + 1:]) == -1, (i, v)


def test_the_oracle_of_the_verification_is_the_definition():
    target = torch.tensor([[[0.5, 0.25, 0.25], [0.0, 0.5, 0.5]]])
    draft = torch.tensor([[[0.25, 0.75, 0.0]]])
    tok = torch.tensor([[1]])
    assert serving.verify(target, tok, torch.tensor([[0.3, 0.4]]), draft)[0].tolist() == [[1, 1]]  # .3 * .75 < .25
    assert serving.verify(target, tok, torch.tensor([[0.4, 0.4]]), draft)[0].tolist() == [[0, -1]]  # w = (.25, 0, .25)
    assert serving.verify(target, tok, torch.tensor([[0.4, 0.5]]), draft)[0].tolist() == [[2, -1]]
    assert serving.verify(target, tok, torch.tensor([[0.3, 0.4]]))[0].tolist() == [[0, -1]]  # one-hot: .3 >= .25


def test_the_oracle_of_the_verification_takes_bad_probabilities_as_zero():
    nan = float("nan")
    target = torch.tensor([[[0.5, 0.25, 0.25], [0.0, 0.5, 0.5]]])
    tok = torch.tensor([[1]])
    for q in (nan, -0.5):
        at = torch.tensor([[[0.25, q, 0.0]]])
        assert serving.verify(target, tok, torch.tensor([[0.99, 0.4]]), at)[0].tolist() == [[1, 1]]  # as q = 0: accepted
        beside = torch.tensor([[[q, 0.75, 0.25]]])  # refused; w = (.5, 0, 0)
        assert serving.verify(target, tok, torch.tensor([[0.5, 0.9]]), beside)[0].tolist() == [[0, -1]]
    target[0, 0, 2], less = -1.0, torch.tensor([[[0.0, 0.75, -2.0]]])  # w = (.5, 0, 0), not (.5, 0, 1)
    assert serving.verify(target, tok, torch.tensor([[0.5, 0.9]]), less)[0].tolist() == [[0, -1]]


@pytest.mark.parametrize("prefix", [128, 256, 384, 512, 4096])
@pytest.mark.parametrize("batch,tokens,q_heads,kv_heads", [(640, 4, 32, 8), (2, 1, 160, 160), (2, 1, 400, 400), (256, 5, 32, 8),
                                                           (64, 1, 32, 8), (16, 1, 8, 2), (1000, 8, 64, 8)])
def test_the_shared_work_leaves_an_eighth_of_the_sms(batch, tokens, q_heads, kv_heads, prefix):
    """Its pieces' part of the workspace is 2 x 128 rows (a row: D sums and two statistics) for each unit and each CTA, or what
    the form without tensor memory needs where that is more: so it bounds the CTAs, of which 7 for 8 of the 148 SMs are allowed."""
    lib = _native.load("attention")
    size = [lib.ckb_attention_workspace(batch, tokens, q_heads, kv_heads, 128, 16, 1024, n) for n in (prefix, 0)]
    rows = (size[0] - size[1]) // (128 * 4 + 8)
    all_rows = batch * tokens * (q_heads // kv_heads)
    units = kv_heads * -(-all_rows // (256 if all_rows > 128 else 128))
    assert 0 < rows and rows / 256 - units < 148 * 7 // 8 + 1


def test_a_wait_that_ran_out_is_raised(monkeypatch):
    class Lib:
        status = 0

        def ckb_attention_status(self, reset):
            assert reset == 1
            status, self.status = self.status, 0
            return status

    lib = Lib()
    monkeypatch.setattr(_native, "load", lambda op: lib)
    attention.check()
    lib.status = 1
    with pytest.raises(RuntimeError, match="ran out"):
        attention.check()
    attention.check()
    lib.status = -700
    with pytest.raises(RuntimeError, match="CUDA error 700"):
        attention.check()
