"""What the training operators do before a GPU is touched, and their reference against the oracle."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import nextdoor_amd as nd
from nextdoor_amd import NextDoorError, _capi, ops
from nextdoor_amd.walk_model import pack_walks
from tests import operators_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_reference_random_numbers_are_the_oracles(oracle):
    for seed, step, n in ((42, 0, 1000), (2 ** 64 - 1, 2 ** 31 - 1, 37), (0xFEDCBA9876543210, 17, 4)):
        want = [oracle.uniform_grouped(seed, o, step, 0) for o in range(n)]
        assert np.array_equal(ref.uniforms(n, seed, step), np.array(want, np.float32))


def test_tensors_on_the_host_are_refused():
    x = torch.zeros(4, 2, 32, dtype=torch.bfloat16)
    h, t = torch.zeros(4, 32, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: ops.dropout_forward(h, 0.5, 1, 1), lambda: ops.vocabulary_loss_forward(h, h, t),
                 lambda: ops.dropout(h, 0.5, 1, 1), lambda: ops.vocabulary_loss(h, h, t),
                 lambda: ops.dropout_forward(h.float().numpy(), 0.5, 1, 1),
                 lambda: ops.PackedSequences([0, 4], device="cpu")):
        with pytest.raises(NextDoorError, match="GPU"):
            call()

    class Plan:
        plan, n_tokens = torch.zeros(16, dtype=torch.uint8), 4
    with pytest.raises(NextDoorError, match="GPU"):
        ops.packed_attention_forward(x, x, x, Plan())


def attention_call(**changes):
    a = _capi.PackedAttention()
    base = 1 << 40
    fields = dict(n_tokens=256, n_covered=256, rounds=6, most_rounds=4, heads=4, kv_heads=2, dim=64, dtype=2, scale=0.125,
                  plan=base, q=base, k=base, v=base, dout=base, q_token=256, q_head=64, k_token=128, k_head=64, v_token=128,
                  v_head=64, dout_token=256, dout_head=64, out=base, lse=base, dq=base, dk=base, dv=base, workspace=base,
                  workspace_bytes=1 << 40)
    fields.update(changes)
    for name, value in fields.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("changes,match", [
    (dict(dtype=0), "16-bit"), (dict(n_tokens=-1), "tokens"), (dict(n_tokens=1 << 40), "tokens"), (dict(n_covered=257), "more tokens"),
    (dict(heads=5), "evenly"), (dict(kv_heads=0), "evenly"), (dict(dim=12), "multiple of 8"), (dict(dim=136), "multiple of 8"),
    (dict(dim=0), "multiple of 8"), (dict(scale=float("nan")), "finite"), (dict(q=None), "null"), (dict(plan=None), "null"),
    (dict(k=(1 << 40) + 8), "aligned"), (dict(q_token=-8), "strides"), (dict(v_head=4), "strides"),
    (dict(k_token=1 << 25), "strides"), (dict(most_rounds=1000), "no plan"), (dict(short_tiles=1000), "no plan"),
    (dict(short_tiles=-1), "no plan")])
def test_attention_calls_are_refused_before_they_touch_a_device(changes, match):
    """The addresses are never dereferenced: every call is refused first."""
    lib = _capi.lib()
    for fn in (lib.nd_packed_attention_forward, lib.nd_packed_attention_backward):
        assert fn(attention_call(**changes), None) != 0
        assert match in lib.nd_last_error().decode(), lib.nd_last_error()
    assert lib.nd_packed_attention_backward(attention_call(workspace_bytes=16), None) != 0
    assert "workspace" in lib.nd_last_error().decode()
    assert lib.nd_packed_attention_forward(None, None) != 0
    assert lib.nd_packed_attention_forward(attention_call(n_tokens=0, n_covered=0, q=None), None) == 0  # nothing to do


def test_loss_calls_are_refused_before_they_touch_a_device():
    lib = _capi.lib()
    base = 1 << 40

    def call(backward, **changes):
        a = _capi.VocabularyLoss()
        fields = dict(rows=10, classes=100, dim=64, dtype=2, hidden=base, weight=base, target=base, loss=base, lse=base, dloss=base,
                      dhidden=base, dweight=base, workspace=base, workspace_bytes=1 << 40)
        fields.update(changes)
        for name, value in fields.items():
            setattr(a, name, value)
        rc = (lib.nd_vocabulary_loss_backward if backward else lib.nd_vocabulary_loss_forward)(a, None)
        return rc, lib.nd_last_error().decode()

    for changes, match in ((dict(dtype=0), "16-bit"), (dict(rows=-1), "rows"), (dict(rows=1 << 40), "rows"), (dict(classes=0), "classes"),
                           (dict(classes=1 << 40), "classes"), (dict(dim=12), "multiple of 8"), (dict(hidden=None), "null"),
                           (dict(weight=base + 8), "aligned"), (dict(target=None), "null"), (dict(workspace_bytes=8), "workspace")):
        for backward in (False, True):
            rc, why = call(backward, **changes)
            assert rc != 0 and match in why, (changes, backward, why)
    assert call(True, dweight=None)[0] != 0 and call(False, loss=None)[0] != 0 and call(True, dloss=None)[0] != 0
    assert call(False, rows=0)[0] == 0
    assert lib.nd_vocabulary_loss_workspace(10, 0, 64, 0) == -1


def test_dropout_calls_are_refused_before_they_touch_a_device():
    lib = _capi.lib()
    base = 1 << 40
    for args, match in (((base, None, base, -1, 0, 0.5, 1, 1), "bad argument"), ((None, None, base, 5, 0, 0.5, 1, 1), "bad argument"),
                        ((base, None, base, 5, 7, 0.5, 1, 1), "type"), ((base, None, base, 5, 0, 1.5, 1, 1), "probability"),
                        ((base, None, base, 5, 0, float("nan"), 1, 1), "probability"), ((base, None, base, 5, 0, 0.5, 1, 1 << 31), "step")):
        assert lib.nd_dropout(*args, None) != 0
        assert match in lib.nd_last_error().decode()
    assert lib.nd_dropout(None, None, None, 0, 0, 0.5, 1, 1, None) == 0


def test_plans_are_refused_before_they_touch_a_device():
    import ctypes as C
    lib = _capi.lib()
    sizes = (C.c_int64 * 3)()

    def plan(starts, n_tokens):
        starts = np.asarray(starts, np.int32)
        rc = lib.nd_packed_plan(starts.ctypes.data, len(starts) - 1, n_tokens, None, None, sizes, None)
        return rc, lib.nd_last_error().decode()

    assert "not 0" in plan([1, 2], 5)[1] and "before it starts" in plan([0, 3, 2], 5)[1]
    assert "tokens in sequences" in plan([0, 6], 5)[1] and "null" in plan([0, 5], 5)[1]
    assert plan([0], 0)[0] == 0 and plan([0, 0, 0], 0)[0] == 0
    # the sizes are the host's: rounds of 64 keys over tiles of 128, the largest, tiles of whole sequences
    plan([0, 300], 300)
    assert list(sizes) == [2 + 4 + 5, 5, 0]
    plan([0, 100, 128, 130, 200, 300], 700)
    assert list(sizes)[2] == 3 + 4  # [0, 128), [128, 200), [200, 300), and the 400 tokens of no sequence
    assert lib.nd_packed_plan_bytes(-1) == -1


def test_a_library_on_another_hip_runtime_is_refused():
    """torch brings a runtime of its own; loaded after the library there are two, which share no streams."""
    code = ("import nextdoor_amd as nd\nnd.app_names()\nfrom nextdoor_amd import ops\n"
            "try:\n  ops._library()\nexcept nd.NextDoorError as e:\n  print('refused', 'import torch' in str(e))\n")
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-500:]
    assert done.stdout.split() == ["refused", "True"]


def test_walks_are_packed_up_to_where_they_end():
    n = 9  # "no vertex"
    samples = np.array([[1, 2, 3], [4, n, n], [n, n, n], [5, 6, n]], np.int32)
    tokens, targets, starts = pack_walks([0, 8, 7, 3], samples, n)
    assert starts.tolist() == [0, 4, 6, 7, 10]
    assert tokens.tolist() == [0, 1, 2, 3, 8, 4, 7, 3, 5, 6]
    assert targets.tolist() == [1, 2, 3, n, 4, n, n, 5, 6, n]
    tokens, targets, starts = pack_walks(np.zeros(0), np.zeros((0, 3)), n)
    assert len(tokens) == 0 and starts.tolist() == [0]


def test_reference_attention_gradient_is_the_derivative():
    """The gradient that the kernels are held to, against differences of the reference's own outputs."""
    starts, t = [0, 5, 6, 20], 22
    gen = torch.Generator().manual_seed(1)
    q, k, v, d = (torch.randn(t, h, 8, generator=gen, dtype=torch.float64) for h in (4, 2, 2, 4))

    class Double:
        dtype = torch.float16

        def __init__(self, x):
            self.x = x

        def double(self):
            return self.x

        def __getitem__(self, i):
            return self.x[i]

    got, _ = ref.attention(*map(Double, (q, k, v)), starts, 0.3, d)
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        direction = torch.randn(x.shape, generator=gen, dtype=torch.float64)
        value = []
        for sign in (1, -1):
            moved = [y + sign * 1e-5 * direction if y is x else y for y in (q, k, v)]
            value.append(float((ref.attention(*map(Double, moved), starts, 0.3)[0]["out"] * d).sum()))
        assert abs((value[0] - value[1]) / 2e-5 - float((got[name] * direction).sum())) < 1e-6


def test_calls_that_one_launch_does_not_hold_are_refused():
    lib = _capi.lib()
    a = attention_call(n_tokens=1 << 26, n_covered=1 << 26, heads=65535, kv_heads=1, dim=8)
    assert lib.nd_packed_attention_forward(a, None) != 0
    assert "one launch" in lib.nd_last_error().decode()
    base = 1 << 40
    for rows, classes, dim in ((1 << 20, 100, 65536), (100, 1 << 30, 64)):
        a = _capi.VocabularyLoss(rows=rows, classes=classes, dim=dim, dtype=2, hidden=base, weight=base, target=base, loss=base, lse=base,
                                 dloss=base, dhidden=base, dweight=base, workspace=base, workspace_bytes=1 << 60)
        for fn in (lib.nd_vocabulary_loss_forward, lib.nd_vocabulary_loss_backward):
            assert fn(a, None) != 0
            assert "elements to a matrix" in lib.nd_last_error().decode()
