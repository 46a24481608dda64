"""Sequence operators on a drain's own device buffers, without a copy."""
import pytest

torch = pytest.importorskip("torch")

import seq_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu


class Words:
    """n rows of `words` floats at a device pointer, as torch takes them."""

    def __init__(self, ptr, n, words):
        self.__cuda_array_interface__ = {"shape": (n, words), "typestr": "<f4", "data": (ptr, False), "version": 3}


def test_features_in_a_drain_s_output_slots(stub_dir):
    """98 words a slot, the features behind two flags: rows of tokens as the drain
    wrote them, normed back into their place."""
    from ssla_hip import abi, events, hybrid, ops
    rec = events.blob_records(1500, seed=3)
    with hybrid.Drain.from_weights_dir(stub_dir) as d:
        d.load_rings([events.to_records(rec)])
        d._outs[0].zero()                       # rows of records that pass no gate
        d.run()
        slots = torch.as_tensor(Words(d._outs[0].ptr, 1500, abi.OUTPUT_DTYPE.itemsize // 4), device="cuda")
        assert slots.data_ptr() == d._outs[0].ptr
        feat = slots[:, 2:].unflatten(1, (2, 48))
        assert feat.stride() == (98, 48, 1)
        was = feat.clone()
        g = torch.full((2,), -0.05, device="cuda")
        got = ops.linear_attention(feat, feat, feat, g, scale=48 ** -0.5)
        R.check_linear_attention(got, None, R.linear_attention(was, was, was, g, [1500], 48 ** -0.5),
                                 torch.float32, 48, 1500)
        ops.group_norm(slots[:, 2:], 2, act="silu", out=slots[:, 2:])
        torch.cuda.synchronize()
        (out,), _ = d.results()                # downloaded from where the norm wrote
        new = torch.from_numpy(out["s3_feat"].copy())
        R.check_group_norm(new, R.group_norm(was.flatten(1), 2, None, None, 1e-5, "silu"), torch.float32)
        assert torch.equal(torch.from_numpy(out["pass3"].copy()), slots[:, 1].view(torch.int32).cpu())
