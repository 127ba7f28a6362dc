"""The status word of the latent operators: 32 bits that the kernels set bits of.  No GPU is needed."""
import pytest
import torch

z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)  # noqa: E731
i32, i64, f64 = torch.int32, torch.int64, torch.float64


def calls():
    from vic_b200 import kernels as K
    return [
        (K.latent_append, dict(kv=z(2, 576), norm_weight=z(512), eps=1e-6, positions=z(2, dtype=i32), slots=z(2, dtype=i64), inv_freq=z(32, dtype=f64), cache=z(3, 8, 576))),
        (K.latent_query, dict(q=z(2, 4, 192), w_uk=z(4, 128, 512), positions=z(2, dtype=i32), inv_freq=z(32, dtype=f64), out=z(2, 4, 576))),
        (K.latent_value, dict(o=z(2, 4, 512), w_uv=z(4, 128, 512), out=z(2, 4, 128))),
        (K.latent_attention, dict(q=z(4, 4, 576), cache=z(9, 8, 576), page_table=z(2, 4, dtype=i32), seq_lens=z(2, dtype=i32), scale=0.1, out=z(4, 4, 512),
                                  workspace=z(16, dtype=torch.uint8)))]


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("bad", [z(1, dtype=torch.uint8), z(4, dtype=torch.int8)[1:2], z(1, dtype=torch.float16), z(1, dtype=i64), z(1, dtype=torch.float32), z(0, dtype=i32)])
def test_other_types_and_empty_tensors_are_refused(which, bad):
    """(An atomic on 32 bits at an odd address faults, and behind one byte it changes three others.)"""
    call, args = calls()[which]
    with pytest.raises(ValueError, match="status"):
        call(**args, status=bad)
