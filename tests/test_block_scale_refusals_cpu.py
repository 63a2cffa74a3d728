"""The params of a block-scaled cache (NaN scales) do not run in a decode that has not been given the block scales, without a
GPU."""
import pytest

NAN = float("nan")
FP16, FP8 = 0, 1


def params(pa, k_scale=1.0, v_scale=1.0):
    p = pa.DecodeParams()
    p.batch, p.num_q_heads, p.num_kv_heads, p.head_dim, p.page_size, p.num_ctas = 2, 8, 2, 128, 16, 4
    p.k_scale, p.v_scale = k_scale, v_scale
    return p


@pytest.mark.parametrize("scales", [(NAN, NAN), (NAN, 1.0), (1.0, NAN)])
def test_nan_scales_are_refused(scales, pa):
    p = params(pa, *scales)
    with pytest.raises(pa.InvalidArgument, match="block-scaled"):
        pa.paged_decode(FP8, p)
    with pytest.raises(pa.InvalidArgument, match="block-scaled"):
        pa.paged_decode_static(FP8, p, 4)
    p.num_ctas = 0                                  # an empty step too
    with pytest.raises(pa.InvalidArgument, match="block-scaled"):
        pa.paged_decode(FP8, p)


def test_scales_that_are_not_used_may_be_nan(pa):
    """The next check (null pointers) is reached: fp16 params, and head scales in place of the tensor's."""
    p = params(pa, NAN, NAN)
    with pytest.raises(pa.InvalidArgument, match="null device pointer"):
        pa.paged_decode(FP16, p)
    with pytest.raises(pa.InvalidArgument, match="null device pointer"):
        pa.paged_decode(FP8, p, d_k_scales=1 << 20, d_v_scales=2 << 20)
    with pytest.raises(pa.InvalidArgument, match="null device pointer"):
        pa.paged_decode(FP8, p, 0, 7, d_block_scales=1 << 20)
    with pytest.raises(pa.InvalidArgument, match="block-scaled"):
        pa.paged_decode(FP8, p, d_k_scales=1 << 20)
