"""Results of a verification that reach into an argument's place: other requests' arguments would be read behind them."""
import pytest
import torch

from test_verify_drafts import make
from tiny_inference_server_b200.kernels import ops


def test_results_that_reach_into_another_place():
    p, q, drafts, u = make(3, 2, 10, 0)
    room = torch.zeros(64, dtype=torch.int32)
    args = dict(target_probs=p, draft_probs=q, drafts=drafts, uniforms=u)
    inner = dict(drafts=room[10:16].view(3, 2))
    numbers = dict(uniforms=room[10:19].view(torch.float32).view(3, 3))
    lens = dict(draft_lens=room[10:13])
    for bad in (dict(inner, tokens=room[7:16].view(3, 3)), dict(inner, tokens=room[15:24].view(3, 3)), dict(inner, tokens=room[2:11].view(3, 3)),
                dict(inner, accepted=room[10:13]), dict(inner, accepted=room[15:18]), dict(inner, accepted=room[8:11]),
                dict(numbers, tokens=room[18:27].view(3, 3)), dict(numbers, tokens=room[2:11].view(3, 3)), dict(numbers, accepted=room[10:13]),
                dict(numbers, accepted=room[18:21]), dict(lens, tokens=room[4:13].view(3, 3)), dict(lens, tokens=room[12:21].view(3, 3)),
                dict(lens, accepted=room[11:14]), dict(lens, accepted=room[9:12]),
                dict(tokens=room[:9].view(3, 3), accepted=room[8:11]), dict(tokens=room[3:12].view(3, 3), accepted=room[1:4])):
        with pytest.raises(ops.KernelError, match="do not lie where"):
            ops.verify_drafts(**{**args, **bad})
    # beside one another, and kept drafts in the place of their lengths: taken (and refused for lying on the host only)
    for good in (dict(inner, tokens=room[16:25].view(3, 3), accepted=room[7:10]), dict(numbers, tokens=room[19:28].view(3, 3), accepted=room[7:10]),
                 dict(lens, accepted=room[10:13], tokens=room[13:22].view(3, 3)), dict(tokens=room[:9].view(3, 3), accepted=room[9:12])):
        with pytest.raises(ops.KernelError, match="CUDA tensors"):
            ops.verify_drafts(**{**args, **good})
    with pytest.raises(ops.KernelError, match="CUDA tensors"):      # no drafts at all
        ops.verify_drafts(p[:, :1], None, drafts[:, :0], u[:, :1].contiguous())
