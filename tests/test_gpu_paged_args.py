"""Arguments of the paged cache's launchers that would be taken for something else are refused, and what is refused writes nothing."""
import pytest
import torch

from test_gpu_paged import ints, make_pool

pytestmark = pytest.mark.gpu


def append_case(rd, hd=128, n=70):
    from yasakani_b200 import kv4, paged
    k, v, table, g = make_pool([n], 2, hd, 32, torch.bfloat16, seed=rd)
    x = torch.randn((n, 8, hd), generator=g, device="cuda").bfloat16()
    rope = torch.empty((128, rd // 2, 2), dtype=torch.float32, device="cuda")
    kv4.launch_rope_table_g(rope, 128, 1e6, rd)
    q_out = torch.full((n, 4, hd), 7.0, dtype=torch.bfloat16, device="cuda")
    a = dict(cache=paged.PagedCache.of(k, v), table=table, k=x[:, 4:6], v=x[:, 6:], seq=ints([0] * n), pos=torch.arange(n, dtype=torch.int32, device="cuda"),
             rope=rope, rd=rd, q=x[:, :4], q_out=q_out)
    return a, k, v, q_out


@pytest.mark.parametrize("made,asked", [(128, 64), (64, 128), (32, 96), (64, 16)])
def test_a_table_of_angles_of_another_width_is_refused(made, asked):
    from yasakani_b200 import paged
    a, k, v, q_out = append_case(made)
    old = k.clone(), v.clone()
    rope = a["rope"]
    for wrong in (rope, rope.view(128, -1), rope.view(-1, 2) if made != asked else rope[:, :, None], rope[None]):
        with pytest.raises(ValueError, match="rope"):
            paged.launch_append(**dict(a, rd=asked, rope=wrong))
    with pytest.raises(ValueError, match="rope"):
        paged.launch_append(**dict(a, rope=rope.view(-1)[:-2]))          # flat, and no whole positions
    torch.cuda.synchronize()
    assert torch.equal(k, old[0]) and torch.equal(v, old[1]) and (q_out == 7.0).all()


def test_angles_in_any_of_their_shapes():
    from yasakani_b200 import paged
    outs = []
    for shape in ((128, 32, 2), (128, 64), (-1,)):
        a, k, v, q_out = append_case(64)
        paged.launch_append(**dict(a, rope=a["rope"].view(shape)))
        outs.append((k, v, q_out))
    assert all(torch.equal(x, y) for o in outs for x, y in zip(o, outs[0])) and not (outs[0][2] == 7.0).any()


def test_an_output_without_its_queries_is_refused():
    from yasakani_b200 import paged
    a, k, v, q_out = append_case(64)
    old = k.clone()
    with pytest.raises(ValueError, match="q_out"):
        paged.launch_append(**dict(a, q=None))
    torch.cuda.synchronize()
    assert torch.equal(k, old) and (q_out == 7.0).all()
    paged.launch_append(**dict(a, q=None, q_out=None))
    torch.cuda.synchronize()
    assert not torch.equal(k, old)
