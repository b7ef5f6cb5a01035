"""A sealed cache beside the loop's compaction: what is sealed stays what the
planes hold."""
import pytest
import torch

from oracle import loop as OL
from tests import loop_cases as LC

MIL = 16


def test_rows_moved_keeps_whole_blocks_in_front():
    from hsd_b200.kv8 import Kv8Cache
    c = Kv8Cache(1, 1, 512, device="cpu")
    for sealed, first, left in ((512, 600, 512), (512, 511, 448), (512, 448, 448), (448, 512, 448),
                                (256, 63, 0), (256, 0, 0), (0, 100, 0)):
        c.sealed = sealed
        assert c.rows_moved(first) == left == c.sealed
    with pytest.raises(ValueError):
        c.rows_moved(-1)


@pytest.mark.gpu
@pytest.mark.parametrize("seed,period,tree", [(0, 1, False), (2, 3, False), (3, 1, True)])
def test_sealed_rows_follow_the_loops_compaction(seed, period, tree):
    """Every whole block in use is sealed before each step; after it, the rows that
    count as sealed are those of the planes, and blocks that left were stale."""
    from hsd_b200.compaction import plane_pointers
    from hsd_b200.kv8 import Kv8Cache
    from hsd_b200.loop import VerifyLoop
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    dev = torch.device("cuda:0")
    prompts, truths, drafts = LC.make_loop_case(seed)
    model = OL.true_text_model(prompts, truths, LC.VOCAB, LC.EOS)
    cap = 4096
    caches = [torch.zeros(2, cap, 128, dtype=torch.bfloat16, device=dev) for _ in range(4)]
    planes = plane_pointers(caches, device=dev)
    kv8 = Kv8Cache(2, 2, cap, device=dev)
    kw = dict(eos_token_id=LC.EOS, max_new_tokens=10 ** 6, pad_token_id=LC.PAD,
              min_input_length=MIL, compact_period=period, enable_tree_decode=tree,
              kv_capacity=cap, device=dev)
    for bad in (dict(kv8=kv8), dict(kv8=kv8, kv_planes=planes, row_bytes=128),
                dict(kv8=kv8, kv_planes=planes[:4], row_bytes=256)):
        with pytest.raises(ValueError):
            VerifyLoop(prompts, drafts, **bad, **kw)
    loop = VerifyLoop(prompts, drafts, kv_planes=planes, row_bytes=256, kv8=kv8, **kw)
    g = torch.Generator(device=dev).manual_seed(seed)
    kept = left = stale = 0
    for it in range(1000):
        ids, pos, mask = loop.inputs()
        total, q = loop.kv_tokens.numel(), ids.numel()
        for c in caches:        # the model's cache update, every row unlike the others
            c[:, total - q:total] = torch.randn(2, q, 128, generator=g, device=dev)
        kv8.seal(planes, total // 64 * 64 - kv8.sealed)
        before = kv8.sealed
        nxt = model(ids.cpu().numpy(), pos.cpu().numpy(), mask.plan().dense_allowed(),
                    loop.kv_tokens.cpu().numpy())
        more = loop.step(torch.from_numpy(nxt).to(dev))
        if not more:
            break
        now = Kv8Cache(2, 2, cap, device=dev)
        now.seal(planes, before)
        n = kv8.sealed
        assert torch.equal(now.data[:, :, :, :n], kv8.data[:, :, :, :n])
        assert torch.equal(now.scale[..., :n // 64], kv8.scale[..., :n // 64])
        kept += n > 0
        left += n < before
        stale += not torch.equal(now.data[:, :, :, n:before], kv8.data[:, :, :, n:before])
    kv8.raise_on_device_error()
    assert kept and left and stale, (kept, left, stale)
