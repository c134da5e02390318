"""The planes of a cache in 4 bits that the cache manager makes, over pages and page counts of every alignment: what the operators take.
And its option of the command line."""
import itertools

import pytest
import torch

from tiny_inference_engine_b200.cache import CacheManager
from tiny_inference_engine_b200.ops import kv4
from tiny_inference_engine_b200.parts.base import CacheNeed


@pytest.mark.parametrize("head_dim", [64, 96, 192, 256, 7])
@pytest.mark.parametrize("kv_heads", [1, 2, 3])
def test_every_plane_is_one_that_the_operators_take(head_dim, kv_heads):
    for page, pages in itertools.product((1, 2, 3, 5, 6, 7, 8, 12), (1, 2, 5, 7, 8)):
        made = CacheManager([CacheNeed("full", kv_heads, head_dim)] * 3, page, num_pages=pages, dtype=torch.bfloat16, device="cpu", kv_bits=4)
        seen = set()
        for entry in range(3):
            four = made.layer_cache(entry, True).kv4
            planes, sizes = kv4._check_cache("planes", four)          # (refuses what is not contiguous or not 16-byte aligned)
            assert sizes == (kv_heads, head_dim, page, pages)
            for t in four[:4]:
                t.fill_(len(seen) + 1)
                seen.add(t.data_ptr())
        assert len(seen) == 12
        values = iter(range(1, 13))
        for entry in range(3):                                        # no plane reaches into another
            assert all(bool((t == next(values)).all()) for t in made.layer_cache(entry, True).kv4[:4])


@pytest.mark.parametrize("page,heads,pages,head_dim", [(5, 2, 7, 64), (6, 1, 7, 64), (2, 1, 5, 64), (1, 1, 3, 128)])
def test_the_operators_reach_their_last_check(page, heads, pages, head_dim):
    """Refused for the device alone, as any CPU tensor is, not for alignment."""
    from tiny_inference_engine_b200 import ops
    from tiny_inference_engine_b200.errors import InvalidArgument
    made = CacheManager([CacheNeed("full", heads, head_dim)] * 2, page, num_pages=pages, dtype=torch.bfloat16, device="cpu", kv_bits=4)
    x, slots = torch.zeros(1, heads * head_dim), torch.zeros(1, dtype=torch.int32)
    for entry in range(2):
        with pytest.raises(InvalidArgument, match="CUDA"):
            ops.kv4_append(x, x, slots, made.layer_cache(entry, True).kv4)


def test_the_command_line_names_the_option_and_refuses_other_bits_before_it_reads_a_model(capsys):
    from tiny_inference_engine_b200.cli.main import main
    assert main(["--help"]) == 0 and "--kv-bits" in capsys.readouterr().out
    assert main(["generate", "-m", "x", "-p", "1", "--kv-bits", "8"]) == 1 and "kv_bits must be 4" in capsys.readouterr().err
