"""BatchDecoder without a GPU: its options."""
import importlib

import pytest
import torch

TINY = dict(n_layers=2, d_model=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn=512, vocab=512,
            max_seq=70)


@pytest.fixture(scope="module")
def batch(pkg):
    return importlib.import_module("artifex-assistantv5_amd.batch_decoder")


def _config(**over):
    dec = importlib.import_module("artifex-assistantv5_amd.decoder")
    return dec.DecoderConfig(**{**TINY, **over})


def test_pages(batch):
    assert batch.check_batch(_config(), 3, None, 16, torch.float16) == (5, 15)
    assert batch.check_batch(_config(), 3, 7, 64, torch.bfloat16) == (2, 7)


@pytest.mark.parametrize("over,args,match", [
    (dict(head_dim=96), (3, None, 16, torch.float16), "glue kernels"),
    (dict(n_heads=18), (3, None, 16, torch.float16), "glue kernels"),
    ({}, (0, None, 16, torch.float16), "sequences"),
    ({}, (4097, None, 16, torch.float16), "sequences"),
    ({}, (3, None, 24, torch.float16), "24 slots"),
    ({}, (3, 0, 16, torch.float16), "0 pages"),
    ({}, (3, None, 16, torch.float32), "float16 or bfloat16"),
])
def test_refusals(batch, over, args, match):
    with pytest.raises(ValueError, match=match):
        batch.check_batch(_config(**over), *args)
