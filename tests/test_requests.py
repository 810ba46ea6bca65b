"""The backbone's paths for many requests (pages, adapters, answers) on the CPU: what they refuse before anything runs."""
import pytest
import torch

from flashact_amd import kv8, lora, paged, prefill

NL = 2


def _shared():
    ln = [torch.zeros(NL, 2048) for _ in range(2)]
    packed = {k: torch.zeros(NL, n, m, dtype=torch.bfloat16)
              for k, n, m in (("wqkv", 4, 8), ("wo", 4, 8), ("wgu", 4, 8), ("wdn", 4, 8))}
    return ln, packed, paged.make_pools(NL, 6, device="cpu"), torch.zeros(2, 3, dtype=torch.int32)


def test_pages_and_adapters_that_do_not_fit():
    ln, packed, pools, table = _shared()
    index = torch.zeros(2, dtype=torch.int32)
    bank = lora.pack([(torch.zeros(8, 2048), torch.zeros(2560, 8), 1.0)])
    tests = ((dict(table=None), "belongs"), (dict(caches=kv8.make_caches(NL, 2, 64, device="cpu")), "belongs"),
             (dict(caches=paged.make_pools(NL, 6, 2, 256, device="cpu")), "caches"), (dict(caches=pools[:1]), "caches"),
             (dict(caches=paged.make_pools(NL, 6, dtype=torch.float16, device="cpu")), "bfloat16"), (dict(table=table[0]), "table"),
             (dict(adapters=([{}], index)), "adapters"), (dict(adapters=([{"wq": bank}] * NL, index)), "adapters"),
             (dict(adapters=([{}] * NL, index.long())), "index"), (dict(adapters=([{}] * NL, index[:1])), "index"))
    for kw, text in tests + ((dict(table=table[:1]), "hold"), (dict(lengths=[97, 1]), "hold")):
        with pytest.raises(ValueError, match=text):
            prefill.prefill_packed(**{"packed": packed, "ln_in": ln[0], "ln_post": ln[1], "x": torch.zeros(100, 2048), "lengths": [10, 10],
                                      "caches": pools, "table": table, **kw})
    for kw, text in tests + ((dict(x=torch.zeros(3, 1, 2048)), "x must"), (dict(x=torch.zeros(2, 33, 2048)), "x must")):
        with pytest.raises(ValueError, match=text):
            prefill.extend(**{"weights": [None] * NL, "ln_in": ln[0], "ln_post": ln[1], "x": torch.zeros(2, 1, 2048), "caches": pools,
                              "lens": index, "table": table, **kw})


def test_answers_that_are_refused():
    x, ln, head = torch.zeros(3, 2048), torch.zeros(2048), torch.zeros(9, 2048, dtype=torch.bfloat16)
    for kw, err, text in ((dict(x=x.half()), TypeError, "float32"), (dict(x=x[:, :8]), ValueError, "x must"), (dict(ln_final=ln[:5]), ValueError, "ln_final"),
                          (dict(head=head.float()), ValueError, "head"), (dict(head=head[:, :8]), ValueError, "head"), (dict(top=0), ValueError, "top")):
        with pytest.raises(err, match=text):
            prefill.answer(**{"head": head, "ln_final": ln, "x": x, **kw})


def test_entries_refuse_more_rows_than_a_grid_has():
    import ctypes
    from flashact_amd import _lib
    from tests import test_lora, test_tokens
    lib = _lib.lib()
    assert lib.fa_lora_add(ctypes.byref(test_lora._args(rows=(1 << 20) + 1, workspace_bytes=1 << 50)), None) == 1
    assert "2^20" in lib.fa_last_error().decode()
    assert lib.fa_token_logprobs(ctypes.byref(test_tokens._args(rows=(1 << 20) + 1, workspace_bytes=1 << 50)), None) == 1
    assert "2^20" in lib.fa_last_error().decode()
