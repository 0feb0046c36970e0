"""Calls of the operators of a cache in 8 bits with block scales, up to their launches: workspaces, addresses, bounds."""
import weakref

import pytest
import torch

import block_scaled_cases as K
from vllm_gcu_b200.ops import cuda as C


class Launches:
    """Stands in for the launches of ``ops.cuda`` on tensors of the host: their names and arguments, and whether the
    workspaces that were made for them are still held."""

    def __init__(self, monkeypatch):
        self.calls, self.made = [], []
        empty, new_empty = torch.empty, torch.Tensor.new_empty

        def recorded(make):
            def made(*args, **kw):
                t = make(*args, **kw)
                self.made.append(weakref.ref(t))
                return t
            return made

        def launch(dev, name, packed):
            self.calls.append((name, packed))
            assert all(t() is not None for t in self.made), f"{name}: a workspace was given back before the launch"

        monkeypatch.setattr(C, "_call_on", launch)
        monkeypatch.setattr(C, "_scaled_slots", lambda rows, int8, dev: (4 if rows <= 4 else 8 if rows <= 8 else 16, 296))
        monkeypatch.setattr(C, "_sms", lambda: 148)
        monkeypatch.setattr(torch, "empty", recorded(empty))
        monkeypatch.setattr(torch.Tensor, "new_empty", recorded(new_empty))

    def packed(self, name, fields):
        return [fields.unpack(p) for n, p in self.calls if n == name]


def _few_rows(cache, q, splits, window=0, first=0):
    """A launch of the kernel for few rows, as if the tensors lay on a GPU."""
    shape = list(C._scaled_cache(*cache.parts()))
    shape[6] = 0
    B, Hq, q, pq, ld, out, po, ldo = C._scaled_query(q, q.clone(), C._scaled_cache(*cache.parts()))
    C._scaled_rows(tuple(shape), B, Hq, q, pq, ld, po, ldo, 0, cache.seq_lens.data_ptr(), cache.tables.data_ptr(), B,
                   cache.tables.shape[1], 1, 0.1, window, first, splits, max(cache.lens))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_workspaces_are_held_until_the_launches_of_few_rows(D, monkeypatch):
    cache = K.Cache(K.FP8, 2, D, 16, [900, 40])
    q = torch.zeros(2, 8, D, dtype=K.BF16)
    launches = Launches(monkeypatch)
    _few_rows(cache, q, 12)
    assert [n for n, _ in launches.calls] == ["b200_block_scaled_rows"] and launches.made


def test_workspaces_are_held_between_expansion_and_attention(monkeypatch):
    q_lens, lens = [130, 200, 90], [130, 700, 333]
    cache = K.Cache(K.FP8, 2, 128, 16, lens)
    q = torch.zeros(sum(q_lens), 8, 128, dtype=K.BF16)
    cu = torch.tensor([0] + q_lens).cumsum(0).int()
    monkeypatch.setattr(C, "SCALED_ROWS", 0)
    monkeypatch.setattr(C, "SCALED_EXPANDED_KEYS", 900)
    out = torch.zeros_like(q)
    launches = Launches(monkeypatch)
    launch = C._call_on

    def one_workspace(dev, name, packed):                 # (the one of an earlier group of requests may go)
        launches.made = launches.made[-1:]
        launch(dev, name, packed)
    monkeypatch.setattr(C, "_call_on", one_workspace)
    C.block_scaled_prefill(q, *cache.parts(), cache.tables, cu, cache.seq_lens, 0.1, q_lens, lens, out=out)
    assert [n for n, _ in launches.calls] == ["b200_block_scaled_expand", "b200_fmha_expanded"] * 3 and launches.made


@pytest.mark.parametrize("D", [64, 128])
def test_queries_that_start_anywhere_are_copied(D, monkeypatch):
    """The kernels read rows 16 bytes at a time: contiguous rows behind an odd number of elements, rows at an odd pitch, one
    row for all tokens."""
    lens = [40, 33]
    cache, width = K.Cache(K.FP8, 2, D, 16, lens), 4 * D
    shape = C._scaled_cache(*cache.parts())
    wide = torch.randn(2 * width + 12).to(K.BF16)
    rows = [wide[o:o + 2 * width].view(2, 4, D) for o in (0, 1, 4, 7)]
    rows += [torch.as_strided(wide, (2, 4, D), (width + 4, D, 1)), wide[:width].view(1, 4, D).expand(2, 4, D)]
    rows.append(wide[3:3 + width].view(1, 4, D))
    for q in rows:
        T, Hq, held, pq, ld, _, _, _ = C._scaled_query(q, None, shape)
        assert pq == held.data_ptr() and pq % 16 == 0 and ld % 8 == 0 and ld >= width and torch.equal(held, q)
    monkeypatch.setattr(C, "SCALED_ROWS", 0)
    launches = Launches(monkeypatch)
    C.block_scaled_prefill(rows[1], *cache.parts(), cache.tables, torch.tensor([0, 1, 2], dtype=torch.int32), cache.seq_lens,
                           0.1, [1, 1], lens)
    assert all(p[0] % 16 == 0 for p in launches.packed("b200_fmha_expanded", C._EXPANDED_CALL))


@pytest.mark.parametrize("first", [2 ** 31 - 1, 2 ** 31 - 20, 2 ** 31 - 130, 5000])
def test_first_tokens_reach_no_further_than_the_tables(first, monkeypatch):
    """Kernels add up to 127 to the number of first tokens in 32 bits."""
    lens = [40, 333]
    cache = K.Cache(K.FP8, 2, 128, 16, lens)
    room = cache.tables.shape[1] * 16
    q, cu = torch.zeros(140, 8, 128, dtype=K.BF16), torch.tensor([0, 10, 140], dtype=torch.int32)
    monkeypatch.setattr(C, "SCALED_ROWS", 0)
    launches = Launches(monkeypatch)
    C.block_scaled_prefill(q, *cache.parts(), cache.tables, cu, cache.seq_lens, 0.1, [10, 130], lens, window=40, first=first)
    for name, fields in (("b200_block_scaled_expand", C._SCALED_EXPAND), ("b200_fmha_expanded", C._EXPANDED_CALL)):
        got, = launches.packed(name, fields)
        assert room in got and first not in got
    monkeypatch.setattr(C, "_scaled_rows", lambda *args: launches.calls.append(("rows", args)))
    C.block_scaled_decode(q[:2], *cache.parts(), cache.tables, cache.seq_lens, 0.1, window=40, first=first)
    assert launches.calls[-1][1][-4:-2] == (40, room)
    assert C._visible(40, 7, room) == (40, 7)


def test_tables_of_more_tokens_than_32_bits_hold_are_refused():
    cache = K.Cache(K.FP8, 2, 128, 16, [40])
    tables = torch.zeros(1, 1, dtype=torch.int32).expand(1, 1 << 27)
    q, cu = torch.zeros(1, 8, 128, dtype=K.BF16), torch.tensor([0, 1], dtype=torch.int32)
    with pytest.raises(ValueError, match="2.31 tokens"):
        C.block_scaled_decode(q, *cache.parts(), tables, cache.seq_lens, 0.1)
    with pytest.raises(ValueError, match="2.31 tokens"):
        C.block_scaled_prefill(q, *cache.parts(), tables, cu, cache.seq_lens, 0.1, [1], [40])


@pytest.mark.parametrize("model,kw,match", [
    ("tiny-fizunex", dict(sliding_window=8, sliding_window_first=4), "alike"),
    ("tiny-deepseek", dict(sliding_window=8, sliding_window_first=4), "alike"),
    ("llama-3-8b", dict(num_hidden_layers=1, hidden_size=64, intermediate_size=64, num_attention_heads=1, head_dim=64,
                        num_key_value_heads=1, vocab_size=64, sliding_window=8, sliding_window_first=-1), "first tokens"),
])
def test_first_tokens_of_models_without_them(model, kw, match):
    """Models whose attention takes no first tokens refuse them in place of leaving them out."""
    from vllm_gcu_b200 import LLM
    with pytest.raises(ValueError, match=match):
        LLM(model, device="cpu", dtype="float32", num_gpu_blocks=16, max_model_len=64, max_num_seqs=2, **kw)
