"""Which kernels the cache, attention and sampling calls launch (recorded without a GPU): LDS limits, and that the GPU tests'
shapes reach every instance."""

import pytest

from launches import LdsLimit, Launch, built, kernels, pointers, record

HEADS = [(48, 4, 128), (24, 2, 256), (32, 8, 128), (32, 4, 64), (16, 16, 128), (20, 4, 96), (7, 1, 32), (3, 3, 8), (6, 2, 72),
         (10, 2, 160), (4, 2, 224), (34, 2, 192)]


def cached(sequences, t, hq, hk, d, max_pages, page, dtype):
    q, kc, ks, vc, vs, table, lengths, out, workspace = pointers(9)
    return "venturi_kv_attention_run", [q, kc, ks, vc, vs, table, lengths, out, workspace, 1 << 40, sequences, t, hq, hk, d, 100, page,
                                        max_pages, 0.1, dtype, None]


def packed(tokens, keys, sequences, hq, hk, d, dtype):
    q, k, v, qo, ko, out, workspace = pointers(7)
    return "venturi_packed_attention_run", [q, k, v, qo, ko, out, workspace, 1 << 40, tokens, keys, sequences, hq, hk, d, 0.1, dtype, None]


def sample(rows, vocab, dtype):
    logits, u, tokens = pointers(3)
    return "venturi_sample_run", [logits, u, None, None, None, None, tokens, None, rows, vocab, dtype, None]


def reached(calls):
    return {kernel for launched in kernels([(0, *call) for call in calls]) for kernel in launched}


def test_cached_attention_tests_reach_every_instance():
    calls = [cached(6, t, hq, hk, d, 9, 32, dtype) for hq, hk, d in HEADS for t in (1, 5) for dtype in (0, 1)]
    calls += [cached(2, t, 2 * hk, hk, d, 9, 32, dtype) for hk, d in ((1, 32), (2, 64), (4, 96), (4, 128), (2, 160), (2, 192), (2, 224), (2, 256))
              for t in (5, 12, 33) for dtype in (0, 1)]
    assert built("kv_attention") | built("kv_attention_join") <= reached(calls)


def test_cached_attention_of_one_short_page_has_no_join():
    launched = kernels([(0, *cached(3, 1, 8, 2, 64, 8, 16, 0)), (0, *cached(3, 1, 8, 2, 64, 9, 16, 0))])
    assert [len(names) for names in launched] == [1, 2]


def test_packed_attention_tests_reach_every_instance():
    calls = [packed(208, 253, 3, hq, hk, d, dtype) for hq, hk, d in HEADS for dtype in (0, 1)]
    calls += [packed(5, 1505, 1, hk, hk, d, dtype) for hk, d in ((1, 32), (1, 64), (1, 96), (1, 128), (1, 160), (1, 192), (1, 224), (1, 256))
              for dtype in (0, 1)]
    assert built("packed_attention") | built("packed_attention_join") <= reached(calls)


def test_packed_attention_splits_only_few_rows_over_many_keys():
    shapes = {(5, 1505, 1): 2, (8192, 8192, 1): 1, (77, 77, 1): 1, (512, 512, 1): 1, (4096, 16000, 11): 1}
    for (tokens, keys, sequences), count in shapes.items():
        assert len(kernels([(0, *packed(tokens, keys, sequences, 48, 4, 128, 0))])[0]) == count


@pytest.mark.parametrize("call", [cached(4, 1, 48, 4, 128, 100, 64, 1), cached(4, 5, 24, 2, 256, 100, 32, 0), sample(3, 1000, 0)])
def test_lds_limits_are_raised_on_every_device(call):
    limits = {}
    for events in record([(device, *call) for device in (0, 1, 0, 70)]):
        large = 0
        for e in events:
            if isinstance(e, LdsLimit):
                limits[e.kernel, e.device] = e.bytes
            elif isinstance(e, Launch) and e.shared > 65536:
                large += 1
                assert limits.get((e.kernel, e.device), 0) >= e.shared
        assert large == 1
