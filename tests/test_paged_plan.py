"""Whether attention over a paged cache takes a workgroup a head or divides the rows: decided from sizes on
the host and, where tokens' sequences are given, from lengths on the device by the rule tested here."""
import ctypes as C

import numpy as np
import pytest

import rustfox_amd as rf

N_CU, UNIT = 256, 64


def plan(n_head, n_kv, cap, n_seqs, length, seq=None, n_cu=N_CU):
    out, length = (C.c_int64 * 4)(), np.ascontiguousarray(length, np.uint32)
    seq = None if seq is None else np.ascontiguousarray(seq, np.uint32)
    rf.probe_lib().fox_gpu_paged_plan_probe(n_head, n_kv, len(length), cap, n_seqs, length.ctypes.data,
                                            None if seq is None else seq.ctypes.data, n_cu, out)
    p = dict(zip(("whole", "either", "workers", "items"), out))
    seen = np.minimum(length, cap).astype(np.int64)
    if seq is not None:
        seen[seq >= n_seqs] = 0
    units = -(-seen // UNIT)
    p["share"] = units.sum() * (p["items"] // len(length)) / (2 * n_cu)
    # the most units that one workgroup walks
    p["walk"] = int(units.max()) if p["whole"] else -(-int(units.sum() * (p["items"] // len(length))) // n_cu)
    return p


def mixed(decoding, longest, others, tokens, past):
    """(lengths, sequences) of one long and some short decoding sequences, and a prompt's tokens of one more."""
    return ([longest] + [others] * (decoding - 1) + [past + i for i in range(tokens)],
            list(range(decoding)) + [decoding] * tokens)


@pytest.mark.parametrize("n_head,n_kv", [(32, 8), (32, 16), (8, 2), (64, 8), (40, 40)])
@pytest.mark.parametrize("batch", [(31, 100000, 1000, 16, 900), (16, 131071, 700, 20, 0), (60, 50000, 300, 40, 5000),
                                   (3, 131071, 10, 500, 2000), (1, 131071, 0, 1000, 1)], ids=str)
def test_a_long_sequence_among_others_is_divided(n_head, n_kv, batch):
    """Tokens that share a sequence say nothing of the others' lengths: no workgroup walks more than twice an
    equal share (one a compute unit of divided rows)."""
    length, seq = mixed(*batch)
    p = plan(n_head, n_kv, 131072, batch[0] + 1, length, seq)
    assert p["walk"] <= 2 * p["share"] + 1, p
    assert not p["whole"] or n_kv == 40                      # (so many heads that each is near a share)


def test_any_batch_is_near_its_share():
    rng = np.random.default_rng(1)
    wholes = 0
    for _ in range(3000):
        M, n_kv = int(rng.integers(2, 1025)), int(rng.choice([1, 2, 4, 8, 16]))
        n_seqs = int(rng.choice([1, 2, 5, M]))
        seq = np.sort(rng.integers(0, n_seqs + 1, M))        # (the last is none)
        length = np.exp(rng.uniform(0, np.log(131072), M)).astype(int) if rng.random() < 0.5 else \
            rng.integers(3000, int(rng.choice([3100, 6000, 131072])), M)
        p = plan(4 * n_kv, n_kv, 131072, n_seqs, length, seq)
        wholes += p["whole"]
        assert p["walk"] <= 2 * p["share"] + 1, p
    assert 300 < wholes < 2700


def test_tokens_of_like_lengths_share_their_rows():
    """Prompts and drafts take a workgroup a head whatever the table's number of sequences."""
    for n_seqs in (1, 64, 512, 65535):
        for M, rows, n_kv in ((512, 9000, 8), (48, 9000, 8), (1024, 131000, 8), (300, 9000, 2), (1000, 1000, 8)):
            length = rows - M + 1 + np.arange(M)
            assert plan(4 * n_kv, n_kv, 131072, n_seqs, length, [0] * M)["whole"]
            # too few heads for the compute units: divided
            assert not plan(4, 1, 131072, n_seqs, length[-40:], [0] * min(M, 40))["whole"]
    drafts = [i for i in range(5) for _ in range(8)]
    assert plan(32, 8, 131072, 5, [4000] * 40, drafts)["whole"]
    # tokens of sequences of their own are divided, and so are those that come in no order
    assert not plan(32, 8, 131072, 512, [9000] * 512, np.arange(512))["whole"]
    assert not plan(32, 8, 131072, 2, [9000] * 512, np.arange(512) % 2)["whole"]


def test_sequences_that_are_none_have_no_rows():
    """Neither their lengths nor their being alike count."""
    length = [9000] * 400 + [131072] * 200
    assert plan(32, 8, 131072, 1, length, [0] * 400 + [7] * 200)["whole"]
    assert not plan(32, 8, 131072, 1, length, [0] * 200 + [7] * 400)["whole"]


def test_without_sequences_the_sizes_decide():
    for n, cap, whole in ((3, 400, True), (3, 416, False), (32, 2048, True), (32, 2064, False), (128, 3584, True),
                          (128, 3600, False)):
        p = plan(32, 8, cap, n, [cap] * n)
        assert p["whole"] == (whole if n > 3 else cap <= 400 + 1648 * (24 / 256) ** 3) and not p["either"]
