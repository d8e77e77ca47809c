"""The streams the library hands out and uses itself: all of the default priority, and queries answered while the builder's stream
is at work."""
import ctypes as C

import numpy as np
import pyarrow as pa
import pytest

import liquid_cache_amd as lc
from liquid_cache_amd import _native as N

pytestmark = pytest.mark.gpu
HINT = lc.CacheExpression.SUBSTRING_SEARCH


def test_a_created_stream_has_the_default_priority(gpu_cache):
    import torch
    torch.cuda.init()
    lib, h = N.load(), C.c_void_p()
    N.check(lib.lc_stream_create(gpu_cache.handle, C.byref(h)), gpu_cache.handle)
    try:
        assert torch.cuda.ExternalStream(h.value).priority == torch.cuda.Stream().priority == 0
    finally:
        N.check(lib.lc_stream_destroy(gpu_cache.handle, h), gpu_cache.handle)


def test_queries_on_one_table_while_another_ones_index_is_built(product_lib):
    """Counts of table A, on a created stream, from before the first LIKE on table B (it starts B's build) until B's index is in
    place; then B's own counts."""
    import torch
    rng = np.random.default_rng(5)
    words = ["google", "yandex", "mail", "maps", "search", "news"]
    cache = (lc.LiquidCacheBuilder.new().with_index_options(like_pipeline_min_entries=1)
             .with_option(N.OPT_LIKE_INDEX_ASYNC, 1).build())
    try:
        tables, want = [], []
        for t in range(4):
            ids, n = [], 0
            for b in range(12):
                rows = ["http://%s.%s/%d" % (words[rng.integers(6)], words[rng.integers(6)], rng.integers(1 << 20))
                        for _ in range(4096)]
                eid = lc.ParquetArrayID.new(t, 0, 2, b)
                cache.insert(eid, pa.array(rows), HINT)
                ids.append(eid)
                n += sum("google" in r for r in rows)
            tables.append(ids)
            want.append(n)
        expr = lc.LiquidExpr.try_new("like", "%google%", pa.string(), HINT)
        lib, h = N.load(), C.c_void_p()
        N.check(lib.lc_stream_create(cache.handle, C.byref(h)), cache.handle)
        side = torch.cuda.ExternalStream(h.value)
        with torch.cuda.stream(side):
            total = torch.zeros(2, dtype=torch.int64, device="cuda")
        scans = [cache.scan(ids) for ids in tables]

        def count(scan, slot):
            scan.eval_count(expr, 0, total.data_ptr() + 8 * slot, 0, 0, h.value)

        count(scans[0], 0)
        scans[0].index_wait()
        for t in (1, 2, 3):
            count(scans[t], 1)  # starts the build
            for _ in range(50):
                count(scans[0], 0)
                side.synchronize()
                assert int(total[0]) == want[0]
            assert int(total[1]) == want[t]
            scans[t].index_wait()
            count(scans[t], 1)
            side.synchronize()
            assert int(total[1]) == want[t]
        for s in scans:
            s.close()
        N.check(lib.lc_stream_destroy(cache.handle, h), cache.handle)
    finally:
        cache.close()


def test_a_background_build_of_several_pieces(product_lib):
    """An index of more workgroups than the builder launches at once (512; a workgroup fills 16 words of each of 512 slices), with
    short dictionaries among the full ones: counts per entry through the bigram and the unigram index it built."""
    rng = np.random.default_rng(6)
    cache = (lc.LiquidCacheBuilder.new().with_index_options(like_pipeline_min_entries=1)
             .with_option(N.OPT_LIKE_INDEX_ASYNC, 1).build())
    try:
        ids, flat = [], []
        for b in range(160):
            n = 8192 if b % 8 else int(rng.integers(1, 300))
            host = rng.integers(0, 40, n)
            rows = ["http://h%02d%s/%x" % (h, "google" if h % 13 == b % 13 else "", x)
                    for h, x in zip(host.tolist(), rng.permutation(1 << 16)[:n].tolist())]
            eid = lc.ParquetArrayID.new(9, b // 16, 2, b % 16)
            cache.insert(eid, pa.array(rows), HINT)
            ids.append(eid)
            flat.append(rows)
        scan = cache.scan(ids)
        # (79 rows of 1,024 hold the first needle and 2 the second: above and below the 16 up to which the bigram index answers)
        for needle, kernel in (("google", "k_str_pred"), ("h07google", "k_like_flat"), ("c", "k_like_scanall<unigram>")):
            want = [sum(needle in r for r in rows) for rows in flat]
            expr = lc.LiquidExpr.try_new("like", "%" + needle + "%", pa.string(), HINT)
            for _ in range(3):  # before or during the build, and through the index
                _, counts = scan.eval_to_host(expr)
                assert counts.astype(np.int64).tolist() == want
                scan.index_wait()
            assert N.LIKE_KERNEL_NAMES[int(scan.info().last_like_kernel)] == kernel
        assert int(scan.info().index_bytes) // (16 * 512 * 8) > 1024  # three pieces at least
        scan.close()
    finally:
        cache.close()
