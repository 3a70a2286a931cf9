"""Pool formats at configuration time: what could never be written is refused before pools are allocated, and the transfer
model charges for what the pools hold."""
import pytest

from distserve_b200 import transfer_model as T
from distserve_b200.config import CacheConfig, KVModelConfig, ParallelConfig
from distserve_b200.worker import KVWorker


@pytest.mark.parametrize("block_size", [1, 6, 18])
def test_quantised_blocks_of_no_multiple_of_four_tokens(block_size):
    CacheConfig(block_size, 8)
    with pytest.raises(ValueError, match="multiple of 4 tokens"):
        CacheConfig(block_size, 8, kv_format="e4m3")


@pytest.mark.parametrize("head_dim,dtype", [(128, "float32"), (72, "float16"), (8, "bfloat16"), (272, "float16")])
def test_quantised_pools_that_no_operator_could_write(head_dim, dtype):
    model = KVModelConfig(2, 4, head_dim, dtype)
    model.check_kv_format("model")
    with pytest.raises(ValueError, match="e4m3 pools hold rows of float16 or bfloat16"):
        model.check_kv_format("e4m3")
    with pytest.raises(ValueError, match="e4m3 pools hold rows of float16 or bfloat16"):
        KVWorker(0, "decoding", model, CacheConfig(16, 8, kv_format="e4m3"))


@pytest.mark.parametrize("head_dim,dtype", [(16, "float16"), (64, "bfloat16"), (80, "float16"), (256, "bfloat16")])
def test_quantised_pools_that_can_be_written(head_dim, dtype):
    KVModelConfig(2, 4, head_dim, dtype).check_kv_format("e4m3")


def test_the_transfer_model_charges_for_what_the_pools_hold():
    model, dec = KVModelConfig(40, 40, 128), ParallelConfig(2, 0, 1, 0)
    whole, quantised = (T.bytes_per_block_per_worker(model, dec, 16, f) for f in ("model", "e4m3"))
    assert whole == T.bytes_per_block_per_worker(model, dec, 16) == 2 * 40 * 20 * 16 * 128 * 2 and quantised == 2 * 40 * 20 * 16 * 132
    link = T.LinkModel(payload_GBps=1.0, awaited_call_us=0.0, chained_call_us=0.0)
    for f in (T.migration_seconds, T.exit_prefill_delay_ms):
        assert f(500, model, dec, 16, link, kv_format="e4m3") / f(500, model, dec, 16, link) == pytest.approx(132 / 256)
    assert T.effective_GBps(500, model, dec, 16, link, kv_format="e4m3") == pytest.approx(1.0)
    # a hand-off that only fits because the pools are quantised
    place = T.DecodePlacement(2, 1, link, 1.0)
    budget = 0.7 * T.exit_prefill_delay_ms(500, model, dec, 16, link)
    with pytest.raises(ValueError, match="no placement"):
        T.pick_decode_placement([place], [500], model, budget)
    assert T.pick_decode_placement([place], [500], model, budget, kv_format="e4m3")[0] is place
