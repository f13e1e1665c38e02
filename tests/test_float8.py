"""CPU: the e4m3 storage type of the binding and the oracle's rounding agree with each other and with torch's."""
import numpy as np
import torch

from cudabackend_b200 import api
from oracle import oracle as o


def test_code_values_match_torch():
    codes = torch.arange(256, dtype=torch.uint8)
    theirs = codes.view(torch.float8_e4m3fn).to(torch.float64).numpy()
    assert np.array_equal(api.FLOAT8_VALUES, theirs, equal_nan=True)
    assert np.nanmax(api.FLOAT8_VALUES) == 448.0


def test_rounding_matches_torch_and_the_oracle():
    r = np.random.default_rng(61)
    grid = api.FLOAT8_VALUES[:0x7F]
    midpoints = (grid[:-1] + grid[1:]) / 2
    v = np.concatenate([grid, midpoints, midpoints * (1 + 1e-6), midpoints * (1 - 1e-6), r.normal(0, 100, 5000), r.normal(0, 1e-2, 5000)])
    v = np.concatenate([v, -v]).astype(np.float32)
    v = v[np.abs(v) <= 448]
    codes = api.float_to_float8_bits(v)
    theirs = torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(codes, theirs)
    assert np.array_equal(api.float8_bits_to_float(codes), o.e4m3_round(v))


def test_saturation_and_nan():
    assert list(api.float_to_float8_bits([500.0, -1e9, np.nan, 0.0, -0.0])) == [0x7E, 0xFE, 0x7F, 0x00, 0x80]


def test_storage_round_trip():
    stored, values = api.to_storage(np.linspace(-448, 448, 1001), "float8_e4m3")
    assert stored.dtype == np.uint8 and api.DTYPE_SIZES["float8_e4m3"] == 1
    again, _ = api.to_storage(values, "float8_e4m3")
    assert np.array_equal(stored, again) and np.array_equal(api.from_storage(stored, "float8_e4m3"), values)


def test_bad_handles_are_refused_before_any_launch(library):
    assert api.call_status("cudaQuantizeBlocks", -1, -1, -1, -1, -1, -1, -1) == api.STATUS["INTERNAL_ERROR"]
    assert api.call_status("cudaRmsNormQuantize", -1, -1, -1, -1, -1, -1, -1, 1e-6, -1, -1, -1, -1) == api.STATUS["INTERNAL_ERROR"]
    assert api.call_status("cudaGemmBlockScaled", -1, 0, 1, None, -1, -1, -1, -1, -1, -1, -1, -1, None, -1, -1) == api.STATUS["INTERNAL_ERROR"]


def test_oracle_product_and_scales():
    r = np.random.default_rng(62)
    x = r.normal(0, 1, (200, 300))
    s1, s128 = o.block_scales(x), o.block_scales(x, 128)
    assert s1.shape == (200, 3) and s128.shape == (2, 3)
    assert np.isclose(s1[7, 2], np.abs(x[7, 256:]).max() / 448) and np.isclose(s128[1, 0], np.abs(x[128:, :128]).max() / 448)
    a = o.e4m3_round(x / o.spread_scales(s1, 200, 300))
    b = o.e4m3_round(x / o.spread_scales(s128, 200, 300, 128))
    got, size = o.gemm_block_scaled(a, s1, b, s128)
    assert np.all(np.abs(got - x @ x.T) <= 2.01 * 2.0 ** -4 * (np.abs(x) @ np.abs(x).T) + 1e-3)
    assert np.all(size >= np.abs(got))
