"""The sweep of the products with a scale per row, and what the comment beside their pick says of it."""
from siglip_b200 import sweep

SCALED_CSV = sweep.PKG / "sweeps" / "b200_scaled.csv"


def test_the_constants_of_the_layers_pick_as_well_as_is_said():
    rows, variants = sweep.read_csv(SCALED_CSV), sweep.variant_tiles()
    assert len(rows) == 1900 and {int(r["M"]) for r in rows} >= {96, 46656} and {min(int(r["N"]) for r in rows), max(int(r["N"]) for r in rows)} == {144, 8192}
    layers = {"INT8": "NONE", "E4M3": "NONE", "INT8_GELU": "GELU", "E4M3_GELU": "GELU"}
    constants = {(cls, v): k for cls, layer in layers.items() for (c, v), k in sweep.cost_constants().items() if c == layer}
    for cls, points in sweep.model_regret(rows, constants, variants).items():
        lost, wide = [x for x, _ in points], [x for x, r in points if int(r["N"]) >= 512]
        assert cls in layers and 0.0085 < sum(lost) / len(lost) < 0.0115 and max(wide) < 0.175, cls
