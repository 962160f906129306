"""Options of the serving paths that the streaming architectures do not have fail their load with the option's name (no GPU needed: they are looked at
before any device is)."""
import pytest

from moonshine_amd import api


@pytest.mark.parametrize("options, says", [({"kv_dtype": "mxfp4"}, "kv_dtype"), ({"kv_dtype": "fp4"}, "kv_dtype"), ({"beam_width": "2"}, "beam_width")])
def test_streaming_architectures_refuse(tmp_path, capfd, options, says):
    with pytest.raises(api.MoonshineError):
        api.Transcriber(str(tmp_path), api.ARCH_TINY_STREAMING, dict({"vad_threshold": "0"}, **options))
    assert f"{says}: the streaming architectures" in capfd.readouterr().err
