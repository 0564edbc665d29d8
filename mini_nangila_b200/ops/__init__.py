"""sm_100a kernel wrappers: codecs (``ops.codecs``) and the device ``.nz``
trajectory pipeline (``ops.trajectory``); the dense half of a decoder layer
(``ops.dense``, ``ops.norm``)."""
