from .history import HistoryEncoder
from .time_encode import TimeEncode

__all__ = ["HistoryEncoder", "TimeEncode"]
